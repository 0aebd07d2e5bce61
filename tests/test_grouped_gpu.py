"""Grouped products with ragged sizes against the same products in 64 bits.

Tolerances.  Products of 16-bit values are exact in FP32 and sums are FP32, so a result is off by the accumulation and by
the rounding to its type.  The accumulation of n terms is held to n * 2^-23 * sum|a||b|: the tensor core may truncate
each partial sum, by at most 2^-23 of a value that never exceeds the sum of magnitudes.  The rounding adds
torch.finfo(t).eps / 2 (bf16 2^-8, fp16 2^-11) of the value, and the smallest subnormal.
"""
import pytest

pytestmark = pytest.mark.gpu

TYPES = {"f16": 1, "bf16": 2}


def make(dev, sizes, n, k, t, seed, pad=3, lead=0):
    torch = dev.torch
    gen = torch.Generator(device=dev.dev).manual_seed(seed)
    rows = lead + sum(sizes) + pad
    off = [lead]
    for s in sizes:
        off.append(off[-1] + s)
    offsets = torch.tensor(off, dtype=torch.int32, device=dev.dev)
    x = torch.randn(rows, k, generator=gen, device=dev.dev).to(t)
    w = (torch.randn(len(sizes), n, k, generator=gen, device=dev.dev) / k ** 0.5).to(t)
    dy = torch.randn(rows, n, generator=gen, device=dev.dev).to(t)
    return rows, off, offsets, x, w, dy


def close(torch, got, want, magnitude, terms):
    """|got - want| <= accumulation + rounding, elementwise; want and magnitude in 64 bits."""
    info = torch.finfo(got.dtype)
    bound = terms * 2.0 ** -23 * magnitude
    if got.dtype != torch.float32:
        bound = bound + info.eps / 2 * (want.abs() + bound) + info.smallest_normal * info.eps
    err = (got.double() - want).abs()
    assert not got.isnan().any()
    worst = (err - bound).max().item() if err.numel() else 0.0
    assert worst <= 0, f"off by {worst} more than allowed, largest error {err.max().item()}"


def call(dev, name, *args):
    dev.check(getattr(dev.lib, f"cudeep_b200_grouped_matmul_{name}")(*args))
    assert dev.sync_status() == 0


CASES = [
    ([1], 64, 64),
    ([5], 128, 128),
    ([0, 7, 0], 256, 64),
    ([16, 33, 1, 64], 256, 192),
    ([300], 512, 256),
    ([257, 0, 31, 129, 128], 384, 320),
    ([40, 3], 130, 72),          # features end inside a tile
    ([17, 50], 77, 101),         # odd row lengths: padded copies
    ([600, 700], 640, 64),
    ([1] * 40, 136, 136),
]


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("sizes,n,k", CASES)
def test_nt(dev, sizes, n, k, dtype):
    torch = dev.torch
    t = {"f16": torch.float16, "bf16": torch.bfloat16}[dtype]
    rows, off, offsets, x, w, _ = make(dev, sizes, n, k, t, 1, lead=2)
    y = torch.full((rows, n), 7.0, dtype=t, device=dev.dev)
    call(dev, "nt", dev.ptr(x), dev.ptr(w), dev.ptr(y), TYPES[dtype], dev.ptr(offsets), len(sizes), rows, n, k, None)
    assert bool((y[:off[0]] == 7).all()) and bool((y[off[-1]:] == 7).all())      # rows of no group
    for g in range(len(sizes)):
        r = slice(off[g], off[g + 1])
        a, b = x[r].double(), w[g].double()
        close(torch, y[r], a @ b.t(), a.abs() @ b.abs().t(), k)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("sizes,n,k", CASES)
def test_nn(dev, sizes, n, k, dtype):
    torch = dev.torch
    t = {"f16": torch.float16, "bf16": torch.bfloat16}[dtype]
    rows, off, offsets, _, w, dy = make(dev, sizes, n, k, t, 2)
    dx = torch.full((rows, k), 7.0, dtype=t, device=dev.dev)
    call(dev, "nn", dev.ptr(dy), dev.ptr(w), dev.ptr(dx), TYPES[dtype], dev.ptr(offsets), len(sizes), rows, k, n, None)
    assert bool((dx[off[-1]:] == 7).all())
    for g in range(len(sizes)):
        r = slice(off[g], off[g + 1])
        a, b = dy[r].double(), w[g].double()
        close(torch, dx[r], a @ b, a.abs() @ b.abs(), n)


@pytest.mark.parametrize("out", ["same", "f32"])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("sizes,n,k", CASES + [([2500, 15, 4100], 136, 200)])
def test_tn(dev, sizes, n, k, dtype, out):
    torch = dev.torch
    t = {"f16": torch.float16, "bf16": torch.bfloat16}[dtype]
    rows, off, offsets, x, _, dy = make(dev, sizes, n, k, t, 3, lead=1)
    # What lies beside a group must not reach its sums.
    x[:off[0]], x[off[-1]:] = float("nan"), float("inf")
    dy[:off[0]], dy[off[-1]:] = float("inf"), float("nan")
    to = torch.float32 if out == "f32" else t
    dw = torch.full((len(sizes), n, k), 7.0, dtype=to, device=dev.dev)
    call(dev, "tn", dev.ptr(dy), dev.ptr(x), dev.ptr(dw), TYPES[dtype], 0 if out == "f32" else TYPES[dtype],
         dev.ptr(offsets), len(sizes), rows, n, k, None)
    for g in range(len(sizes)):
        r = slice(off[g], off[g + 1])
        a, b = dy[r].double(), x[r].double()
        close(torch, dw[g], a.t() @ b, a.abs().t() @ b.abs(), max(1, sizes[g]))


# Few tiles of long sums: clusters of CTAs share them, each with a range of K; and few rows for each of many groups.
FEW = [
    ([1], 64, 4096),
    ([3, 0, 2, 1], 130, 2050),
    ([20, 0, 13], 256, 1600),
    ([100], 300, 1100),
    ([0, 1, 0, 0, 2] + [0] * 20 + [1, 0, 3, 0, 0, 1], 208, 4091),
    ([5, 6], 512, 520),
    ([1] * 37, 520, 192),        # tiles of fewer than 128 features
    ([4, 0, 9] * 5, 1000, 256),
    ([2] * 70, 300, 72),
]


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("sizes,features,k", FEW)
def test_few_tiles_of_long_sums(dev, sizes, features, k, dtype):
    """nt sums over k, nn the transposed weight over k: as the other sizes, and the same bits again."""
    torch = dev.torch
    t = {"f16": torch.float16, "bf16": torch.bfloat16}[dtype]
    rows, off, offsets, x, w, _ = make(dev, sizes, features, k, t, 4, lead=1)
    wt = w.transpose(1, 2).contiguous()
    for name, weight in (("nt", w), ("nn", wt)):
        results = []
        for _ in range(2):
            y = torch.full((rows, features), 7.0, dtype=t, device=dev.dev)
            call(dev, name, dev.ptr(x), dev.ptr(weight), dev.ptr(y), TYPES[dtype], dev.ptr(offsets), len(sizes), rows, features, k,
                 None)
            results.append(y)
        y = results[0]
        assert torch.equal(y, results[1])
        assert bool((y[:off[0]] == 7).all()) and bool((y[off[-1]:] == 7).all())
        for g in range(len(sizes)):
            r = slice(off[g], off[g + 1])
            a, b = x[r].double(), w[g].double()
            close(torch, y[r], a @ b.t(), a.abs() @ b.abs().t(), k)


def test_few_tiles_with_bad_offsets(dev):
    """Ranges that overlap make more tiles than the rows can have: reported, and nothing outside the matrix is written."""
    torch = dev.torch
    rows, n, k, groups = 4, 128, 4096, 12
    x = torch.ones(rows, k, dtype=torch.bfloat16, device=dev.dev)
    w = torch.ones(groups, n, k, dtype=torch.bfloat16, device=dev.dev)
    offsets = torch.tensor([0, 4] * 6 + [0], dtype=torch.int32, device=dev.dev)
    y = torch.full((rows + 8, n), 7.0, dtype=torch.bfloat16, device=dev.dev)
    dev.check(dev.lib.cudeep_b200_grouped_matmul_nt(dev.ptr(x), dev.ptr(w), dev.ptr(y[4]), 2, dev.ptr(offsets), groups, rows, n, k,
                                                    None))
    assert dev.sync_status() == 6
    assert bool((y[:4] == 7).all()) and bool((y[8:] == 7).all())
