"""The weight's gradient from activations kept in 8 bits when the rows' scales differ by more than FP16's exponents hold.

Tolerances as in test_fp8_linear_gpu.py: x enters the product without rounding, dz rounded to FP16 (2^-11 of it and half a
subnormal step, 2^-25), and the sum of m terms (2 m where dz comes in two parts) loses at most 2^-23 of the magnitudes for each.
"""
import pytest

pytestmark = pytest.mark.gpu

CODES = {"f32": 0, "f16": 1, "bf16": 2}
ACTS = {"none": 0, "relu": 1, "silu": 3}


def kept(dev, x):
    """x as quantize_fp8 keeps it: codes, scales, and the values they stand for in 64 bits."""
    torch = dev.torch
    m, k = x.shape
    q = torch.empty(m, k, dtype=torch.uint8, device=dev.dev)
    s = torch.empty(-(-k // 128), m, device=dev.dev)
    dev.check(dev.lib.cudeep_b200_quantize_fp8(dev.ptr(x), 0, m, k, 1, dev.ptr(q), dev.ptr(s), None))
    return q, s, q.view(torch.float8_e4m3fn).double() * s.double().t().repeat_interleave(128, 1)[:, :k]


def gradient(dev, dy, x8, xs, z8, zs, act, w, m, n, k, out, asked=("dx", "dw", "db")):
    torch = dev.torch
    t = torch.float32 if out == "f32" else torch.float16
    res = {"dx": torch.full((m, k), float("nan"), device=dev.dev, dtype=torch.float16),
           "dw": torch.full((n, k), float("nan"), device=dev.dev, dtype=t), "db": torch.full((n,), float("nan"), device=dev.dev)}
    p = dev.ptr
    dev.check(dev.lib.cudeep_b200_linear_backward_saved_fp8(
        p(dy), 1, p(x8), p(xs), p(z8) if act else None, p(zs) if act else None, act, p(w),
        p(res["dx"]) if "dx" in asked else None, p(res["dw"]), CODES[out], p(res["db"]) if "db" in asked else None, m, n, k, None))
    assert dev.sync_status() == 0
    return res


def rows(torch, gen, m, k, kind, dev):
    """Activations: `tiny` ones (1e-6) with rows of zeros among them, whose scale is 1; `outlier`: one row 2^30 times the others;
    `columns`: blocks of columns of very different sizes in every row, rows apart too; `near`: within FP16's reach."""
    x = torch.randn(m, k, generator=gen, device=dev)
    x[:, 0] += 2 * torch.sign(x[:, 0])
    if kind == "tiny":
        x *= 1e-6
        x[1::3] = 0
    elif kind == "outlier":
        x[m // 2] *= 2.0 ** 30
    elif kind == "columns":
        x *= torch.exp2(torch.randint(-20, 21, (m, -(-k // 128)), generator=gen, device=dev).float()).repeat_interleave(128, 1)[:, :k]
    return x


@pytest.mark.parametrize("out", ["f16", "f32"])
@pytest.mark.parametrize("act", sorted(ACTS))
@pytest.mark.parametrize("kind", ["tiny", "outlier", "columns", "near"])
@pytest.mark.parametrize("m,n,k", [(40, 130, 72), (333, 77, 101), (300, 256, 384), (64, 300, 520), (2500, 64, 136), (1100, 512, 512),
                                   (150, 2600, 1900), (4100, 2048, 1024)])
def test_gradient_of_the_weight(dev, m, n, k, kind, act, out):
    torch = dev.torch
    gen = torch.Generator(device=dev.dev).manual_seed(m + n + k)
    x = rows(torch, gen, m, k, kind, dev.dev)
    x8, xs, x64 = kept(dev, x)
    z8, zs, z = kept(dev, torch.randn(m, n, generator=gen, device=dev.dev))
    dy = torch.randn(m, n, generator=gen, device=dev.dev).half()
    if kind == "outlier":
        dy[m // 2] = 0      # nothing of the large row may be left in the others' gradient, nor of them be lost beside it
    w = (torch.randn(n, k, generator=gen, device=dev.dev) / n ** 0.5).half()
    res = gradient(dev, dy, x8, xs, z8, zs, ACTS[act], w, m, n, k, out)
    slope = {"none": torch.ones_like(z), "relu": (z > 0).double(), "silu": torch.sigmoid(z) * (1 + z * torch.sigmoid(-z))}[act]
    dz = dy.double() * slope
    off = 0 * dz
    if act == "silu":      # the slope in FP32: see test_fp8_linear_gpu.py
        off = dy.double().abs() * 2.0 ** -20 * z.abs().clamp(min=1)
    if act != "none":
        off = off + 2.0 ** -11 * dz.abs() + 2.0 ** -25
    want = dz.t() @ x64
    off = off * (dy != 0)      # zero stays zero
    bound = off.t() @ x64.abs()
    bound = bound + 2 * m * 2.0 ** -23 * (dz.abs().t() @ x64.abs())
    if out == "f16":
        bound = bound + 2.0 ** -11 * (want.abs() + bound) + 2.0 ** -25
        big = want.abs() + bound >= 65504      # a value that FP16 holds as infinity
        got = torch.where(big, want, res["dw"].double())
    else:
        got = res["dw"].double()
    assert not got.isnan().any()
    worst = ((got - want).abs() - bound).max().item()
    assert worst <= 0, worst
    if kind == "tiny" and out == "f32":      # and it is the gradient, not zeros
        assert (got - want).norm() <= 0.01 * want.norm()
    only = gradient(dev, dy, x8, xs, z8, zs, ACTS[act], w, m, n, k, out, ("dw",))
    assert torch.equal(only["dw"], res["dw"])


def test_scales_that_are_zero_not_powers_of_two_or_not_finite(dev):
    """A zero scale stands for zeros; other scales enter as they are (rounded to 16 bits with the code); NaN stays in its columns."""
    torch = dev.torch
    m, n, k = 200, 136, 300
    gen = torch.Generator(device=dev.dev).manual_seed(3)
    x8, xs, _ = kept(dev, torch.randn(m, k, generator=gen, device=dev.dev))
    dy = torch.randn(m, n, generator=gen, device=dev.dev).half()
    w = torch.randn(n, k, generator=gen, device=dev.dev).half()
    for wide in (False, True):
        s = (torch.rand(xs.shape, generator=gen, device=dev.dev) + 0.5) * 2.0 ** -9
        s[:, 5] = 0
        if wide:
            s[:, ::7] *= 2.0 ** -30
        s[1, 9] = float("nan")
        res = gradient(dev, dy, x8, s, None, None, 0, w, m, n, k, "f32")["dw"].double()
        x = x8.view(torch.float8_e4m3fn).double() * s.double().t().repeat_interleave(128, 1)[:, :k]
        keep = torch.ones(k, dtype=torch.bool, device=dev.dev)
        keep[128:256] = False
        assert res[:, 128:256].isnan().all()
        want, size = dy.double().t() @ x[:, keep], dy.double().abs().t() @ x.abs()[:, keep]
        # x rounded: 2^-8 of it where it is taken in bfloat16, else 2^-11 and half a subnormal step of the largest scale.
        bound = size * (2.0 ** -8 if wide else 2.0 ** -11) + 2 * m * 2.0 ** -23 * size
        if not wide:
            bound = bound + 2.0 ** -25 * s.nan_to_num().max().double() * dy.double().abs().sum(0)[:, None]
        assert ((res[:, keep] - want).abs() <= bound).all()


@pytest.mark.parametrize("kind", ["tiny", "near"])
def test_infinities_stay_in_their_features(dev, kind):
    torch = dev.torch
    m, n, k = 200, 136, 264
    gen = torch.Generator(device=dev.dev).manual_seed(4)
    x8, xs, x64 = kept(dev, rows(torch, gen, m, k, kind, dev.dev))
    dy = torch.randn(m, n, generator=gen, device=dev.dev).half()
    dy[0, 3], dy[0, 70], dy[2, 130] = float("inf"), float("nan"), -float("inf")
    w = torch.zeros(n, k, dtype=torch.float16, device=dev.dev)
    got = gradient(dev, dy, x8, xs, None, None, 0, w, m, n, k, "f32", ("dw",))["dw"].double()
    want = dy.double().t() @ x64
    fine = torch.ones(n, dtype=torch.bool, device=dev.dev)
    fine[[3, 70, 130]] = False
    assert ((got - want)[fine].abs() <= 2 * m * 2.0 ** -23 * (dy[:, fine].double().abs().t() @ x64.abs())).all()
    assert torch.equal(got[~fine].isnan(), want[~fine].isnan())
    inf = want.isinf()
    assert torch.equal(got[inf], want[inf]) and bool(inf.any())


@pytest.mark.parametrize("m,n,k,act", [(333, 77, 101, 3), (1, 64, 64, 0), (2500, 64, 136, 0), (1030, 520, 264, 1)])
def test_captured_calls_follow_the_scales_of_each_replay(dev, m, n, k, act):
    """Which form x is taken in is decided on the device: a graph replayed on other activations gives what a call of its own
    gives, and two graphs side by side do not share what they decide by."""
    torch = dev.torch
    gen = torch.Generator(device=dev.dev).manual_seed(11)
    p = dev.ptr
    z8, zs, _ = kept(dev, torch.randn(m, n, generator=gen, device=dev.dev))
    dy = torch.randn(m, n, generator=gen, device=dev.dev).half()
    w = (torch.randn(n, k, generator=gen, device=dev.dev) / n ** 0.5).half()
    kinds = ["near", "tiny", "columns", "near", "outlier"]
    inputs = [kept(dev, rows(torch, gen, m, k, kind, dev.dev))[:2] for kind in kinds]
    want = [gradient(dev, dy, x8, xs, z8, zs, act, w, m, n, k, "f32", ("dx", "dw", "db")) for x8, xs in inputs]
    slots, graphs = [], []
    for _ in range(2):
        x8, xs = (t.clone() for t in inputs[0])
        dx, dw, db = (torch.full_like(t, float("nan")) for t in (want[0]["dx"], want[0]["dw"], want[0]["db"]))
        g = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(g):
            stream = torch.cuda.current_stream().cuda_stream
            dev.check(dev.lib.cudeep_b200_linear_backward_saved_fp8(p(dy), 1, p(x8), p(xs), p(z8) if act else None,
                                                                    p(zs) if act else None, act, p(w), p(dx), p(dw), 0, p(db),
                                                                    m, n, k, stream))
        slots.append((x8, xs, dx, dw, db))
        graphs.append(g)
    side = [torch.cuda.Stream() for _ in range(2)]
    for i in range(len(kinds)):
        pair = (i, (i + 1) % len(kinds))
        for j, at in enumerate(pair):
            slots[j][0].copy_(inputs[at][0])
            slots[j][1].copy_(inputs[at][1])
            for t in slots[j][2:]:
                t.fill_(float("nan"))
        torch.cuda.synchronize()
        for j in range(2):
            with torch.cuda.stream(side[j]):
                graphs[j].replay()
        assert dev.sync_status() == 0
        for j, at in enumerate(pair):
            for t, key in zip(slots[j][2:], ("dx", "dw", "db")):
                assert torch.equal(t, want[at][key])
