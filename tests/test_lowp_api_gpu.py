"""The low-precision and grouped products as a program uses them: layers, streams, captured graphs, sizes at the edges."""
import ctypes

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def cd(lib, cuda):
    import cudeep_b200
    return cudeep_b200


def rel(a, b):
    a, b = np.asarray(a, np.float64), np.asarray(b, np.float64)
    return np.linalg.norm(a - b) / np.linalg.norm(b)


def bf16(a):
    """float32 values rounded to bfloat16 (nearest even)."""
    u = np.ascontiguousarray(a, np.float32).view(np.uint32)
    return ((u + 0x7fff + ((u >> 16) & 1)) & np.uint32(0xffff0000)).view(np.float32)


def gelu64(z):
    return z / (1 + np.exp(-2 * np.sqrt(2 / np.pi) * (z + 0.044715 * z ** 3)))


def slope64(f, z, h=1e-4):
    """Central differences: off by h^2 / 6 times a third derivative below 3, 5e-9."""
    return (f(z + h) - f(z - h)) / (2 * h)


# ---- layers ---------------------------------------------------------------------------------------------------------------


def test_cast_and_host_copies(cd):
    rng = np.random.default_rng(0)
    x = rng.standard_normal((37, 51)).astype(np.float32)
    t = cd.Tensor.from_numpy(x)
    b = t.to(cd.DType.bfloat16)
    assert np.array_equal(b.numpy(), bf16(x))
    assert np.array_equal(b.to(cd.DType.float32).numpy(), bf16(x))
    i = np.arange(9, dtype=np.int32)
    assert np.array_equal(cd.Tensor.from_numpy(i).numpy(), i)


@pytest.mark.parametrize("tiles", [False, True])
def test_quantize_round_trip(cd, tiles):
    """A value is off by at most half a step of e4m3: 2^-4 of it, or half the smallest step (2^-10 of the scale)."""
    rng = np.random.default_rng(1)
    x = (rng.standard_normal((130, 300)) * np.exp(rng.standard_normal((130, 1)))).astype(np.float32)
    q = cd.quantize_fp8(cd.Tensor.from_numpy(x), tiles)
    y = q.dequantize().numpy()
    s = q.scales.numpy()
    spread = (np.repeat(np.repeat(s, 128, 0)[:130], 128, 1) if tiles else np.repeat(s.T, 128, 1))[:, :300]
    assert (np.abs(y - x) <= np.maximum(2.0 ** -4 * np.abs(x), 2.0 ** -10 * spread)).all()
    assert np.array_equal(q.data.numpy() * spread, y)
    # Kept in a little over a byte per value: a scale per 128 columns of a row, or per block.
    assert q.nbytes() == 130 * 300 + 4 * (2 * 3 if tiles else 3 * 130)


@pytest.mark.parametrize("activation", [None, "gelu", "relu"])
def test_linear_fp8_training_step(cd, activation):
    """Forward, what is kept, and backward of one layer together, against 64 bits on the very values that were kept."""
    rng = np.random.default_rng(2)
    m, n, k = 200, 130, 264
    layer = cd.nn.LinearFp8(k, n)
    w = (rng.standard_normal((n, k)) / np.sqrt(k)).astype(np.float32)
    layer.load_state_dict({"weight": w, "bias": rng.standard_normal(n).astype(np.float32)})
    x = rng.standard_normal((m, k)).astype(np.float32)
    y, saved = layer.forward_saved(cd.Tensor.from_numpy(x), activation)
    x64 = saved[0].dequantize().numpy().astype(np.float64)
    w64 = layer.weight_fp8().dequantize().numpy().astype(np.float64)
    b64 = layer._parameters["bias"].numpy().astype(np.float64)
    z64 = x64 @ w64.T + b64
    f = {None: lambda z: z, "gelu": gelu64, "relu": lambda z: np.maximum(z, 0)}[activation]
    assert rel(y.numpy(), f(z64)) <= 1e-5            # FP32 sums and activations of exact products
    assert np.array_equal(layer(cd.Tensor.from_numpy(x)).numpy(), layer.forward_saved(cd.Tensor.from_numpy(x))[0].numpy())
    dy = bf16(rng.standard_normal((m, n)))
    dx, dw, db = layer.backward(cd.Tensor.from_numpy(dy).to(cd.DType.bfloat16), saved)
    if activation is None:
        dz = dy.astype(np.float64)
    else:
        z_kept = saved[1].dequantize().numpy().astype(np.float64)
        dz = dy * (slope64(f, z_kept) if activation == "gelu" else (z_kept > 0))
    # dz enters the products rounded to bfloat16, and so does dx leave: each off by at most 2^-8 of a value.
    step = 2.0 ** -8
    assert rel(db.numpy(), dz.sum(0)) <= 1e-5
    assert rel(dw.numpy(), dz.T @ x64) <= (step if activation else 1e-5)
    assert rel(dx.numpy(), dz @ bf16(w).astype(np.float64)) <= 2 * step


def test_linear_fp8_in_sequential_and_refresh(cd):
    rng = np.random.default_rng(3)
    x = cd.Tensor.from_numpy(rng.standard_normal((33, 96)).astype(np.float32))
    a, b = cd.nn.LinearFp8(96, 160), cd.nn.LinearFp8(160, 40, bias=False)
    fused = cd.nn.Sequential(a, cd.nn.GELU(), b)(x).numpy()
    plain = cd.nn.Sequential(a, cd.nn.GELU(), b, fuse=False)(x).numpy()
    # The same products; the two forms of GELU differ in the last bits, which may move a code of the second layer's input
    # by a step (2^-3 of one of 160 terms) now and then.
    assert rel(fused, plain) <= 1e-2
    before = b(cd.Tensor.ones([4, 160])).numpy()
    b._parameters["weight"].fill_(0.5)
    b.refresh()
    assert np.array_equal(b(cd.Tensor.ones([4, 160])).numpy(), np.full((4, 40), 80, np.float32)) and before.shape == (4, 40)
    b.load_state_dict({"weight": np.full((40, 160), 0.25, np.float32)})
    assert np.array_equal(b(cd.Tensor.ones([4, 160])).numpy(), np.full((4, 40), 40, np.float32))
    y16 = a(x.to(cd.DType.bfloat16))
    assert y16.dtype() == cd.DType.bfloat16 and y16.shape() == [33, 160]


def test_grouped_layer_is_adjoint(cd):
    """<dy, x W^T> = <dx, x> = <dW, W>: the products are linear, so their gradients have to give the same number."""
    rng = np.random.default_rng(4)
    sizes = [5, 0, 130, 64, 1]
    rows, k, n = sum(sizes) + 3, 72, 136
    layer = cd.nn.GroupedLinear(len(sizes), k, n)
    off = cd.Tensor.from_numpy(np.concatenate([[0], np.cumsum(sizes)]).astype(np.int32))
    xn, gn = bf16(rng.standard_normal((rows, k))), bf16(rng.standard_normal((rows, n)))
    x, g = (cd.Tensor.from_numpy(v).to(cd.DType.bfloat16) for v in (xn, gn))
    y = layer(x, off).numpy().astype(np.float64)
    dx, dw = layer.backward(g, x, off)
    dx, dw = dx.numpy().astype(np.float64), dw.numpy().astype(np.float64)
    w = layer.weight_bf16().numpy().astype(np.float64)
    used = sum(sizes)
    assert (y[used:] == 0).all() and (dx[used:] == 0).all() and (dw[1] == 0).all()
    a, b, c = (gn * y).sum(), (dx * xn).sum(), (dw * w).sum()
    # y and dx are rounded by at most 2^-8 of each value.
    assert abs(a - c) <= 2.0 ** -8 * np.abs(gn * y).sum() and abs(b - c) <= 2.0 ** -8 * np.abs(dx * xn).sum()
    start = 0
    for i, s in enumerate(sizes):
        r = slice(start, start + s)
        assert s == 0 or rel(y[r], xn[r].astype(np.float64) @ w[i].T) <= 2.0 ** -8
        start += s


def test_activation_by_name_code_or_none(cd):
    rng = np.random.default_rng(4)
    x = cd.Tensor.from_numpy(rng.standard_normal((5, 96)).astype(np.float32))
    layer = cd.nn.LinearFp8(96, 40)
    plain = layer.forward_saved(x)
    for none in ("none", 0):
        y, saved = layer.forward_saved(x, none)
        assert np.array_equal(y.numpy(), plain[0].numpy()) and saved[1] is None
        dy = cd.Tensor.from_numpy(rng.standard_normal((5, 40)).astype(np.float32)).to(cd.DType.bfloat16)
        for a, b in zip(layer.backward(dy, saved), layer.backward(dy, plain[1])):
            assert np.array_equal(a.numpy(), b.numpy())
    assert np.array_equal(layer.forward_saved(x, 3)[0].numpy(), layer.forward_saved(x, "silu")[0].numpy())
    for bad in ("tanh", 5):
        with pytest.raises(RuntimeError, match="unknown"):
            layer.forward_saved(x, bad)


def test_sequential_of_bfloat16_rows(cd):
    """LinearFp8 takes the activation behind it into its epilogue whatever the type of x."""
    rng = np.random.default_rng(6)
    x = cd.Tensor.from_numpy(rng.standard_normal((33, 96)).astype(np.float32)).to(cd.DType.bfloat16)
    a, b = cd.nn.LinearFp8(96, 160), cd.nn.LinearFp8(160, 40)
    y = cd.nn.Sequential(a, cd.nn.SiLU(), b)(x)
    assert y.dtype() == cd.DType.bfloat16
    assert np.array_equal(y.numpy(), b(a(x, "silu")).numpy())


def test_layers_on_a_stream_of_their_own(cd):
    """The first use of a weight, its replacement and the gradients on another stream than the parameter's, while the
    parameter's stream is busy: as on one stream, bit for bit."""
    rng = np.random.default_rng(5)
    m, n, k, groups = 260, 392, 520, 3
    x32 = rng.standard_normal((m, k)).astype(np.float32)
    dy32 = rng.standard_normal((m, n)).astype(np.float32)
    offsets = cd.Tensor.from_numpy(np.array([0, 100, 100, m], np.int32))
    weights = [(rng.standard_normal((n, k)) / 20).astype(np.float32) for _ in range(2)]
    experts = [(rng.standard_normal((groups, n, k)) / 20).astype(np.float32) for _ in range(2)]
    busy = cd.Tensor.ones([4096, 4096])

    def run(stream):
        linear, grouped, got = cd.nn.LinearFp8(k, n), cd.nn.GroupedLinear(groups, k, n), []
        for w, e in zip(weights, experts):
            linear.load_state_dict({"weight": w})
            grouped.load_state_dict({"weight": e})
            x = cd.Tensor.from_numpy(x32)
            dy = cd.Tensor.from_numpy(dy32)
            if stream is not None:
                x.set_stream(stream)
                dy.set_stream(stream)
                for _ in range(4):
                    busy.matmul(busy)
            x16, dy16 = x.to(cd.DType.bfloat16), dy.to(cd.DType.bfloat16)
            y, saved = linear.forward_saved(x, "gelu")
            out = [y, *linear.backward(dy16, saved), grouped(x16, offsets), *grouped.backward(dy16, x16, offsets)]
            linear.refresh()
            grouped.refresh()
            got.append([t.numpy() for t in out])
        return got

    for a, b in zip(run(None), run(cd.Stream())):
        assert all(np.array_equal(p, q) for p, q in zip(a, b))


# ---- streams, graphs, repeats ----------------------------------------------------------------------------------------------


def step_buffers(dev, m, n, k, groups, seed):
    torch = dev.torch
    gen = torch.Generator(device=dev.dev).manual_seed(seed)
    cuts = torch.sort(torch.randint(0, m + 1, (groups - 1,), generator=gen, device=dev.dev)).values
    b = {"x": torch.randn(m, k, generator=gen, device=dev.dev).bfloat16(),
         "w": (torch.randn(groups, n, k, generator=gen, device=dev.dev) / k ** 0.5).bfloat16(),
         "dy": torch.randn(m, n, generator=gen, device=dev.dev).bfloat16(),
         "off": torch.cat([torch.zeros(1, device=dev.dev), cuts, torch.full((1,), m, device=dev.dev)]).to(torch.int32)}
    return b


def outputs(dev, m, n, k, groups):
    torch = dev.torch
    e = lambda *s, t=torch.float32: torch.zeros(*s, dtype=t, device=dev.dev)      # noqa: E731
    return {"x8": e(m, k, t=torch.uint8), "xs": e(-(-k // 128), m), "w8": e(n, k, t=torch.uint8),
            "ws": e(-(-n // 128), -(-k // 128)), "z": e(m, n, t=torch.bfloat16), "z8": e(m, n, t=torch.uint8),
            "zs": e(-(-n // 128), m), "dx": e(m, k, t=torch.bfloat16), "dw": e(n, k), "db": e(n),
            "y": e(m, n, t=torch.bfloat16), "gdx": e(m, k, t=torch.bfloat16), "gdw": e(groups, n, k)}


def step(dev, b, o, m, n, k, groups, stream):
    """Quantise, 8-bit product, its backward pass, and the grouped products, one after the other."""
    lib, p = dev.lib, dev.ptr
    w0 = b["w"][0].contiguous() if groups == 1 else b["w"][0]
    for rc in (
        lib.cudeep_b200_quantize_fp8(p(b["x"]), 2, m, k, 1, p(o["x8"]), p(o["xs"]), stream),
        lib.cudeep_b200_quantize_fp8(p(w0), 2, n, k, 128, p(o["w8"]), p(o["ws"]), stream),
        lib.cudeep_b200_linear_forward_fp8(p(o["x8"]), p(o["xs"]), p(o["w8"]), p(o["ws"]), None, p(o["z"]), 2, m, n, k, 0,
                                           stream),
        lib.cudeep_b200_quantize_fp8(p(o["z"]), 2, m, n, 1, p(o["z8"]), p(o["zs"]), stream),
        lib.cudeep_b200_linear_backward_saved_fp8(p(b["dy"]), 2, p(o["x8"]), p(o["xs"]), p(o["z8"]), p(o["zs"]), 3, p(w0),
                                                  p(o["dx"]), p(o["dw"]), 0, p(o["db"]), m, n, k, stream),
        lib.cudeep_b200_grouped_matmul_nt(p(b["x"]), p(b["w"]), p(o["y"]), 2, p(b["off"]), groups, m, n, k, stream),
        lib.cudeep_b200_grouped_matmul_nn(p(b["dy"]), p(b["w"]), p(o["gdx"]), 2, p(b["off"]), groups, m, k, n, stream),
        lib.cudeep_b200_grouped_matmul_tn(p(b["dy"]), p(b["x"]), p(o["gdw"]), 2, 0, p(b["off"]), groups, m, n, k, stream),
    ):
        dev.check(rc)


def assert_same(dev, a, b):
    for key in a:
        assert dev.torch.equal(a[key], b[key]), key


SHAPE = (1000, 200, 333, 6)      # odd row lengths: every operand goes through a padded temporary


def test_repeats_are_bitwise_equal_and_streams_do_not_mix(dev):
    torch = dev.torch
    b = [step_buffers(dev, *SHAPE, seed) for seed in (1, 2)]
    want = [outputs(dev, *SHAPE) for _ in range(2)]
    for i in range(2):
        step(dev, b[i], want[i], *SHAPE, None)
    assert dev.sync_status() == 0
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[outputs(dev, *SHAPE) for _ in range(3)] for _ in range(2)]
    torch.cuda.synchronize()
    for r in range(3):
        for i in range(2):
            step(dev, b[i], got[i][r], *SHAPE, ctypes.c_void_p(streams[i].cuda_stream))
    assert dev.sync_status() == 0
    for i in range(2):
        for r in range(3):
            assert_same(dev, got[i][r], want[i])


def test_captured_graphs_replay_on_new_values(dev):
    """Two graphs whose temporaries come from the same pool, replayed in turn and side by side, on inputs and group sizes that
    changed after the capture."""
    torch = dev.torch
    b = [step_buffers(dev, *SHAPE, seed) for seed in (3, 4)]
    o = [outputs(dev, *SHAPE) for _ in range(2)]
    graphs = []
    for i in range(2):
        step(dev, b[i], o[i], *SHAPE, None)      # kernels are loaded before the capture
    torch.cuda.synchronize()
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            step(dev, b[i], o[i], *SHAPE, ctypes.c_void_p(torch.cuda.current_stream().cuda_stream))
        graphs.append(g)
    want = []
    for i in range(2):
        fresh = step_buffers(dev, *SHAPE, 10 + i)
        want.append(outputs(dev, *SHAPE))
        step(dev, fresh, want[i], *SHAPE, None)
        for key in b[i]:
            b[i][key].copy_(fresh[key])
    torch.cuda.synchronize()
    for _ in range(2):
        for i in range(2):
            graphs[i].replay()
    torch.cuda.synchronize()
    for i in range(2):
        assert_same(dev, o[i], want[i])
        for key in o[i]:
            o[i][key].zero_()
    torch.cuda.synchronize()
    side = [torch.cuda.Stream() for _ in range(2)]
    for i in range(2):
        with torch.cuda.stream(side[i]):
            graphs[i].replay()
    assert dev.sync_status() == 0
    for i in range(2):
        assert_same(dev, o[i], want[i])


# ---- edges ------------------------------------------------------------------------------------------------------------------


def test_bad_offsets_are_reported_and_stay_inside(dev):
    """Offsets that decrease or leave the rows: unspecified rows of the result, nothing outside it, status 6."""
    torch = dev.torch
    m, n, k, groups = 64, 128, 128, 3
    b = step_buffers(dev, m, n, k, groups, 5)
    guard = torch.full((m + 64, n), 7.0, dtype=torch.bfloat16, device=dev.dev)
    y = guard[32:32 + m]
    b["off"].copy_(torch.tensor([-5, 50, 20, 900], dtype=torch.int32))
    dev.check(dev.lib.cudeep_b200_grouped_matmul_nt(dev.ptr(b["x"]), dev.ptr(b["w"]), dev.ptr(y), 2, dev.ptr(b["off"]), groups,
                                                    m, n, k, None))
    assert dev.sync_status() == 6
    assert bool((guard[:32] == 7).all()) and bool((guard[32 + m:] == 7).all())
    dw = torch.full((groups + 2, n, k), 7.0, device=dev.dev)
    dev.check(dev.lib.cudeep_b200_grouped_matmul_tn(dev.ptr(b["dy"]), dev.ptr(b["x"]), dev.ptr(dw[1:]), 2, 0,
                                                    dev.ptr(b["off"]), groups, m, n, k, None))
    assert dev.sync_status() == 6
    assert bool((dw[0] == 7).all()) and bool((dw[-1] == 7).all())


def test_all_groups_empty_and_no_rows(dev):
    torch = dev.torch
    m, n, k, groups = 32, 64, 64, 1024
    off = torch.full((groups + 1,), 9, dtype=torch.int32, device=dev.dev)
    x, dy = (torch.full((m, d), float("nan"), dtype=torch.bfloat16, device=dev.dev) for d in (k, n))
    w = torch.randn(groups, n, k, device=dev.dev).bfloat16()
    y = torch.full((m, n), 7.0, dtype=torch.bfloat16, device=dev.dev)
    dw = torch.full((groups, n, k), 7.0, dtype=torch.bfloat16, device=dev.dev)
    dev.check(dev.lib.cudeep_b200_grouped_matmul_nt(dev.ptr(x), dev.ptr(w), dev.ptr(y), 2, dev.ptr(off), groups, m, n, k, None))
    dev.check(dev.lib.cudeep_b200_grouped_matmul_tn(dev.ptr(dy), dev.ptr(x), dev.ptr(dw), 2, 2, dev.ptr(off), groups, m, n, k,
                                                    None))
    assert dev.sync_status() == 0
    assert bool((y == 7).all()) and bool((dw == 0).all())
    dw.fill_(7.0)
    db = torch.full((n,), 7.0, device=dev.dev)
    dev.check(dev.lib.cudeep_b200_grouped_matmul_tn(dev.ptr(dy), dev.ptr(x), dev.ptr(dw), 2, 2, dev.ptr(off), groups, 0, n, k,
                                                    None))
    dev.check(dev.lib.cudeep_b200_linear_backward_saved_fp8(dev.ptr(dy), 2, dev.ptr(x), dev.ptr(db), None, None, 0, dev.ptr(w),
                                                            dev.ptr(y), dev.ptr(dw[1:]), 2, dev.ptr(db), 0, n, k, None))
    assert dev.sync_status() == 0
    assert bool((dw == 0).all()) and bool((db == 0).all()) and bool((y == 7).all())


@pytest.mark.parametrize("lead", [0, 1, 3])
def test_unaligned_bases(dev, lead):
    """Every operand and result starting `lead` elements into a buffer, with values around the results that stay."""
    torch = dev.torch
    m, n, k = 70, 136, 144

    def inside(t):
        buf = torch.full((t.numel() + lead + 8,), 7, dtype=t.dtype, device=dev.dev)
        buf[lead:lead + t.numel()] = t.reshape(-1)
        return buf, buf[lead:lead + t.numel()].view(t.shape)

    gen = torch.Generator(device=dev.dev).manual_seed(6)
    x, w = torch.randn(m, k, generator=gen, device=dev.dev).bfloat16(), torch.randn(2, n, k, generator=gen, device=dev.dev).bfloat16()
    dy = torch.randn(m, n, generator=gen, device=dev.dev).bfloat16()
    off = torch.tensor([0, 30, m], dtype=torch.int32, device=dev.dev)
    q = torch.randint(0, 120, (m, k), generator=gen, device=dev.dev, dtype=torch.int32).to(torch.uint8)
    wq = torch.randint(0, 120, (n, k), generator=gen, device=dev.dev, dtype=torch.int32).to(torch.uint8)
    xs, ws = torch.full((2, m), 0.125, device=dev.dev), torch.full((2, 2), 0.25, device=dev.dev)
    results = []
    for move in (lambda t: (None, t), inside):
        xv, wv, dv, qv, wqv = (move(t)[1] for t in (x, w, dy, q, wq))
        outs = [move(torch.zeros(s, dtype=t, device=dev.dev)) for s, t in
                (((m, n), torch.bfloat16), ((m, k), torch.bfloat16), ((2, n, k), torch.float32), ((m, n), torch.float32),
                 ((m, n), torch.bfloat16))]
        y, dx, dw, l32, l16 = (o[1] for o in outs)
        lib, p = dev.lib, dev.ptr
        dev.check(lib.cudeep_b200_grouped_matmul_nt(p(xv), p(wv), p(y), 2, p(off), 2, m, n, k, None))
        dev.check(lib.cudeep_b200_grouped_matmul_nn(p(dv), p(wv), p(dx), 2, p(off), 2, m, k, n, None))
        dev.check(lib.cudeep_b200_grouped_matmul_tn(p(dv), p(xv), p(dw), 2, 0, p(off), 2, m, n, k, None))
        dev.check(lib.cudeep_b200_linear_forward_fp8(p(qv), p(xs), p(wqv), p(ws), None, p(l32), 0, m, n, k, 0, None))
        dev.check(lib.cudeep_b200_linear_forward_fp8(p(qv), p(xs), p(wqv), p(ws), None, p(l16), 2, m, n, k, 0, None))
        assert dev.sync_status() == 0
        for buf, o in outs:
            if buf is not None:
                assert bool((buf[:lead] == 7).all()) and bool((buf[lead + o.numel():] == 7).all())
        results.append([o[1].clone() for o in outs])
    for a, b in zip(*results):
        assert torch.equal(a, b)


def test_offsets_beyond_32_bits(dev):
    """Matrices of more than 2^31 elements: their last rows are those of the same rows alone."""
    torch = dev.torch
    m, n, k = 66000, 33024, 256
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("needs 24 GB")
    gen = torch.Generator(device=dev.dev).manual_seed(7)
    x8 = torch.randint(0, 120, (m, k), generator=gen, device=dev.dev, dtype=torch.int32).to(torch.uint8)
    w8 = torch.randint(0, 120, (n, k), generator=gen, device=dev.dev, dtype=torch.int32).to(torch.uint8)
    xs, ws = torch.full((2, m), 0.125, device=dev.dev), torch.full((-(-n // 128), 2), 0.25, device=dev.dev)
    y = torch.empty(m, n, dtype=torch.bfloat16, device=dev.dev)
    lib, p = dev.lib, dev.ptr
    dev.check(lib.cudeep_b200_linear_forward_fp8(p(x8), p(xs), p(w8), p(ws), None, p(y), 2, m, n, k, 0, None))
    last = torch.empty(300, n, dtype=torch.bfloat16, device=dev.dev)
    tail, tail_s = x8[-300:].contiguous(), xs[:, -300:].contiguous()
    dev.check(lib.cudeep_b200_linear_forward_fp8(p(tail), p(tail_s), p(w8), p(ws), None, p(last), 2, 300, n, k, 0, None))
    assert dev.sync_status() == 0
    # The large product and the small one sum in different orders.  All terms are positive, so each FP32 sum is within
    # (128 + 2) * 2^-23 = 2^-15.9 of the exact value, far below bfloat16's half step: the two roundings of values that near can
    # only be equal or neighbours, 2^-7 of the value apart.
    assert ((y[-300:].double() - last.double()).abs() <= 2.0 ** -7 * last.double()).all()
    last = y[-300:].clone()
    q = torch.empty(m, n, dtype=torch.uint8, device=dev.dev)
    s = torch.empty(-(-n // 128), m, device=dev.dev)
    dev.check(lib.cudeep_b200_quantize_fp8(p(y), 2, m, n, 1, p(q), p(s), None))
    q1, s1 = torch.empty(300, n, dtype=torch.uint8, device=dev.dev), torch.empty(-(-n // 128), 300, device=dev.dev)
    dev.check(lib.cudeep_b200_quantize_fp8(p(last), 2, 300, n, 1, p(q1), p(s1), None))
    assert dev.sync_status() == 0
    assert torch.equal(q[-300:], q1) and torch.equal(s[:, -300:], s1)
    # One group at the very end of the rows, and its gradients.
    off = torch.tensor([m - 300, m], dtype=torch.int32, device=dev.dev)
    small = torch.randn(128, n, generator=gen, device=dev.dev).bfloat16()      # [features, n]
    out = torch.zeros(m, 128, dtype=torch.bfloat16, device=dev.dev)
    dev.check(lib.cudeep_b200_grouped_matmul_nt(p(y), p(small), p(out), 2, p(off), 1, m, 128, n, None))
    dy = torch.randn(m, 128, generator=gen, device=dev.dev).bfloat16()
    dw = torch.empty(128, n, device=dev.dev)
    dev.check(lib.cudeep_b200_grouped_matmul_tn(p(dy), p(y), p(dw), 2, 0, p(off), 1, m, 128, n, None))
    assert dev.sync_status() == 0
    want = last.double() @ small.double().t()
    assert (out[-300:].double() - want).norm() <= 2.0 ** -8 * want.norm() and bool((out[:-300] == 0).all())
    want = dy[-300:].double().t() @ last.double()
    assert (dw.double() - want).norm() <= 1e-5 * want.norm()


def test_gradients_asked_for_one_by_one(dev):
    torch = dev.torch
    m, n, k = 150, 72, 200
    gen = torch.Generator(device=dev.dev).manual_seed(9)
    dy, w = torch.randn(m, n, generator=gen, device=dev.dev).bfloat16(), torch.randn(n, k, generator=gen, device=dev.dev).bfloat16()
    x8, z8 = (torch.randint(0, 120, (m, d), generator=gen, device=dev.dev, dtype=torch.int32).to(torch.uint8) for d in (k, n))
    xs, zs = torch.full((2, m), 0.125, device=dev.dev), torch.full((1, m), 0.02, device=dev.dev)
    lib, p = dev.lib, dev.ptr
    for act in (0, 3):
        z = (p(z8), p(zs)) if act else (None, None)
        make = lambda: [torch.full(s, 7.0, dtype=t, device=dev.dev) for s, t in      # noqa: E731
                        (((m, k), torch.bfloat16), ((n, k), torch.bfloat16), ((n,), torch.float32))]
        whole = make()
        dev.check(lib.cudeep_b200_linear_backward_saved_fp8(p(dy), 2, p(x8), p(xs), *z, act, p(w), p(whole[0]), p(whole[1]), 2,
                                                            p(whole[2]), m, n, k, None))
        for i in range(3):
            part = make()
            dx, dw, db = (p(part[j]) if j == i else None for j in range(3))
            dev.check(lib.cudeep_b200_linear_backward_saved_fp8(
                p(dy), 2, p(x8) if dw else None, p(xs) if dw else None, *z, act, p(w) if dx else None, dx, dw, 2, db, m, n, k,
                None))
            assert dev.sync_status() == 0
            for j in range(3):
                assert torch.equal(part[j], whole[j]) if j == i else bool((part[j] == 7).all())


def test_many_rows(dev):
    """More rows than a grid's second dimension holds bands."""
    torch = dev.torch
    m, n = 5_000_001, 64
    x = torch.randn(m, n, device=dev.dev).bfloat16()
    lib, p = dev.lib, dev.ptr
    for block_rows in (1, 128):
        q, s = torch.empty(m, n, dtype=torch.uint8, device=dev.dev), torch.empty(m if block_rows == 1 else -(-m // 128), device=dev.dev)
        dev.check(lib.cudeep_b200_quantize_fp8(p(x), 2, m, n, block_rows, p(q), p(s), None))
        part = x[-129:].contiguous()      # the last block of 128 rows begins at a multiple of 128: 5000001 = 39062 * 128 + 65
        if block_rows == 128:
            part = x[-65:].contiguous()
        r = part.shape[0]
        q1, s1 = torch.empty(r, n, dtype=torch.uint8, device=dev.dev), torch.empty(r if block_rows == 1 else 1, device=dev.dev)
        dev.check(lib.cudeep_b200_quantize_fp8(p(part), 2, r, n, block_rows, p(q1), p(s1), None))
        assert dev.sync_status() == 0
        assert torch.equal(q[-r:], q1) and torch.equal(s[-s1.numel():], s1)
    z8, zs = torch.full((m, n), 0x38, dtype=torch.uint8, device=dev.dev), torch.ones(m, device=dev.dev)
    db = torch.empty(n, device=dev.dev)
    dev.check(lib.cudeep_b200_linear_backward_saved_fp8(p(x), 2, None, None, p(z8), p(zs), 1, None, None, None, 2, p(db), m, n, 8,
                                                        None))
    assert dev.sync_status() == 0
    want = x.double().sum(0)
    # FP32 sums of 5e6 terms in bands: each band and the sum of the bands may lose 2^-24 of the magnitudes per addition.
    assert ((db.double() - want).abs() <= (300 + 80000 / 8) * 2.0 ** -24 * x.double().abs().sum(0)).all()


def test_nan_codes_and_infinities(dev):
    """A NaN in one row or group shows in that row or group and nowhere else."""
    torch = dev.torch
    m, n, k = 300, 256, 256
    gen = torch.Generator(device=dev.dev).manual_seed(8)
    x = torch.randn(m, k, generator=gen, device=dev.dev)
    x[7, 3], x[150, 200] = float("inf"), float("nan")
    w = torch.randn(n, k, generator=gen, device=dev.dev)
    lib, p = dev.lib, dev.ptr
    for rows in (300, 100):
        xr = x[:rows].contiguous()
        x8, xs = torch.empty(rows, k, dtype=torch.uint8, device=dev.dev), torch.empty(2, rows, device=dev.dev)
        w8, ws = torch.empty(n, k, dtype=torch.uint8, device=dev.dev), torch.empty(2, 2, device=dev.dev)
        dev.check(lib.cudeep_b200_quantize_fp8(p(xr), 0, rows, k, 1, p(x8), p(xs), None))
        dev.check(lib.cudeep_b200_quantize_fp8(p(w), 0, n, k, 128, p(w8), p(ws), None))
        for act in range(5):
            y = torch.zeros(rows, n, device=dev.dev)
            dev.check(lib.cudeep_b200_linear_forward_fp8(p(x8), p(xs), p(w8), p(ws), None, p(y), 0, rows, n, k, act, None))
            bad = y.isnan().any(1).nonzero().flatten().tolist()
            assert bad == ([] if act == 1 else [r for r in (7, 150) if r < rows])      # the epilogue's ReLU drops NaN
    assert dev.sync_status() == 0
