"""Activations and their slopes far from zero, against the same formulas in 64 bits."""
import pytest

pytestmark = pytest.mark.gpu

CODES = {"f32": 0, "f16": 1, "bf16": 2}
ACTS = {"gelu": 2, "silu": 3, "sigmoid": 4}


def exponent64(torch, z, act):
    """t of sigmoid(t), and its slope."""
    if act != "gelu":
        return z, torch.ones_like(z)
    c = 2 * (2 / torch.pi) ** 0.5
    return c * (z + 0.044715 * z ** 3), c * (1 + 3 * 0.044715 * z * z)


def relative_bound(torch, t):
    """sigmoid(t) in FP32: the exponent u = t log2(e) carries up to six relative roundings (its coefficients and its products)
    of 2^-24, which are ln2 |u| as much of the result, 4.2 |u| 2^-24 in all; ex2.approx and rcp.approx add 2^-22 and 2^-23 and
    the products around them a rounding each: 16 * 2^-24 covers those."""
    return (4.2 * t.abs() * 1.4427 + 16) * 2.0 ** -24


def planted(dev, m, n, k, scale):
    """Operands whose product is x[r] * w[f] * scale exactly: one column holds them, the others are zero."""
    torch = dev.torch
    x8 = torch.zeros(m, k, dtype=torch.uint8, device=dev.dev)
    w8 = torch.zeros(n, k, dtype=torch.uint8, device=dev.dev)
    x8[:, 3] = 0x38 + (torch.arange(m, device=dev.dev) % 8).to(torch.uint8)              # 1 to 1.875
    w8[:, 3] = 0x30 + (torch.arange(n, device=dev.dev) % 40).to(torch.uint8) + 128       # -0.5 to -15
    w8[::16, 3] -= 128
    xs = torch.ones(-(-k // 128), m, device=dev.dev)
    ws = torch.full((-(-n // 128), -(-k // 128)), scale, device=dev.dev)
    value = lambda q: q[:, 3].contiguous().view(torch.float8_e4m3fn).double()      # noqa: E731
    return x8, xs, w8, ws, value(x8)[:, None] * value(w8)[None] * scale


SHAPES = [(5, 320, 128), (16, 1000, 4096), (300, 520, 256), (1100, 4096, 512), (4096, 4096, 2048)]


@pytest.mark.parametrize("out", ["f32", "bf16"])
@pytest.mark.parametrize("act", sorted(ACTS))
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_activations_far_below_zero(dev, act, m, n, k, out):
    """Right relative to themselves as long as sigmoid is a normal FP32 number, 2^-126 at least; where it is less, at most that
    times z."""
    torch = dev.torch
    x8, xs, w8, ws, z = planted(dev, m, n, k, 0.5 if act == "gelu" else 8.0)
    y = torch.full((m, n), float("nan"), device=dev.dev, dtype=torch.float32 if out == "f32" else torch.bfloat16)
    dev.check(dev.lib.cudeep_b200_linear_forward_fp8(dev.ptr(x8), dev.ptr(xs), dev.ptr(w8), dev.ptr(ws), None, dev.ptr(y),
                                                     CODES[out], m, n, k, ACTS[act], None))
    assert dev.sync_status() == 0
    t, _ = exponent64(torch, z, act)
    s = torch.sigmoid(t)
    want = s if act == "sigmoid" else z * s
    normal = s >= 2.0 ** -126 * 1.001
    assert bool((z < -20).any() if act != "gelu" else (z < -8).any()) and bool((~normal).any()) and bool((z > 1).any())
    rel = relative_bound(torch, t)
    if out == "bf16":
        rel = rel + torch.finfo(torch.bfloat16).eps / 2
    err = (y.double() - want).abs()
    assert not y.isnan().any()
    assert (err[normal] <= (rel * want.abs())[normal]).all()
    assert (y.double().abs()[~normal] <= (z.abs().clamp(min=1) * 2.0 ** -126 * 1.01)[~normal]).all()


@pytest.mark.parametrize("act", sorted(ACTS))
def test_slopes_far_from_zero(dev, act):
    """db of a single row is the slope itself: s + z s (1 - s) dt/dz (sigmoid: s (1 - s)), each term as far off as s is, the
    second with two roundings and an s more."""
    torch = dev.torch
    n = 4096
    codes = torch.arange(256, device=dev.dev).repeat(n // 256)
    z8 = torch.where(codes % 128 == 127, codes - 1, codes).to(torch.uint8).reshape(1, n).contiguous()
    zs = torch.exp2(torch.arange(n // 128, device=dev.dev).float() % 12 - 9).reshape(n // 128, 1).contiguous()
    z = z8.view(torch.float8_e4m3fn).double() * zs.double().repeat_interleave(128)[None]
    dy = torch.ones(1, n, dtype=torch.bfloat16, device=dev.dev)
    db = torch.full((n,), float("nan"), device=dev.dev)
    dev.check(dev.lib.cudeep_b200_linear_backward_saved_fp8(dev.ptr(dy), 2, None, None, dev.ptr(z8), dev.ptr(zs), ACTS[act], None,
                                                            None, None, 2, dev.ptr(db), 1, n, 8, None))
    assert dev.sync_status() == 0
    t, dt = exponent64(torch, z, act)
    s, rest = torch.sigmoid(t), torch.sigmoid(-t)
    first, second = (0 * z, s * rest) if act == "sigmoid" else (s, z * s * rest * dt)
    least = torch.minimum(s, rest) if act == "sigmoid" else s
    normal = least >= 2.0 ** -126 * 1.001
    assert bool((z < -50).any()) and bool((~normal).any())
    err = (db[None].double() - (first + second)).abs()
    bound = 2 * relative_bound(torch, t) * (first.abs() + second.abs())
    # sigmoid's complement below the least normal number may be off by that much, and so the terms it multiplies.
    bound = bound + (z.abs() * dt).clamp(min=1) * (rest < 2.0 ** -126 * 1.001) * 2.0 ** -126 * 1.01
    assert not db.isnan().any()
    assert (err[normal] <= bound[normal]).all()
    tail = ((z.abs() * dt + 1) * 2.0 ** -126 * 1.01)
    assert (db[None].double().abs()[~normal] <= tail[~normal]).all()
