"""8-bit integers: storage, linear layers, gated MLPs and expert layers against plain implementations in 64 bits.

Tolerances.  The integers of a row and the products' sums are exact, so a linear layer differs from scale·scale·sum + bias by fp32
roundings alone: the two scales', the sum's, two multiplications' and an addition's are at most 8 2^-24 of the terms' magnitudes,
and by the output's, u |y| + s (u half a unit in the last place, s half the smallest subnormal).

A gated MLP's hidden states are off by what g and u are, carried through the activation (slope at most 1.13, value within 2e-6),
ahead of their rounding to the output's type.  That puts every one of them between two 16-bit numbers, its row's largest magnitude
between two others, and its integer between the two that these give: what follows is held to the two ends.

The 2-norm is held too.  An output's rounding is at most u / sqrt(3) of it: 0.6 u.  Hidden states that are off by d = 2^-21 of their size
(an exponential and a reciprocal of one unit each, a few products) cross a border of their 16-bit type, ulp apart, with probability
2 d / ulp, and that moves their integer by a step with probability ulp / step: a mean square of 2 d step, in units of the hidden
states' own.  A step is at most 0.16 of their root mean square (a largest one of 20 times that), so this is 4e-4 of the norm.  It is
a mean, held where there are thousands of hidden states.
"""

import ctypes
import math

import pytest
import torch

from test_experts import ACT, HALF, SUB, U, device, gen, normal, route64
from triton_gated_mlp import FusedGatedMLP, GatedMoE, Q8GatedMLP, _cabi
from triton_gated_mlp.ops import moe, quant

gpu = pytest.mark.gpu
F = 2.0**-24


# ------------------------------------------------------------------ plain implementations
def integers64(v):
    """(n, scale) of rows [..., cols] in float64; the scale as it is rounded to fp32."""
    v = v.double()
    top = v.abs().amax(-1, keepdim=True)
    n = (127.0 * v / torch.where(top > 0, top, 1.0)).round()
    return n, (top.float() / 127.0).double()


def numbers_of(q, where="cpu"):
    """The integers of a single Q8Weight as float64 [rows, cols], looked up one place at a time."""
    flat, blocks = q.codes.to(where).reshape(-1), q.codes.shape[-5]
    r, c = torch.arange(q.rows, device=where).unsqueeze(1), torch.arange(q.cols, device=where).unsqueeze(0)
    at = ((r // 16) * blocks + c // 128) * 2048 + (c % 128 // 64) * 1024 + (c % 64 // 16) * 256 + (r % 16) * 16 + c % 16
    return flat[at].double()


def weight_of(q):
    return numbers_of(q), q.scales.cpu().double().unsqueeze(0)


def sliced(q, e):
    return quant.Q8Weight(q.codes[e], q.scales[e], q.rows, q.cols)


def product64(x, w, b):
    """(y, bound) of a product ahead of its rounding to 16 bits."""
    n, s = integers64(x)
    y = (n @ w[0].T) * s * w[1]
    mass = y.abs()
    if b is not None:
        y, mass = y + b.double(), mass + b.double().abs()
    return y, 8 * F * mass


def hidden64(x, gate, bg, up, bu, act, dtype):
    """Hidden states of x's type: the likeliest, the lowest and the highest."""
    g, dg = product64(x, gate, bg)
    u, du = product64(x, up, bu)
    a = ACT[act](g)
    h = a * u
    d = (1.13 * dg + 2e-6 * (1 + a.abs())) * (u.abs() + du) + a.abs() * du + 2 * F * h.abs()
    return h.to(dtype), (h - d).to(dtype), (h + d).to(dtype)


def down64(h, down, b):
    """(y, bound) of what hidden states between two ends give."""
    mid, lo, hi = h
    y, off = product64(mid, down, b)
    n, s = integers64(mid)
    tops = torch.stack([lo.double().abs(), hi.double().abs()])
    low = torch.where(lo.double() * hi.double() <= 0, 0.0, tops.amin(0)).amax(-1, keepdim=True)
    high = tops.amax(0).amax(-1, keepdim=True)
    ends = []
    for v in (lo, hi):
        for top in (low, high):
            k = (127.0 * v.double() / torch.where(top > 0, top, 1.0)).round().clamp(-127, 127)
            ends.append((k * top / 127.0 - n * s).abs())
    reach = torch.stack(ends).amax(0)
    return y, off + (reach @ down[0].abs().T) * down[1]


def mlp64(x, gate, bg, up, bu, down, bd, act, dtype):
    return down64(hidden64(x, gate, bg, up, bu, act, dtype), down, bd)


def moe64(x, logits, k, normalize, act, dtype, weights):
    """weights(e) -> gate, up, down."""
    w, experts = route64(logits, k, normalize)
    y, bound, mass = (torch.zeros(x.shape, dtype=torch.float64) for _ in range(3))
    for e in sorted(set(experts.reshape(-1).tolist())):
        t, j = torch.nonzero((experts == e) & (w > 0), as_tuple=True)
        if len(t) == 0:
            continue
        gate, up, down = weights(e)
        out, off = mlp64(x[t], gate, None, up, None, down, None, act, dtype)
        y[t] += w[t, j, None] * out
        bound[t] += w[t, j, None] * (off + 1e-6 * out.abs())  # (a weight is within 1e-6 of its own)
        mass[t] += (w[t, j, None] * out).abs()
    return y, bound + (k + 2) * F * mass


def hold(got, y, bound, dtype, hidden=None):
    """hidden: how many hidden states there are in between, if any."""
    got = got.detach().double().cpu().reshape(y.shape)
    assert torch.isfinite(got).all()
    off, bound = (got - y).abs(), bound + U[dtype] * (y.abs() + bound) + SUB[dtype]
    assert (off <= bound).all(), f"off by {(off / bound).max().item():.3f} of the bound"
    if y.numel() >= 64 and y.norm() > 0 and (hidden is None or hidden >= 4096):
        rel = (off.norm() / y.norm()).item()
        assert rel <= 0.6 * U[dtype] + (0.0 if hidden is None else 4e-4), f"2-norm off by {rel / U[dtype]:.3f} u"


def q8(shape, dtype, g):
    return quant.quantize_q8(normal(shape, 0.02, dtype, g).to(device()))


def on(t):
    return None if t is None else t.to(device())


# ------------------------------------------------------------------ without a GPU
def test_expert_layers_refuse_more_token_rows_than_offsets_reach():
    lib = _cabi.lib()
    raw = ctypes.create_string_buffer(4096 + 64)
    a = (ctypes.addressof(raw) + 63) & ~63
    moe_fwd = lambda M, K: lib.gmlp_q8_moe_fwd(a, a, a, a, a, a, a, a, a, M, K, 8, 512, 1, 1, 0, 0, 0, a, 0, None)
    assert moe_fwd(16384, 131072) == -2 and "M * K" in lib.gmlp_last_error().decode()
    assert moe_fwd(16383, 131072) == -1 and "workspace" in lib.gmlp_last_error().decode()


def test_what_a_launch_has_threads_for_is_taken_and_no_more():
    lib = _cabi.lib()
    raw = ctypes.create_string_buffer(4096 + 64)
    a = (ctypes.addressof(raw) + 63) & ~63
    err = lambda: lib.gmlp_last_error().decode()
    linear = lambda M, C: lib.gmlp_q8_linear_fwd(a, a, a, None, a, M, 8, C, 0, a, 0, None)
    for M, C in ((65536, 262144), (65536, (1 << 21) - 64), (1, (1 << 27) - 16), (1 << 20, (1 << 17) - 64)):
        assert linear(M, C) == -1 and "workspace" in err()
    for M, C in ((65536, 1 << 21), (1, 1 << 27), (1 << 21, 1 << 16), (1 << 21, 1 << 18)):
        assert linear(M, C) == -2 and "too large" in err()
    mlp = lambda M, K, N: lib.gmlp_q8_mlp_fwd(a, a, a, a, a, a, a, None, None, None, a, M, K, N, 0, 0, a, 0, None)
    assert mlp(65536, 131072, 131072) == -1 and mlp(1 << 22, 131072, 64) == -2 and mlp(1 << 22, 64, 131072) == -2 and "too large" in err()
    moe_fwd = lambda M, K, N, E, k: lib.gmlp_q8_moe_fwd(a, a, a, a, a, a, a, a, a, M, K, N, E, k, 1, 0, 0, 0, a, 0, None)
    assert moe_fwd(65536, 8, 131072, 512, 1) == -1 and "workspace" in err()
    assert moe_fwd(1, 131072, 131072, 512, 16) == -1 and moe_fwd(384, 131072, 131072, 512, 16) == -1 and moe_fwd(1536, 131072, 131072, 512, 16) == -1


def test_refusals_of_the_c_interface():
    lib = _cabi.lib()
    raw = ctypes.create_string_buffer(4096 + 64)
    a = (ctypes.addressof(raw) + 63) & ~63
    err = lambda: lib.gmlp_last_error().decode()
    need = lib.gmlp_q8_linear_workspace_bytes(3, 64, 64, 0)
    assert need >= 16 * 128 and lib.gmlp_q8_linear_workspace_bytes(0, 64, 64, 0) == 0
    assert lib.gmlp_q8_linear_workspace_bytes(3, 64, 64, 2) == 0 and lib.gmlp_q8_linear_workspace_bytes(3, 1 << 18, 64, 0) == 0

    def linear(x=a, codes=a, scales=a, bias=None, y=a, M=3, R=64, C=64, dtype=0, ws=a, n=need):
        return lib.gmlp_q8_linear_fwd(x, codes, scales, bias, y, M, R, C, dtype, ws, n, None)

    assert linear(x=None) == -1 and "NULL" in err()
    assert linear(codes=None) == -1 and linear(scales=None) == -1 and linear(y=None) == -1 and linear(ws=None) == -1
    assert linear(dtype=2) == -2 and linear(dtype=7) == -1
    assert linear(M=0) == -2 and linear(R=60) == -2 and "multiple of 8" in err()
    assert linear(C=68) == -2 and linear(R=131080) == -2 and "32 bits" in err()
    assert linear(x=a + 8) == -3 and linear(bias=a + 2) == -3 and linear(scales=a + 4) == -3
    assert linear(n=need - 1) == -1 and "workspace" in err()
    assert linear(M=(1 << 23) + 1) == -2 and "2^23" in err()
    assert linear(M=1 << 23, C=1 << 20) == -2 and "too large" in err()

    need = lib.gmlp_q8_mlp_workspace_bytes(3, 64, 64, 1)

    def mlp(x=a, w=a, s=a, y=a, M=3, K=64, N=64, dtype=1, act=0, ws=a, n=need):
        return lib.gmlp_q8_mlp_fwd(x, w, s, w, s, w, s, None, None, None, y, M, K, N, dtype, act, ws, n, None)

    assert mlp(x=None) == -1 and mlp(w=None) == -1 and mlp(s=None) == -1 and mlp(y=None) == -1 and mlp(ws=None) == -1
    assert mlp(act=7) == -1 and "act" in err()
    assert mlp(dtype=2) == -2 and mlp(M=0) == -2 and mlp(K=4) == -2 and mlp(N=12) == -2 and mlp(N=131080) == -2 and mlp(n=0) == -1
    assert mlp(w=a + 8) == -3

    need = lib.gmlp_q8_moe_workspace_bytes(4, 64, 64, 8, 2, 0)
    assert lib.gmlp_q8_moe_workspace_bytes(40000, 64, 64, 8, 2, 0) == 0 and lib.gmlp_q8_moe_workspace_bytes(4, 64, 64, 8, 17, 0) == 0

    def layer(x=a, logits=a, w=a, s=a, y=a, M=4, K=64, N=64, E=8, k=2, dtype=0, ld=2, act=0, ws=a, n=need):
        return lib.gmlp_q8_moe_fwd(x, logits, w, w, w, s, s, s, y, M, K, N, E, k, 1, dtype, ld, act, ws, n, None)

    assert layer(x=None) == -1 and layer(logits=None) == -1 and layer(w=None) == -1 and layer(s=None) == -1 and layer(ws=None) == -1
    assert layer(M=0) == -2 and layer(M=32769) == -2 and "choices" in err()
    assert layer(k=9) == -2 and layer(k=0) == -2 and layer(E=513) == -2 and layer(K=60) == -2 and layer(N=4) == -2
    assert layer(dtype=2) == -2 and layer(ld=3) == -1 and layer(act=9) == -1 and layer(n=need - 1) == -1 and layer(x=a + 4) == -3

    for call in (lib.gmlp_q8_quantize, lib.gmlp_q8_dequantize):
        assert call(a, None, a, 1, 16, 128, 0, None) == -1
        assert call(a, a, a, 0, 16, 128, 0, None) == -2 and call(a, a, a, 1, 12, 128, 0, None) == -2
        assert call(a, a, a, 1, 16, 128, 2, None) == -2 and call(a, a, a, 1, 16, 131080, 0, None) == -2
        assert call(a, a, a, 65536, 16, 128, 0, None) == -2 and call(a, a, a, 1 << 40, 16, 128, 0, None) == -2
        assert call(a, a, a, 1, (1 << 23) + 1, 128, 0, None) == -2 and call(a, a, a, 1, 1 << 20, 1 << 17, 0, None) == -2
        assert call(a + 8, a, a, 1, 16, 128, 0, None) == -3


def cpu_weight(lead=(), rows=64, cols=64):
    return quant.Q8Weight(torch.zeros((*lead, rows // 16, -(-cols // 128), 2, 4, 16, 16), dtype=torch.int8), torch.zeros((*lead, rows)), rows, cols)


def test_cpu_tensors_transforms_and_gradients_are_refused():
    import torch.autograd.forward_ad as fw

    x, b, logits = torch.zeros(3, 64, dtype=torch.float16), torch.zeros(64, dtype=torch.float16), torch.zeros(3, 2)
    w, we = cpu_weight(), cpu_weight((2,))
    with_scales = lambda q, s: q._replace(scales=s)
    calls = [
        (lambda t: quant.quantize_q8(t), x), (lambda t: quant.dequantize_q8(with_scales(w, t), torch.float16), w.scales),
        (lambda t: quant.q8_linear_fwd(t, w), x), (lambda t: quant.q8_linear_fwd(x, w, t), b),
        (lambda t: quant.q8_linear_fwd(x, with_scales(w, t)), w.scales),
        (lambda t: quant.q8_mlp_fwd(t, w, None, w, None, w, None), x),
        *((lambda t, i=i: quant.q8_mlp_fwd(x, *(v for j in range(3) for v in (w, t if j == i else None))), b) for i in range(3)),
        *((lambda t, i=i: quant.q8_mlp_fwd(x, *(v for j in range(3) for v in (with_scales(w, t) if j == i else w, None))), w.scales)
          for i in range(3)),
        (lambda t: moe.moe_mlp_fwd(t, logits, we, we, we, 2), x), (lambda t: moe.moe_mlp_fwd(x, t, we, we, we, 2), logits),
        *((lambda t, i=i: moe.moe_mlp_fwd(x, logits, *(with_scales(we, t) if j == i else we for j in range(3)), 2), we.scales) for i in range(3)),
    ]
    for call, t in calls:
        with pytest.raises(RuntimeError, match="AMD GPU"):
            call(t)
        with fw.dual_level(), torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
            call(fw.make_dual(t, t))
        with pytest.raises(RuntimeError, match="functorch"):
            torch.vmap(call)(t[None])
        with pytest.raises(RuntimeError, match="no backward"):
            call(t.clone().requires_grad_(True))
    with pytest.raises(TypeError, match="all Q8Weight"):
        moe.moe_mlp_fwd(x, logits, we, we, torch.zeros(2, 64, 64, dtype=torch.float16), 2)
    with pytest.raises(ValueError, match="bits"):
        GatedMoE(64, 64, 2, 1).quantize_(bits=5)


# ------------------------------------------------------------------ storage
@gpu
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("shape", [(8, 8), (16, 128), (40, 200), (24, 9000), (3, 24, 328), (70, 40, 136)])
def test_quantize_and_dequantize(shape, dtype):
    w = normal(shape, 0.02, dtype, gen(1))
    w[..., 0, :] = 0
    w[..., 1, :] *= 1000
    w[..., 2, :] = (w[..., 2, :].float() * (2.0**120 if dtype == torch.bfloat16 else 2.0**14)).to(dtype)
    w[..., 3, :] = (w[..., 3, :].float() * (2.0**-125 if dtype == torch.bfloat16 else 2.0**-14)).to(dtype)
    w[..., 4, :] = torch.linspace(-1, 1, shape[-1]).to(dtype)  # halves among them
    q = quant.quantize_q8(w.to(device()))
    back = quant.dequantize_q8(q, dtype)
    assert back.shape == w.shape and back.dtype == dtype and q.codes.dtype == torch.int8 and q.scales.shape == shape[:-1]
    for e in [None] if w.dim() == 2 else range(0, shape[0], 23):
        dense, one, again = (w, q, back) if e is None else (w[e], sliced(q, e), back[e])
        n, s = integers64(dense)
        assert torch.equal(numbers_of(one), n)
        assert torch.equal(one.scales.cpu().double(), s[:, 0])
        assert torch.equal(again.cpu(), (n.float() * s.float()).to(dtype))
        full = quant.Q8Weight(one.codes, one.scales, one.codes.shape[0] * 16, one.codes.shape[1] * 128)
        everything = numbers_of(full)
        assert (everything[shape[-2] :] == 0).all() and (everything[:, shape[-1] :] == 0).all()


@gpu
@pytest.mark.parametrize("dtype,bits,unit", [(torch.float16, 11, 5), (torch.float16, 11, -15), (torch.bfloat16, 8, 113), (torch.bfloat16, 8, -7),
                                             (torch.bfloat16, 8, -67), (torch.bfloat16, 8, -117)])
def test_every_quotient_is_rounded_to_the_nearest(dtype, bits, unit):
    """A row for every mantissa b of the largest, b 2^unit, and in it every mantissa a of numbers a 2^(unit - k) up to it, for each gap k
    of exponents that leaves a quotient 127 a / (b 2^k) of a half or more; k = 9 leaves none.  In whole numbers."""
    some = torch.arange(1 << (bits - 1), 1 << bits, device=device())
    b = some[:, None]
    numbers, expected = [b], [torch.full_like(b, 127)]
    for k in range(10):
        a = some[None, :] * (some[None, :] <= b if k == 0 else torch.ones_like(b))
        sign = 1 - 2 * (some[None, :] + b + k & 1)
        whole, rest = 127 * a // (b << k), 127 * a % (b << k)
        up = (2 * rest > b << k) | ((2 * rest == b << k) & (whole % 2 == 1))
        numbers.append((sign * a).double() * 2.0**-k)
        expected.append(sign * (whole + up))
    numbers, expected = torch.cat([n.double() for n in numbers], 1), torch.cat(expected, 1)
    fill = -numbers.shape[1] % 8
    w = (torch.nn.functional.pad(numbers, (0, fill)) * 2.0**unit).to(dtype)
    assert torch.equal(w[:, : numbers.shape[1]].double(), numbers * 2.0**unit)
    got = numbers_of(quant.quantize_q8(w), w.device)
    assert torch.equal(got, torch.nn.functional.pad(expected, (0, fill)).double())
    assert (expected[:, -len(some) :] == 0).all() and expected[:, -2 * len(some) :].any()


# Every form in which rows become integers: by how many rows there are, and by their length (kept by the threads in 1, 2, 4 or 8 pieces, or read
# twice).
@gpu
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("cols", [264, 5000, 16392, 20488, 32768, 32776, 40008])
@pytest.mark.parametrize("shape", [(24,), (1032,), (3, 360)])
def test_dense_rows_of_every_length(shape, cols, dtype):
    w = normal((*shape, cols), 1.0, dtype, gen(cols))
    q = quant.quantize_q8(on(w))
    # (divided on the CPU: on the GPU torch multiplies by fl(1/127))
    assert torch.equal(q.scales.cpu(), w.abs().amax(-1).float() / 127.0)
    for e in [None] if len(shape) == 1 else range(shape[0]):
        n, _ = integers64(on(w if e is None else w[e]))
        assert torch.equal(numbers_of(q if e is None else sliced(q, e), n.device), n)


@gpu
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("M,R,C", [(1032, 20488, 40), (1032, 32768, 24), (1040, 33000, 24), (1009, 16392, 136)])
def test_q8_linear_of_many_long_rows(M, R, C, dtype):
    g = gen(M + R)
    x, q = normal((M, R), 1.0, dtype, g), q8((C, R), dtype, g)
    y = quant.q8_linear_fwd(on(x), q)
    n, s = integers64(on(x))
    ref = (n @ numbers_of(q, n.device).T) * s * q.scales.double()
    hold(y, ref.cpu(), 8 * F * ref.abs().cpu(), dtype)


@gpu
def test_rows_that_are_not_finite_are_nan_and_stand_alone():
    for dtype in HALF:
        w = normal((24, 136), 1.0, dtype, gen(3))
        w[5, 7], w[9, 135], w[17, 0] = math.inf, math.nan, -math.inf
        q = quant.quantize_q8(w.to(device()))
        bad = torch.zeros(24, dtype=torch.bool)
        bad[[5, 9, 17]] = True
        assert torch.equal(q.scales.cpu().isnan(), bad) and (numbers_of(q)[bad] == 0).all()
        assert torch.equal(numbers_of(q)[~bad], integers64(w[~bad])[0])
        for M in (8, 24, 300):
            x = normal((M, 264), 1.0, dtype, gen(4))
            x[2, 100], x[M - 2, 1], x[M - 5] = math.nan, math.inf, 0
            y = quant.q8_linear_fwd(x.to(device()), q8((40, 264), dtype, gen(5))).cpu()
            rows = torch.zeros(M, dtype=torch.bool)
            rows[[2, M - 2]] = True
            assert torch.equal(y.isnan().any(1), rows) and torch.equal(y.isnan().all(1), rows) and (y[M - 5] == 0).all()


# ------------------------------------------------------------------ linear layers
@gpu
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize(
    "M,R,C,bias",
    [
        (1, 8, 8, False), (1, 128, 16, True), (1, 2048, 2048, False), (2, 1160, 3096, True), (7, 264, 72, True), (1, 20000, 40, False),
        (1, 40000, 24, True), (2, 40000, 72, False), (16, 2048, 264, True), (12, 136, 16400, False), (3, 1160, 8200, True),
        (16, 4096, 40, False), (17, 1000, 136, False), (32, 136, 1000, True), (33, 520, 264, True), (64, 1032, 520, False),
        (65, 264, 392, True), (77, 1160, 3096, True), (130, 4096, 264, False), (300, 1160, 264, False), (515, 8200, 520, True),
        (1024, 392, 2056, True), (2100, 264, 4104, False), (257, 136, 8200, False),
    ],
)
def test_q8_linear(M, R, C, bias, dtype):
    g = gen(M + R)
    x, q = normal((M, R), 1.0, dtype, g), q8((C, R), dtype, g)
    b = normal((C,), 0.5, dtype, g) if bias else None
    y = quant.q8_linear_fwd(on(x), q, on(b))
    ref, bound = product64(x, weight_of(q), b)
    hold(y, ref, bound, dtype)


# A long batch goes in pieces of 65536 rows, which its rows do not see.
@gpu
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("more", [17, 300])
def test_rows_around_the_cut_of_a_long_batch(more, dtype):
    M, K, N = 65536 + more, 72, 40
    g = gen(more)
    x = on(normal((M, K), 1.0, dtype, g))
    w = [q8((N, K), dtype, g), q8((N, K), dtype, g), q8((K, N), dtype, g)]
    b = [normal((n,), 0.3, dtype, g) for n in (N, N, K)]
    rows = torch.tensor([0, 1, 127, 40000, 65534, 65535, 65536, 65537, M - 2, M - 1])
    y = quant.q8_linear_fwd(x, w[0], on(b[0]))
    ref, bound = product64(x[on(rows)].cpu(), weight_of(w[0]), b[0])
    hold(y[on(rows)], ref, bound, dtype)
    assert torch.equal(y[:65536], quant.q8_linear_fwd(x[:65536], w[0], on(b[0])))
    y = quant.q8_mlp_fwd(x, w[0], on(b[0]), w[1], on(b[1]), w[2], on(b[2]))
    ref, bound = mlp64(x[on(rows)].cpu(), weight_of(w[0]), b[0], weight_of(w[1]), b[1], weight_of(w[2]), b[2], "silu", dtype)
    hold(y[on(rows)], ref, bound, dtype, len(rows) * N)
    assert torch.equal(y[:65536], quant.q8_mlp_fwd(x[:65536], w[0], on(b[0]), w[1], on(b[1]), w[2], on(b[2])))


@gpu
@pytest.mark.parametrize("M,C", [(65536 + 17, 262144), (3000, (1 << 23) - 8)])
def test_a_long_batch_through_a_wide_weight(M, C):
    """A vocabulary projection, and the widest weight that can be quantised.  (34 and 50 GB of outputs.)"""
    dtype, K = torch.float16, 8
    g = gen(C % 1000)
    x, q = on(normal((M, K), 1.0, dtype, g)), quant.quantize_q8(torch.randn((C, K), device=device()).to(dtype))
    y = quant.q8_linear_fwd(x, q)
    rows = on(torch.tensor([0, 1, 127, 128, 2047, 2048, M - 1081, M - 18, M - 17, M - 1]))
    cols = on(torch.cat([torch.arange(32), torch.randint(0, C, (200,), generator=g), torch.arange(C - 32, C)]))
    n, s = integers64(x[rows])
    ref = (n @ numbers_of(q, x.device)[cols].T) * s * q.scales.double()[cols]
    hold(y[rows][:, cols], ref.cpu(), (8 * F * ref.abs()).cpu(), dtype)
    del y
    torch.cuda.empty_cache()


@gpu
@pytest.mark.parametrize("M", [1, 16, 100, 700])
def test_the_largest_sums(M):
    """127 in every place of the longest reduction: 32 bits hold it."""
    R, C = 131072, 16
    x, w = torch.ones(M, R, dtype=torch.bfloat16), torch.ones(C, R, dtype=torch.bfloat16)
    w[1::2] = -1
    y = quant.q8_linear_fwd(on(x), quant.quantize_q8(on(w))).cpu()
    sign = torch.tensor([1.0, -1.0]).repeat(C // 2)
    assert torch.equal(y.float(), (131072.0 * sign).expand(M, C))


@gpu
def test_leading_dimensions_strides_and_no_rows():
    dtype = torch.float16
    g = gen(8)
    x, q = normal((2, 3, 5, 272), 1.0, dtype, g), q8((48, 264), dtype, g)
    view = on(x)[..., 4:268]  # neither contiguous nor aligned
    y = quant.q8_linear_fwd(view, q)
    assert y.shape == (2, 3, 5, 48)
    ref, bound = product64(x[..., 4:268].reshape(30, 264), weight_of(q), None)
    hold(y, ref, bound, dtype)
    flat = torch.zeros(264 * 4 + 1, dtype=dtype, device=device())[1:].view(4, 264)  # contiguous, 2 bytes off
    flat.copy_(on(x)[0, 0, :4, :264])
    assert torch.equal(quant.q8_linear_fwd(flat, q), quant.q8_linear_fwd(flat.clone(), q))
    transposed = normal((264, 6), 1.0, dtype, g)
    assert torch.equal(quant.q8_linear_fwd(on(transposed).T, q), quant.q8_linear_fwd(on(transposed).T.contiguous(), q))
    assert quant.q8_linear_fwd(on(x)[:0, 0, 0, :264], q).shape == (0, 48)
    assert quant.q8_mlp_fwd(on(x)[:0, 0, 0, :264], q, None, q, None, q8((264, 48), dtype, g), None).shape == (0, 264)
    experts = [q8((2, 48, 264), dtype, g), q8((2, 48, 264), dtype, g), q8((2, 264, 48), dtype, g)]
    assert moe.moe_mlp_fwd(on(x)[:0, 0, 0, :264], torch.zeros(0, 2, device=device()), *experts, 1).shape == (0, 264)


@gpu
def test_refusals_of_tensors():
    dtype = torch.bfloat16
    x, q = torch.zeros(3, 264, dtype=dtype, device=device()), q8((48, 264), dtype, gen(9))
    for call, error in [
        (lambda: quant.q8_linear_fwd(x.float(), q), TypeError),
        (lambda: quant.q8_linear_fwd(x[:, :256], q), ValueError),
        (lambda: quant.q8_linear_fwd(x, q, torch.zeros(40, dtype=dtype, device=device())), ValueError),
        (lambda: quant.q8_linear_fwd(x, q, torch.zeros(48, dtype=torch.float16, device=device())), TypeError),
        (lambda: quant.q8_linear_fwd(x, q._replace(codes=q.codes.view(torch.uint8))), TypeError),
        (lambda: quant.q8_linear_fwd(x, q._replace(scales=q.scales.half())), TypeError),
        (lambda: quant.q8_linear_fwd(x, q._replace(scales=q.scales[:40])), ValueError),
        (lambda: quant.q8_linear_fwd(x, q._replace(scales=q.scales.cpu())), RuntimeError),
        (lambda: quant.q8_linear_fwd(x, q._replace(rows=40)), ValueError),
        (lambda: quant.q8_mlp_fwd(x, q, None, q, None, q, None), ValueError),
        (lambda: quant.q8_mlp_fwd(x, q, None, q, None, q8((264, 48), dtype, gen(9)), None, act_fn="nothing"), NotImplementedError),
        (lambda: quant.quantize_q8(x.float()), TypeError),
        (lambda: quant.quantize_q8(x[0]), ValueError),
        (lambda: quant.quantize_q8(x[:, :260]), NotImplementedError),
        (lambda: quant.dequantize_q8(q, torch.float32), TypeError),
    ]:
        with pytest.raises(error):
            call()


# ------------------------------------------------------------------ gated MLPs
@gpu
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize(
    "M,K,N,bias,act",
    [
        (1, 8, 16, True, "silu"), (1, 1160, 3096, False, "silu"), (3, 264, 520, True, "gelu"), (16, 2048, 392, False, "relu"),
        (20, 136, 1000, True, "tanh"), (48, 520, 264, False, "sigmoid"), (64, 264, 1032, True, "no_act"), (65, 520, 776, False, "leaky_relu"),
        (200, 264, 2056, True, "silu"), (300, 1032, 520, False, "gelu"), (1100, 392, 1160, True, "silu"), (2050, 136, 2056, False, "relu"),
    ],
)
def test_q8_mlp(M, K, N, bias, act, dtype):
    g = gen(M + K + N)
    x = normal((M, K), 1.0, dtype, g)
    w = [q8((N, K), dtype, g), q8((N, K), dtype, g), q8((K, N), dtype, g)]
    b = [normal((n,), 0.3, dtype, g) if bias else None for n in (N, N, K)]
    y = quant.q8_mlp_fwd(on(x), w[0], on(b[0]), w[1], on(b[1]), w[2], on(b[2]), act_fn=act)
    ref, bound = mlp64(x, weight_of(w[0]), b[0], weight_of(w[1]), b[1], weight_of(w[2]), b[2], act, dtype)
    hold(y, ref, bound, dtype, M * N)


# ------------------------------------------------------------------ expert layers
@gpu
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize(
    "M,K,N,E,k,act,normalize",
    [
        (1, 8, 8, 1, 1, "silu", True), (1, 1160, 520, 8, 2, "silu", True), (1, 264, 136, 64, 8, "gelu", False), (3, 136, 264, 60, 6, "relu", True),
        (16, 520, 392, 4, 2, "silu", False), (40, 264, 136, 5, 3, "silu", True), (96, 264, 136, 64, 8, "silu", True), (70, 136, 264, 3, 1, "tanh", True),
        (1, 264, 136, 20, 16, "silu", True), (1, 520, 264, 200, 9, "relu", False), (1, 136, 264, 300, 3, "silu", True), (1, 40008, 16, 3, 2, "silu", True),
        (2, 136, 264, 9, 9, "silu", True), (20, 264, 136, 100, 4, "silu", False), (10, 136, 264, 200, 3, "tanh", True), (7, 264, 136, 400, 5, "silu", True),
        (128, 136, 264, 16, 2, "silu", True), (129, 136, 264, 16, 2, "silu", False), (260, 264, 136, 1, 1, "gelu", True), (700, 136, 264, 9, 1, "silu", True),
        (300, 264, 392, 8, 2, "silu", False), (600, 136, 520, 16, 4, "gelu", True), (1500, 136, 264, 4, 2, "silu", True), (130, 264, 136, 512, 16, "silu", True),
    ],
)
def test_q8_moe(M, K, N, E, k, act, normalize, dtype):
    g = gen(M + K + N + E)
    x, logits = normal((M, K), 1.0, dtype, g), normal((M, E), 1.5, torch.float32, g)
    w = [q8((E, N, K), dtype, g), q8((E, N, K), dtype, g), q8((E, K, N), dtype, g)]
    y = moe.moe_mlp_fwd(on(x), on(logits), *w, k, normalize=normalize, act_fn=act)
    ref, bound = moe64(x, logits, k, normalize, act, dtype, lambda e: [weight_of(sliced(q, e)) for q in w])
    hold(y, ref, bound, dtype, M * N)


@gpu
@pytest.mark.parametrize("M,E,k", [(2, 4, 2), (50, 6, 3), (400, 3, 2), (400, 40, 1)])
def test_q8_moe_with_masked_experts_and_crowds(M, E, k):
    """Experts that a token cannot have, tokens that have none, experts without a token, and one that has them all."""
    dtype, K, N = torch.bfloat16, 136, 264
    g = gen(M + E)
    x, logits = normal((M, K), 1.0, dtype, g), normal((M, E), 1.0, torch.float32, g)
    logits[:, 0] += 20
    logits[:, E - 1] = -math.inf
    logits[1, 1:] = -math.inf  # fewer experts than choices
    logits[M - 1] = -math.inf
    w = [q8((E, N, K), dtype, g), q8((E, N, K), dtype, g), q8((E, K, N), dtype, g)]
    for q in w:
        q.scales[E - 1] = math.nan  # of an expert that nobody has
    y = moe.moe_mlp_fwd(on(x), on(logits), *w, k)
    assert (y[M - 1] == 0).all()
    ref, bound = moe64(x, logits, k, True, "silu", dtype, lambda e: [weight_of(sliced(q, e)) for q in w])
    hold(y, ref, bound, dtype, M * N)


# The way an expert layer runs is chosen by the rows an expert has on average; routers have popular experts.  Up to 12, 24 and 48 rows an
# expert and beyond, each with an expert that has many times as many and experts that have a few or none.
@gpu
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize(
    "M,K,N,E,k,act",
    [
        (40, 264, 520, 20, 2, "silu"), (100, 136, 264, 60, 6, "gelu"), (150, 264, 392, 16, 2, "silu"), (90, 4104, 2056, 8, 2, "relu"),
        (200, 264, 136, 12, 2, "silu"), (320, 136, 520, 64, 8, "tanh"), (700, 264, 520, 10, 2, "silu"), (1200, 520, 264, 32, 4, "gelu"),
    ],
)
def test_q8_moe_with_popular_experts(M, K, N, E, k, act, dtype):
    g = gen(M + E)
    x = normal((M, K), 1.0, dtype, g)
    logits = normal((M, E), 1.5, torch.float32, g) - torch.linspace(0, 9, E)[torch.randperm(E, generator=g)]
    rows = torch.bincount(route64(logits, k, True)[1].reshape(-1), minlength=E)
    assert rows.max() > 3 * M * k / E and rows.min() < M * k / E / 3
    w = [q8((E, N, K), dtype, g), q8((E, N, K), dtype, g), q8((E, K, N), dtype, g)]
    y = moe.moe_mlp_fwd(on(x), on(logits), *w, k, act_fn=act)
    ref, bound = moe64(x, logits, k, True, act, dtype, lambda e: [weight_of(sliced(q, e)) for q in w])
    hold(y, ref, bound, dtype, M * N)


@gpu
@pytest.mark.parametrize("E", [4, 70, 300])
def test_the_only_token_with_masked_experts(E):
    dtype, K, N, k = torch.float16, 136, 264, 3
    g = gen(E)
    x, logits = normal((1, K), 1.0, dtype, g), normal((1, E), 1.0, torch.float32, g)
    w = [q8((E, N, K), dtype, g), q8((E, N, K), dtype, g), q8((E, K, N), dtype, g)]
    logits[0, 2:] = -math.inf  # two experts for three choices
    y = moe.moe_mlp_fwd(on(x), on(logits), *w, k)
    ref, bound = moe64(x, logits, k, True, "silu", dtype, lambda e: [weight_of(sliced(q, e)) for q in w])
    hold(y, ref, bound, dtype, N)
    logits[:] = -math.inf
    assert (moe.moe_mlp_fwd(on(x), on(logits), *w, k) == 0).all()
    logits[0, 1], logits[0, 3] = 0.0, -200.0  # a weight that is 0: its expert is not run
    w[2].scales[3] = math.nan
    assert moe.moe_mlp_fwd(on(x), on(logits), *w, 2).isfinite().all()


# Shapes for every kernel that the rules choose: tiles of weight rows a workgroup, wavefronts and stages of the streaming kernels for
# each number of token tiles, rows made integers inside or before, and the GEMM's classes with and without split reductions and a launch
# for the columns that whole rounds leave.  References on the GPU, in float64, whose sums of integers are exact.
@gpu
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize(
    "M,R,C",
    [
        (3, 264, 264), (3, 2056, 264), (3, 264, 8200), (3, 2056, 8200), (3, 2056, 16400), (16, 1600, 4104), (16, 1600, 8200), (16, 2056, 264),
        (16, 2056, 8200), (16, 2056, 16400), (20, 264, 264), (20, 8200, 264), (20, 264, 8200), (40, 264, 264), (40, 264, 8200), (40, 264, 12296),
        (100, 264, 264), (100, 264, 8200), (100, 264, 12296), (129, 264, 520), (129, 2056, 520), (129, 14344, 5640), (300, 4104, 20488),
        (512, 2056, 20488), (1000, 2056, 16392), (2300, 4104, 10248),
    ],
)
def test_q8_linear_on_every_kernel(M, R, C, dtype):
    g = gen(M + C)
    x, q = on(normal((M, R), 1.0, dtype, g)), q8((C, R), dtype, g)
    b = on(normal((C,), 0.5, dtype, g))
    y = quant.q8_linear_fwd(x, q, b)
    n, s = integers64(x)
    ref = (n @ numbers_of(q, x.device).T) * s * q.scales.double()
    bound = 8 * F * (ref.abs() + b.double().abs())
    hold(y, (ref + b.double()).cpu(), bound.cpu(), dtype)


@gpu
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize(
    "M,K,N,act",
    [
        (3, 264, 264, "silu"), (3, 2056, 8200, "silu"), (3, 8200, 264, "gelu"), (16, 1600, 4104, "silu"), (16, 2056, 8200, "silu"), (16, 8200, 264, "gelu"),
        (20, 264, 264, "silu"), (20, 8200, 264, "silu"), (20, 264, 4104, "gelu"), (40, 264, 264, "silu"), (40, 264, 4104, "silu"), (100, 264, 264, "silu"),
        (100, 264, 4104, "silu"), (100, 264, 8200, "gelu"), (129, 264, 520, "silu"), (129, 264, 520, "gelu"), (200, 2056, 520, "silu"),
        (200, 2056, 520, "gelu"), (300, 14344, 2056, "silu"), (300, 14344, 2056, "tanh"), (129, 4104, 14344, "silu"), (129, 4104, 14344, "gelu"),
        (129, 2056, 20488, "silu"), (129, 2056, 20488, "relu"), (512, 2056, 16392, "silu"), (512, 2056, 16392, "gelu"), (2048, 8200, 5640, "silu"),
    ],
)
def test_q8_mlp_on_every_kernel(M, K, N, act, dtype):
    """The hidden states, read through a down projection that picks one column for each output: 127·127/127 of its integer."""
    g = gen(M + N)
    x = on(normal((M, K), 1.0, dtype, g))
    w = [q8((N, K), dtype, g), q8((N, K), dtype, g)]
    at = torch.arange(K, device="cuda") % N if K > N else torch.linspace(0, N - 1, K, device="cuda").long()
    pick = torch.zeros(K, N, dtype=dtype, device="cuda")
    pick[torch.arange(K, device="cuda"), at] = 1
    y = quant.q8_mlp_fwd(x, w[0], None, w[1], None, quant.quantize_q8(pick), None, act_fn=act)
    n, s = integers64(x)
    gate, up = ((n @ numbers_of(q, x.device).T) * s * q.scales.double() for q in w)
    a = ACT[act](gate)
    h = a * up
    d = (1.13 * 8 * F * gate.abs() + 2e-6 * (1 + a.abs())) * (up.abs() + 8 * F * up.abs()) + 8 * F * a.abs() * up.abs() + 2 * F * h.abs()
    lo, hi = (h - d).to(dtype), (h + d).to(dtype)
    top = torch.maximum(lo.abs(), hi.abs()).double().amax(1, keepdim=True)
    # a rounding to 16 bits, half a step of the row's integers and of y's own 16 bits
    off = (y.double() - h[:, at]).abs()
    assert (off <= (hi.double() - lo.double()).abs()[:, at] + 2 * U[dtype] * h[:, at].abs() + 0.51 * top / 127 + SUB[dtype]).all()


# An expert's tokens through its layer alone: with one choice of weight 1 the same integers and sums.  An expert's sum is a float, rounded to
# 16 bits when the choices are joined; a layer's alone may be rounded to 16 bits from the product itself, which for float16 an
# instruction does.  A product v = n·(s_x·s_w) and its float rn32(v) lie between the same neighbouring 16-bit numbers a <= b (both
# are floats, and rounding is monotonic), so that each result is a or b: one step apart at most.
@gpu
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize(
    "M,K,N,E",
    [
        (3, 264, 2056, 2), (3, 4104, 2056, 2), (3, 8200, 2056, 2), (3, 2056, 8200, 2), (3, 8200, 264, 2), (4, 264, 520, 1), (3, 264, 2056, 1), (2, 8200, 264, 1), (3, 8200, 2056, 1), (2, 16400, 2056, 1), (3, 2056, 8200, 1),
        (10, 264, 520, 1), (10, 264, 2056, 1), (10, 8200, 264, 1), (10, 8200, 2056, 1), (10, 16400, 2056, 1), (10, 2056, 8200, 1),
        (20, 264, 520, 1), (20, 264, 8200, 1), (20, 8200, 264, 1), (40, 264, 520, 1), (40, 8200, 4104, 1), (40, 12296, 264, 1),
        (60, 264, 520, 1), (60, 8200, 4104, 1), (60, 12296, 8200, 1), (50, 264, 520, 6), (300, 264, 520, 9), (700, 520, 264, 9),
        (300, 264, 264, 1), (900, 2056, 8200, 2), (1500, 4104, 2056, 5), (1500, 4104, 4104, 5), (4500, 2056, 4104, 2), (2300, 2056, 8200, 8),
    ],
)
@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_q8_experts_on_every_kernel(M, K, N, E, act, dtype):
    g = gen(M + K)
    x, choice = on(normal((M, K), 1.0, dtype, g)), torch.arange(M) * 7 % E
    if M // E > 128:
        choice[torch.arange(M) % 10 == 9] = E - 1  # (one with more rows than the others; all of them by the GEMM)
    logits = on(torch.nn.functional.one_hot(choice, E).float() * 5)
    w = [q8((E, N, K), dtype, g), q8((E, N, K), dtype, g), q8((E, K, N), dtype, g)]
    y = moe.moe_mlp_fwd(x, logits, *w, 1, act_fn=act)
    for e in range(E):
        rows = on((choice == e).nonzero()[:, 0])
        gate, up, down = (sliced(q, e) for q in w)
        alone = quant.q8_mlp_fwd(x[rows], gate, None, up, None, down, None, act_fn=act)
        assert alone.isfinite().all() and ((alone == y[rows]) | ((alone.view(torch.int16).int() - y[rows].view(torch.int16).int()).abs() <= 1)).all()


@gpu
@pytest.mark.parametrize("M", [2, 128, 129])
@pytest.mark.parametrize("logits_dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("E,k", [(3, 3), (16, 4), (60, 6), (100, 5), (250, 16), (500, 2)])
def test_q8_experts_by_logits_of_each_type(M, logits_dtype, E, k):
    dtype, K, N = torch.bfloat16, 72, 40
    g = gen(E)
    x, logits = normal((M, K), 1.0, dtype, g), normal((M, E), 2.0, logits_dtype, g)
    w = [q8((E, N, K), dtype, g), q8((E, N, K), dtype, g), q8((E, K, N), dtype, g)]
    y = moe.moe_mlp_fwd(on(x), on(logits), *w, k)
    ref, bound = moe64(x, logits, k, True, "silu", dtype, lambda e: [weight_of(sliced(q, e)) for q in w])
    hold(y, ref, bound, dtype, N)


@gpu
@pytest.mark.parametrize("M", [1, 20, 200])
def test_rows_of_q8_layers_stand_alone(M):
    """What is not finite stays with its token; other rows are as without it, bit for bit; calls repeat bit for bit."""
    dtype, K, N, E, k = torch.float16, 264, 136, 6, 2
    g = gen(M)
    x, logits = on(normal((M, K), 1.0, dtype, g)), on(normal((M, E), 1.0, torch.float32, g))
    w = [q8((E, N, K), dtype, g), q8((E, N, K), dtype, g), q8((E, K, N), dtype, g)]
    y = moe.moe_mlp_fwd(x, logits, *w, k)
    assert torch.equal(y, moe.moe_mlp_fwd(x, logits, *w, k))
    bad = x.clone()
    bad[M // 2, 5] = math.nan
    z = moe.moe_mlp_fwd(bad, logits, *w, k)
    rest = torch.arange(M, device=x.device) != M // 2
    assert z[M // 2].isnan().all() and torch.equal(z[rest], y[rest])
    logits[M // 2, 3] = math.nan  # (weights NaN)
    z = moe.moe_mlp_fwd(x, logits, *w, k)
    assert z[M // 2].isnan().all() and torch.equal(z[rest], y[rest])


@gpu
def test_logits_of_every_type_and_a_long_batch():
    dtype, K, N, E, k = torch.bfloat16, 64, 64, 16, 16
    g = gen(12)
    w = [q8((E, N, K), dtype, g), q8((E, N, K), dtype, g), q8((E, K, N), dtype, g)]
    M = 4200  # more choices than a call of the library takes
    x = normal((M, K), 1.0, dtype, g)
    for logits_dtype in (torch.float32, torch.float16, torch.bfloat16):
        logits = normal((M, E), 1.5, logits_dtype, g)
        y = moe.moe_mlp_fwd(on(x), on(logits), *w, k)
        rows = torch.tensor([0, 1, 4095, 4096, 4097, M - 1])
        ref, bound = moe64(x[rows], logits[rows], k, True, "silu", dtype, lambda e: [weight_of(sliced(q, e)) for q in w])
        hold(y[on(rows)], ref, bound, dtype, len(rows) * N)


@gpu
@pytest.mark.parametrize("rows", [1, 3, 100, 500])
def test_operators_on_another_stream_and_in_a_graph(rows):
    dtype, K, N, E = torch.bfloat16, 264, 392, 8
    g = gen(rows)
    w = [q8((E, N, K), dtype, g), q8((E, N, K), dtype, g), q8((E, K, N), dtype, g)]
    one = [sliced(q, 1) for q in w]
    x, logits = on(normal((rows, K), 1.0, dtype, g)), on(normal((rows, E), 1.0, torch.float32, g))

    def everything():
        return (quant.q8_linear_fwd(x, one[0]), quant.q8_mlp_fwd(x, one[0], None, one[1], None, one[2], None),
                moe.moe_mlp_fwd(x, logits, *w, 2))

    eager = everything()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = everything()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(eager, other))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = everything()
    for seed in range(4):
        x.copy_(normal((rows, K), 1.0, dtype, gen(100 + seed)))
        logits.copy_(normal((rows, E), 1.0, torch.float32, gen(200 + seed)))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(captured, everything()):
            assert torch.equal(a, b)


# ------------------------------------------------------------------ modules
@gpu
@pytest.mark.parametrize("rows", [2, 90])
def test_modules(rows, tmp_path):
    dtype = torch.bfloat16
    torch.manual_seed(0)
    mlp = FusedGatedMLP(264, 520, bias=True).to(device()).to(dtype).eval()
    x = on(normal((rows, 264), 1.0, dtype, gen(1)))
    q = Q8GatedMLP.from_float(mlp)
    with torch.no_grad():
        y = q(x.view(1, rows, 264))
    assert y.shape == (1, rows, 264)
    w = [quant.quantize_q8(getattr(mlp, n).weight.detach()) for n in ("gate_proj", "up_proj", "down_proj")]
    b = [getattr(mlp, n).bias.detach() for n in ("gate_proj", "up_proj", "down_proj")]
    assert torch.equal(y[0], quant.q8_mlp_fwd(x, w[0], b[0], w[1], b[1], w[2], b[2]))
    # the scales stay as they are whatever the module is converted to
    before = q.gate_proj.scales.clone()
    q.half()
    assert torch.equal(q.gate_proj.scales, before) and q.b_gate.dtype == torch.float16 and q.gate_proj.codes.dtype == torch.int8
    again = Q8GatedMLP.from_float(mlp)
    again.load_state_dict({k: v.to(dtype) if k.startswith("b_") else v for k, v in q.state_dict().items()})
    with torch.no_grad():
        assert torch.equal(again(x), y[0])
    layer = GatedMoE(264, 136, 6, 2).to(device()).to(dtype)
    with torch.no_grad():
        gate, up, down = (quant.quantize_q8(getattr(layer, n).detach()) for n in ("gate_proj", "up_proj", "down_proj"))
        layer.quantize_(bits=8)
        assert layer.quantized
        logits = layer.route_logits(x)
        assert torch.equal(layer(x), moe.moe_mlp_fwd(x, logits, gate, up, down, 2))
        assert layer(x[:0]).shape == (0, 264)


@gpu
def test_the_decode_example_runs_in_8_bits():
    from triton_gated_mlp.decode_example import main

    assert main(["--tokens", "2", "--layers", "2", "--hidden", "256", "--intermediate", "512", "--expert", "128", "--experts", "8", "--top-k", "2",
                 "--bits", "8", "--steps", "3"]) > 0
