"""4-bit weights, expert routing and expert layers against plain implementations in 64 bits.

Tolerances.  u is half a unit in the last place of the output type (2^-11 fp16, 2^-8 bf16), s the smallest subnormal's half.
A sum of n products accumulated in fp32 (rounded or truncated at each addition) is off by at most (n + 16) 2^-23 of the sum
of their magnitudes.  So a linear layer is held, element by element, to u |y| + (n + 16) 2^-23 (|x| |W|ᵀ + |b|) + s.  A gated
MLP adds what its hidden states are off by, carried through |W_down|: their own rounding, and act(g) u with g and u off by
their sums' bounds (every activation's slope is at most 1.13, the device's activations are within 2e-6 of theirs).  Those
bounds grow with n while errors grow with its root, so the 2-norm is held too: a rounding is at most u / sqrt(3) in the mean
square, two of them 0.82 u, so the norm of the error is at most u times the result's (one rounding: 0.6 u).
"""

import math

import pytest
import torch

from triton_gated_mlp import _cabi
from triton_gated_mlp.ops import moe, quant

U = {torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}
SUB = {torch.float16: 2.0**-25, torch.bfloat16: 2.0**-134}
HALF = [torch.float16, torch.bfloat16]


# ------------------------------------------------------------------ plain implementations
def numbers_of(q):
    """(n, scale of each) of a single Q4Weight as float64 [rows, cols], looked up one place at a time."""
    codes, scales = q.codes.cpu().reshape(-1), q.scales.cpu().double().reshape(-1)
    KB, g = q.codes.shape[-5], q.group_size
    r = torch.arange(q.rows).unsqueeze(1)
    c = torch.arange(q.cols).unsqueeze(0)
    block = (r // 16) * KB + c // 128
    nibble = torch.where(c % 2 == 0, (c % 8) // 2, 4 + (c % 8) // 2)
    byte = block * 1024 + ((c % 32) // 8) * 256 + (r % 16) * 16 + ((c % 128) // 32) * 4 + nibble // 2
    n = ((codes[byte].int() >> (4 * (nibble % 2))) & 15) - 8
    at = block * (16 * 128 // g) + ((r % 16) // 4) * (4 * 128 // g) + ((c % 128) // g) * 4 + r % 4
    return n.double(), scales[at]


def weights_of(q):
    n, s = numbers_of(q)
    return n * s


def sliced(q, e):
    return quant.Q4Weight(q.codes[e], q.scales[e], q.rows, q.cols, q.group_size)


ACT = {
    "silu": lambda g: g * torch.sigmoid(g),
    "gelu": torch.nn.functional.gelu,
    "relu": torch.relu,
    "leaky_relu": torch.nn.functional.leaky_relu,
    "sigmoid": torch.sigmoid,
    "tanh": torch.tanh,
    "no_act": lambda g: g,
}


def linear64(x, w, b, dtype):
    """(y, bound) in float64."""
    y, mass = x @ w.T, x.abs() @ w.abs().T
    if b is not None:
        y, mass = y + b, mass + b.abs()
    return y, U[dtype] * y.abs() + (x.shape[1] + 16) * 2.0**-23 * mass + SUB[dtype]


def mlp64(x, wg, bg, wu, bu, wd, bd, act, dtype):
    """(y, bound) before the rounding of y, in float64."""
    u = U[dtype]
    g, dg = linear64(x, wg, bg, dtype)
    v, dv = linear64(x, wu, bu, dtype)
    dg, dv = dg - u * g.abs(), dv - u * v.abs()  # these two stay in fp32
    a = ACT[act](g)
    h = a * v
    da = 1.13 * dg + 2e-6 * (1 + a.abs())
    dh = da * (v.abs() + dv) + a.abs() * dv + u * h.abs() + SUB[dtype]
    y, mass = h @ wd.T, h.abs() @ wd.abs().T
    if bd is not None:
        y, mass = y + bd, mass + bd.abs()
    return y, dh @ wd.abs().T + (h.shape[1] + 16) * 2.0**-23 * mass


def route64(logits, k, normalize):
    """(weights, experts): the largest that is left, one after the other."""
    rows = []
    for row in logits.double().tolist():
        left = list(range(len(row)))
        picks = []
        for _ in range(k):
            best = left[0]
            for e in left[1:]:
                if row[e] > row[best]:
                    best = e
            picks.append(best)
            left.remove(best)
        top = max(row)
        if top == -math.inf:
            rows.append(([0.0] * k, picks))
            continue
        p = [math.exp(v - top) for v in row]
        total = sum(p[e] for e in picks) if normalize else sum(p)
        rows.append(([p[e] / total for e in picks], picks))
    return torch.tensor([w for w, _ in rows], dtype=torch.float64), torch.tensor([e for _, e in rows])


def moe64(x, logits, k, normalize, act, dtype, weights):
    """weights(e) -> (W_gate, W_up, W_down) in float64; (y, bound)."""
    w, experts = route64(logits, k, normalize)
    y, bound = torch.zeros_like(x), torch.zeros_like(x)
    mass = torch.zeros_like(x)
    for e in sorted(set(experts.reshape(-1).tolist())):
        t, j = torch.nonzero((experts == e) & (w > 0), as_tuple=True)
        if len(t) == 0:
            continue
        wg, wu, wd = weights(e)
        out, off = mlp64(x[t], wg, None, wu, None, wd, None, act, dtype)
        y[t] += w[t, j, None] * out
        bound[t] += w[t, j, None] * (off + 1e-6 * out.abs())  # (a weight is within 1e-6 of its own)
        mass[t] += (w[t, j, None] * out).abs()
    return y, bound + U[dtype] * y.abs() + (k + 16) * 2.0**-23 * mass + SUB[dtype]


def hold(got, y, bound, dtype, roundings):
    got = got.detach().double().cpu().reshape(y.shape)
    assert torch.isfinite(got).all()
    off = (got - y).abs()
    assert (off <= bound).all(), f"off by {(off / bound).max().item():.3f} of the bound"
    if y.numel() >= 64 and y.norm() > 0:
        rel = ((got - y).norm() / y.norm()).item()
        assert rel <= U[dtype] * (0.6 if roundings == 1 else 1.0), f"2-norm off by {rel / U[dtype]:.3f} u"


def gen(seed):
    return torch.Generator().manual_seed(seed)


def normal(shape, std, dtype, g):
    return (std * torch.randn(shape, generator=g)).to(dtype)


# ------------------------------------------------------------------ without a GPU
def test_refusals_of_the_c_interface():
    import ctypes

    lib = _cabi.lib()
    raw = ctypes.create_string_buffer(4096 + 64)
    a = (ctypes.addressof(raw) + 63) & ~63
    err = lambda: lib.gmlp_last_error().decode()
    # NULL, group size, dtype, widths, rows, alignment
    assert lib.gmlp_q4_linear_fwd(None, a, a, None, a, 1, 64, 64, 128, 0, None, 0, None) == -1 and "NULL" in err()
    assert lib.gmlp_q4_linear_fwd(a, a, a, None, a, 1, 64, 64, 48, 0, None, 0, None) == -1 and "group" in err()
    assert lib.gmlp_q4_linear_fwd(a, a, a, None, a, 1, 64, 64, 128, 2, None, 0, None) == -2
    assert lib.gmlp_q4_linear_fwd(a, a, a, None, a, 1, 64, 64, 128, 9, None, 0, None) == -1
    assert lib.gmlp_q4_linear_fwd(a, a, a, None, a, 1, 60, 64, 128, 0, None, 0, None) == -2 and "multiple of 8" in err()
    assert lib.gmlp_q4_linear_fwd(a, a, a, None, a, 1, 64, 60, 128, 0, None, 0, None) == -2
    assert lib.gmlp_q4_linear_fwd(a, a, a, None, a, 65, 64, 64, 128, 0, None, 0, None) == -2 and "64" in err()
    assert lib.gmlp_q4_linear_fwd(a, a, a, None, a, 0, 64, 64, 128, 0, None, 0, None) == -2
    assert lib.gmlp_q4_linear_fwd(a + 8, a, a, None, a, 1, 64, 64, 128, 0, None, 0, None) == -3
    assert lib.gmlp_q4_linear_fwd(a, a, a, a + 2, a, 1, 64, 64, 128, 0, None, 0, None) == -3
    mlp = lambda x, M, K, N, group, dtype, act: lib.gmlp_q4_mlp_fwd(x, a, a, a, a, a, a, None, None, None, a, a, M, K, N, group, dtype, act, None, 0, None)
    assert mlp(None, 1, 64, 64, 32, 0, 0) == -1 and mlp(a, 1, 64, 64, 32, 0, 7) == -1 and "act" in err()
    assert mlp(a, 1, 64, 68, 32, 0, 0) == -2 and mlp(a, 65, 64, 64, 32, 0, 0) == -2 and mlp(a, 1, 64, 64, 16, 0, 0) == -1
    for quantize in (lib.gmlp_q4_quantize, lib.gmlp_q4_dequantize):
        assert quantize(a, None, a, 1, 16, 128, 32, 0, None) == -1
        assert quantize(a, a, a, 1, 16, 128, 100, 0, None) == -1
        assert quantize(a, a, a, 0, 16, 128, 32, 0, None) == -2
        assert quantize(a, a, a, 1, 12, 128, 32, 0, None) == -2
        assert quantize(a, a, a, 1, 16, 128, 32, 2, None) == -2
        assert quantize(a, a, a, 1 << 40, 16, 128, 32, 0, None) == -2
    assert lib.gmlp_moe_route(a, a, None, 1, 8, 2, 1, 2, None) == -1
    assert lib.gmlp_moe_route(a, a, a, 1, 8, 9, 1, 2, None) == -2 and "top_k" in err()
    assert lib.gmlp_moe_route(a, a, a, 1, 8, 0, 1, 2, None) == -2
    assert lib.gmlp_moe_route(a, a, a, 1, 513, 2, 1, 2, None) == -2
    assert lib.gmlp_moe_route(a, a, a, 1, 64, 17, 1, 2, None) == -2
    assert lib.gmlp_moe_route(a, a, a, 0, 8, 2, 1, 2, None) == -2
    assert lib.gmlp_moe_route(a, a, a, 1, 8, 2, 1, 5, None) == -1
    need = lib.gmlp_moe_workspace_bytes(4, 64, 64, 8, 2, 0, 0)
    assert need >= 4 * 2 * 64 * 2
    assert lib.gmlp_moe_workspace_bytes(65, 64, 64, 8, 2, 0, 0) == 0

    def layer(x=a, logits=a, s=None, y=a, M=4, K=64, N=64, E=8, k=2, group=0, dtype=0, ld=2, act=0, ws=a, n=need):
        return lib.gmlp_moe_fwd(x, logits, a, a, a, s, s, s, y, M, K, N, E, k, 1, group, dtype, ld, act, ws, n, None)

    assert layer(x=None) == -1 and layer(logits=None) == -1 and layer(ws=None) == -1
    assert layer(n=need - 1) == -1 and "workspace" in err()
    assert layer(M=65) == -2 and layer(M=0) == -2 and layer(K=60) == -2 and layer(N=4) == -2 and layer(k=9) == -2 and layer(E=600) == -2
    assert layer(group=128) == -1 and layer(group=5, s=a) == -1 and layer(dtype=2) == -2 and layer(ld=3) == -1 and layer(act=9) == -1
    assert layer(x=a + 4) == -3 and layer(ws=a + 8) == -3


def test_storage_that_a_launch_has_no_threads_for_is_refused():
    """A wavefront of 64 threads per 1 KiB of codes, and less than 2^32 in a launch: 2^26 of them are too many."""
    import ctypes

    lib = _cabi.lib()
    raw = ctypes.create_string_buffer(64 + 64)
    a = (ctypes.addressof(raw) + 63) & ~63
    for call in (lib.gmlp_q4_quantize, lib.gmlp_q4_dequantize):
        for count, rows, cols in ((1 << 26, 8, 8), (1 << 20, 1024, 72), (1, 1 << 20, 1 << 17), (1 << 31, 16, 128)):
            assert call(a, a, a, count, rows, cols, 32, 0, None) == -2 and "too large" in lib.gmlp_last_error().decode()


def test_expert_layers_that_a_launch_has_no_threads_for_are_refused():
    """256 experts in use times 2^20 / 16 tiles of gate/up, 256 threads each, are 2^32 threads."""
    import ctypes

    lib = _cabi.lib()
    raw = ctypes.create_string_buffer(64 + 64)
    a = (ctypes.addressof(raw) + 63) & ~63

    def layer(N, group, s):  # (a workspace of no bytes: what the sizes leave is refused behind them)
        return lib.gmlp_moe_fwd(a, a, a, a, a, s, s, s, a, 16, 8, N, 256, 16, 1, group, 0, 2, 0, a, 0, None)

    for group, s in ((0, None), (128, a)):
        assert layer(1 << 20, group, s) == -2 and "too large" in lib.gmlp_last_error().decode()
        assert layer((1 << 20) - 16, group, s) == -1 and "workspace" in lib.gmlp_last_error().decode()


def test_cpu_tensors_are_refused():
    x = torch.zeros(2, 64, dtype=torch.float16)
    with pytest.raises(RuntimeError, match="AMD GPU"):
        moe.moe_route(torch.zeros(2, 8), 2)
    with pytest.raises(RuntimeError, match="AMD GPU"):
        quant.quantize_q4(x)
    w = torch.zeros(8, 64, 64, dtype=torch.float16)
    with pytest.raises(RuntimeError, match="AMD GPU"):
        moe.moe_mlp_fwd(x, torch.zeros(2, 8), w, w, w, 2)


def test_forward_mode_and_functorch_are_refused():
    """Each operator for each tensor that a tangent could come with (a result without it would be wrong)."""
    import torch.autograd.forward_ad as fw

    half = lambda *shape: torch.zeros(shape, dtype=torch.float16)
    codes = lambda *lead: torch.zeros((*lead, 4, 1, 4, 16, 4, 4), dtype=torch.uint8)
    q = lambda scales: quant.Q4Weight(codes(), scales, 64, 64, 128)
    qe = lambda scales: quant.Q4Weight(codes(2), scales, 64, 64, 128)
    x, b, s, se, w, wr = half(3, 64), half(64), half(4, 1, 4, 1, 4), half(2, 4, 1, 4, 1, 4), half(2, 64, 64), half(4, 64)
    logits = torch.zeros(3, 2)
    calls = [
        (lambda t: quant.quantize_q4(t), x), (lambda t: quant.dequantize_q4(q(t)), s),
        (lambda t: quant.q4_linear_fwd(t, q(s)), x), (lambda t: quant.q4_linear_fwd(x, q(t)), s), (lambda t: quant.q4_linear_fwd(x, q(s), t), b),
        *((lambda t, i=i: quant.q4_mlp_fwd(*(t if j == i else v for j, v in enumerate((x, q(s), b, q(s), b, q(s), b)))), x if i == 0 else b)
          for i in (0, 2, 4, 6)),
        *((lambda t, i=i: quant.q4_mlp_fwd(x, *(v for j in range(3) for v in (q(t if j == i else s), None))), s) for i in range(3)),
        (lambda t: moe.moe_logits(t, wr), x), (lambda t: moe.moe_logits(x, t), wr), (lambda t: moe.moe_route(t, 2), logits),
        *((lambda t, i=i: moe.moe_mlp_fwd(*(t if j == i else v for j, v in enumerate((x, logits, w, w, w))), 2), (x, logits, w, w, w)[i])
          for i in range(5)),
        (lambda t: moe.moe_mlp_fwd(t, logits, qe(se), qe(se), qe(se), 2), x),
        *((lambda t, i=i: moe.moe_mlp_fwd(x, logits, *(qe(t if j == i else se) for j in range(3)), 2), se) for i in range(3)),
    ]
    for call, t in calls:
        with pytest.raises(RuntimeError, match="AMD GPU"):  # without a transform it gets as far as the device
            call(t)
        with fw.dual_level(), torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
            call(fw.make_dual(t, t))
        with pytest.raises(RuntimeError, match="functorch"):
            torch.vmap(call)(t[None])
        with pytest.raises(RuntimeError, match="functorch"):
            torch.func.jvp(call, (t,), (t,))
        with pytest.raises(RuntimeError, match="no backward"):
            call(t.clone().requires_grad_(True))


# ------------------------------------------------------------------ 4-bit weights
gpu = pytest.mark.gpu


def device():
    assert torch.cuda.is_available(), "GPU tests need a visible AMD GPU"
    return torch.device("cuda", 0)


@gpu
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("shape", [(8, 8), (16, 128), (40, 200), (3, 24, 328)])
def test_quantize_and_dequantize(shape, group, dtype):
    w = normal(shape, 0.02, dtype, gen(1))
    w[..., 0, :] = 0  # a row of zeros
    q = quant.quantize_q4(w.to(device()), group)
    back = quant.dequantize_q4(q)
    assert back.shape == w.shape and back.dtype == dtype
    experts = [(w, q, back)] if w.dim() == 2 else [(w[e], sliced(q, e), back[e]) for e in range(shape[0])]
    for dense, one, again in experts:
        n, s = numbers_of(one)
        cols = dense.shape[1]
        for first in range(0, cols, group):
            part = dense[:, first : first + group].float()
            scale = (part.abs().amax(1) / 7).to(dtype)
            assert torch.equal(s[:, first].to(dtype), scale)
            step = torch.where(scale > 0, scale.float(), 1.0).unsqueeze(1)
            assert torch.equal(n[:, first : first + group], (part / step).round().clamp(-8, 7).double())
        assert torch.equal(again.cpu(), (n * s).to(dtype))  # (a product of 11 by 4 bits is exact in fp32)
    # the padding holds n = 0
    full = quant.Q4Weight(q.codes, q.scales, q.codes.shape[-6] * 16, q.codes.shape[-5] * 128, group)
    one = full if w.dim() == 2 else sliced(full, 0)
    n, _ = numbers_of(one)
    assert (n[w.shape[-2] :] == 0).all() and (n[:, w.shape[-1] :] == 0).all()


def q4(shape, group, dtype, g):
    return quant.quantize_q4(normal(shape, 0.02, dtype, g).to(device()), group)


@gpu
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize(
    "M,R,C,group,bias",
    [
        (1, 8, 8, 128, False), (1, 128, 16, 32, True), (1, 2048, 256, 128, False), (2, 1160, 3096, 32, True), (7, 264, 72, 64, True),
        (16, 4096, 40, 128, False), (17, 1000, 136, 64, False), (32, 136, 1000, 32, False), (33, 520, 264, 32, True),
        (64, 1032, 520, 128, True), (64, 2048, 48, 64, False), (65, 264, 392, 64, True), (300, 1160, 264, 32, False),
        (1, 136, 4360, 32, True), (3, 1160, 4120, 128, False), (4, 1160, 4120, 32, False), (9, 392, 4360, 64, True),
        (16, 1160, 4360, 32, False), (5, 264, 8456, 128, False), (7, 1160, 8456, 64, False), (20, 136, 4360, 128, True), (60, 136, 4360, 32, False),
        (18, 4360, 136, 128, True), (33, 2824, 72, 32, True), (64, 2184, 200, 64, False), (64, 2184, 200, 32, True),
    ],
)
def test_q4_linear(M, R, C, group, bias, dtype):
    g = gen(M + R)
    x, q = normal((M, R), 1.0, dtype, g), q4((C, R), group, dtype, g)
    b = normal((C,), 0.5, dtype, g) if bias else None
    y = quant.q4_linear_fwd(x.to(device()), q, None if b is None else b.to(device()))
    w = weights_of(q)
    if M > 64:  # on the weights rounded to 16 bits
        w = w.to(dtype).double()
    ref, bound = linear64(x.double(), w, None if b is None else b.double(), dtype)
    hold(y, ref, bound, dtype, 1)


@gpu
@pytest.mark.parametrize("dtype", HALF)
def test_q4_linear_takes_every_code_scale_and_padding(dtype):
    """All sixteen numbers in all places, a scale for every row and group, and padding that holds something else."""
    dev, g = device(), gen(5)
    rows, cols, group = 24, 200, 32
    codes = torch.randint(0, 256, (2, 2, 4, 16, 4, 4), generator=g, dtype=torch.uint8)
    scales = (0.01 + torch.rand((2, 2, 4, 4, 4), generator=g)).to(dtype)
    q = quant.Q4Weight(codes.to(dev), scales.to(dev), rows, cols, group)
    x = normal((3, cols), 1.0, dtype, g)
    ref, bound = linear64(x.double(), weights_of(q), None, dtype)
    hold(quant.q4_linear_fwd(x.to(dev), q), ref, bound, dtype, 1)
    # one column at a time: the result is scale * n, rounded once
    eye = torch.eye(cols, dtype=dtype)[:64]
    assert torch.equal(quant.q4_linear_fwd(eye.to(dev), q).cpu(), weights_of(q)[:, :64].T.to(dtype))


@gpu
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize(
    "M,K,N,group,bias,act",
    [
        (1, 8, 8, 32, False, "silu"), (1, 2048, 264, 128, False, "silu"), (3, 264, 1032, 32, True, "gelu"), (16, 520, 640, 64, True, "tanh"),
        (17, 136, 392, 128, False, "relu"), (48, 264, 520, 64, True, "gelu"), (64, 1032, 264, 32, False, "leaky_relu"),
        (5, 128, 128, 128, True, "sigmoid"), (9, 256, 384, 32, False, "no_act"), (130, 264, 520, 64, True, "silu"),
        (48, 72, 2824, 64, True, "gelu"),
        (20, 1672, 72, 32, True, "silu"), (40, 72, 4360, 64, False, "silu"), (64, 1672, 4360, 128, False, "relu"), (60, 136, 8456, 128, True, "silu"),
    ],
)
def test_q4_mlp(M, K, N, group, bias, act, dtype):
    dev, g = device(), gen(M + K)
    x = normal((M, K), 1.0, dtype, g)
    qs = [q4((N, K), group, dtype, g), q4((N, K), group, dtype, g), q4((K, N), group, dtype, g)]
    bs = [normal((n,), 0.1, dtype, g) if bias else None for n in (N, N, K)]
    on = [None if b is None else b.to(dev) for b in bs]
    y = quant.q4_mlp_fwd(x.to(dev), qs[0], on[0], qs[1], on[1], qs[2], on[2], act_fn=act)
    ws = [weights_of(q) for q in qs]
    if M > 64:
        ws = [w.to(dtype).double() for w in ws]
    b64 = [None if b is None else b.double() for b in bs]
    ref, bound = mlp64(x.double(), ws[0], b64[0], ws[1], b64[1], ws[2], b64[2], act, dtype)
    hold(y, ref, bound + U[dtype] * ref.abs() + SUB[dtype], dtype, 2)


@gpu
@pytest.mark.parametrize("M", [1, 2, 3, 16, 17, 64])
def test_q4_mlp_writes_as_much_scratch_as_the_header_says(M):
    """h of GMLP_Q4_MLP_H_ELEMENTS, all of it in use, and nothing behind it."""
    import re
    from pathlib import Path

    header = (Path(__file__).resolve().parent.parent / "include" / "gmlp.h").read_text()
    pairs = int(re.search(r"#define GMLP_H_PAIR_ROWS_Q4 (\d+)", header).group(1))
    assert re.search(r"GMLP_Q4_MLP_H_ELEMENTS\(M, N\) \(\(\(M\) <= GMLP_H_PAIR_ROWS_Q4 \? 2 : 1\) \* \(M\) \* \(N\)\)", header)
    dev, dtype, K, N, group = device(), torch.bfloat16, 136, 264, 64
    g = gen(M)
    qs = [q4((N, K), group, dtype, g), q4((N, K), group, dtype, g), q4((K, N), group, dtype, g)]
    x = normal((M, K), 1.0, dtype, g).to(dev)
    used = (2 if M <= pairs else 1) * M * N
    h = torch.full((used + 4 * 64 * N,), math.nan, dtype=dtype, device=dev)
    y = torch.full((M + 1, K), math.nan, dtype=dtype, device=dev)
    weights = [t.data_ptr() for q in qs for t in (q.codes, q.scales)]
    rc = _cabi.lib().gmlp_q4_mlp_fwd(x.data_ptr(), *weights, None, None, None, h.data_ptr(), y.data_ptr(), M, K, N, group, 1, 0, None, 0,
                                     _cabi.stream_ptr(dev))
    assert rc == 0
    torch.cuda.synchronize()
    assert torch.isfinite(h[:used]).all() and torch.isnan(h[used:]).all()
    assert torch.isfinite(y[:M]).all() and torch.isnan(y[M]).all()


@gpu
def test_q4_operators_take_leading_dimensions_strides_and_no_rows():
    dev, g, dtype = device(), gen(3), torch.bfloat16
    q = q4((72, 136), 64, dtype, g)
    x = normal((136, 6), 1.0, dtype, g).to(dev)
    y = quant.q4_linear_fwd(x.T.contiguous(), q)
    assert torch.equal(quant.q4_linear_fwd(x.T, q), y)
    assert torch.equal(quant.q4_linear_fwd(x.T.reshape(2, 3, 136), q), y.reshape(2, 3, 72))
    assert torch.equal(quant.q4_linear_fwd(x.T[1], q), y[1])
    wide = torch.zeros(6, 272, dtype=dtype, device=dev)
    wide[:, ::2] = x.T
    assert torch.equal(quant.q4_linear_fwd(wide[:, ::2], q), y)
    assert quant.q4_linear_fwd(x.T[:0], q).shape == (0, 72)
    up, down = q4((72, 136), 64, dtype, g), q4((136, 72), 64, dtype, g)
    out = quant.q4_mlp_fwd(x.T, q, None, up, None, down, None)
    assert torch.equal(quant.q4_mlp_fwd(x.T.reshape(3, 2, 136), q, None, up, None, down, None), out.reshape(3, 2, 136))
    assert quant.q4_mlp_fwd(x.T[:0], q, None, up, None, down, None).shape == (0, 136)
    # a row's result does not depend on the rows beside it in a tile
    for m in (0, 5):
        assert torch.equal(quant.q4_linear_fwd(x.T[m : m + 1], q)[0], y[m])


@gpu
def test_q4_refusals():
    dev, g, dtype = device(), gen(3), torch.float16
    q = q4((72, 136), 64, dtype, g)
    x = normal((4, 136), 1.0, dtype, g).to(dev)
    with pytest.raises(ValueError, match="expected"):
        quant.q4_linear_fwd(x[:, :128].contiguous(), q)
    with pytest.raises(TypeError):
        quant.q4_linear_fwd(x.bfloat16(), q)
    with pytest.raises(TypeError):
        quant.q4_linear_fwd(x.float(), q)
    with pytest.raises(ValueError, match="bias"):
        quant.q4_linear_fwd(x, q, torch.zeros(71, dtype=dtype, device=dev))
    with pytest.raises(ValueError, match="group size"):
        quant.q4_linear_fwd(x, q._replace(group_size=16))
    with pytest.raises(ValueError, match="codes"):
        quant.q4_linear_fwd(x, q._replace(codes=q.codes[:4]))
    with pytest.raises(ValueError, match="scales"):
        quant.q4_linear_fwd(x, q._replace(scales=q.scales.reshape(-1)))
    with pytest.raises(TypeError, match="uint8"):
        quant.q4_linear_fwd(x, q._replace(codes=q.codes.to(torch.int8)))
    with pytest.raises(RuntimeError, match="device"):
        quant.q4_linear_fwd(x, q._replace(codes=q.codes.cpu()))
    with pytest.raises(RuntimeError, match="no backward"):
        quant.q4_linear_fwd(x.clone().requires_grad_(True), q)
    with torch.no_grad():
        quant.q4_linear_fwd(x.clone().requires_grad_(True), q)
    with pytest.raises(RuntimeError, match="traced"):
        torch.jit.trace(lambda t: quant.q4_linear_fwd(t, q), (x,))
    with pytest.raises(ValueError):
        quant.quantize_q4(x[0])
    with pytest.raises(ValueError, match="group size"):
        quant.quantize_q4(x, 48)
    with pytest.raises(NotImplementedError):
        quant.quantize_q4(torch.zeros(12, 128, dtype=dtype, device=dev))
    with pytest.raises(TypeError):
        quant.quantize_q4(x.float())
    with pytest.raises(ValueError, match="group sizes"):
        quant.q4_mlp_fwd(x, q, None, q, None, q4((136, 72), 32, dtype, g), None)
    with pytest.raises(NotImplementedError):
        quant.q4_mlp_fwd(x, q, None, q, None, q4((136, 72), 64, dtype, g), None, act_fn="softsign")


# ------------------------------------------------------------------ routing
@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("normalize", [True, False])
@pytest.mark.parametrize("M,E,k", [(1, 1, 1), (1, 8, 2), (5, 60, 6), (64, 64, 8), (3, 65, 4), (9, 128, 8), (130, 160, 6), (4, 257, 1), (7, 512, 16), (2, 16, 16)])
def test_route(M, E, k, normalize, dtype):
    logits = normal((M, E), 1.5, dtype, gen(M + E))
    w, e = moe.moe_route(logits.to(device()), k, normalize)
    assert w.dtype == torch.float32 and e.dtype == torch.int64 and w.shape == e.shape == (M, k)
    ref, experts = route64(logits, k, normalize)
    assert torch.equal(e.cpu(), experts)
    # an exponential and a quotient in fp32, over a sum of at most 512 terms
    assert torch.allclose(w.cpu().double(), ref, rtol=5e-6, atol=1e-30)


@gpu
@pytest.mark.parametrize("E", [8, 70, 300])
def test_route_ties_masks_and_what_is_not_finite(E):
    inf, nan, low = math.inf, math.nan, torch.finfo(torch.float32).min
    logits = torch.full((8, E), -inf)
    logits[1] = 0.25                      # all equal
    logits[2, 3] = 1.0                    # one is available
    logits[3, 1::2] = torch.arange(len(logits[3, 1::2])).float() % 3  # ties among every other one
    logits[4] = low                       # the type's lowest value is a number
    logits[5], logits[5, 2] = 0.0, -0.0   # the two zeros are equal
    logits[6], logits[6, 4] = 0.0, nan
    logits[7], logits[7, 5] = 0.0, inf
    for normalize in (True, False):
        w, e = moe.moe_route(logits.to(device()), 4, normalize)
        w, e = w.cpu(), e.cpu()
        ref, experts = route64(logits[:6], 4, normalize)
        assert torch.equal(e[:6], experts)
        assert torch.allclose(w[:6].double(), ref, rtol=5e-6, atol=1e-30)
        assert (w[0] == 0).all() and (w[2, 1:] == 0).all()
        assert torch.isnan(w[6]).all() and torch.isnan(w[7]).any()
        assert e[6, 0] == 4 and e[7, 0] == 5


@gpu
def test_route_strides_leading_dimensions_and_refusals():
    dev = device()
    logits = normal((6, 24), 1.5, torch.bfloat16, gen(1)).to(dev)
    w, e = moe.moe_route(logits, 3)
    for view in (logits.T.contiguous().T, logits.reshape(2, 3, 24)):
        w2, e2 = moe.moe_route(view, 3)
        assert w2.shape == (*view.shape[:-1], 3)
        assert torch.equal(w2.reshape(6, 3), w) and torch.equal(e2.reshape(6, 3), e)
    # rows that begin at odd addresses
    odd = torch.empty(1 + 6 * 24, dtype=torch.bfloat16, device=dev)[1:].reshape(6, 24).copy_(logits)
    assert torch.equal(moe.moe_route(odd, 3).weights, w)
    assert moe.moe_route(logits[:0], 3).experts.shape == (0, 3)
    for k in (0, 25):
        with pytest.raises(ValueError, match="top_k"):
            moe.moe_route(logits, k)
    with pytest.raises(NotImplementedError):
        moe.moe_route(torch.zeros(2, 600, device=dev), 2)
    with pytest.raises(NotImplementedError):
        moe.moe_route(torch.zeros(2, 64, device=dev), 17)
    with pytest.raises(TypeError):
        moe.moe_route(logits.double(), 2)
    with pytest.raises(RuntimeError, match="no backward"):
        moe.moe_route(torch.zeros(2, 8, device=dev, requires_grad=True), 2)


@gpu
@pytest.mark.parametrize("M,E", [(2**28 + 9, 2), (2**26 + 5, 257)])
def test_route_of_more_rows_than_a_launch_has_threads_for(M, E):
    """(16 threads a row up to 256 experts, 64 beyond, and less than 2^32 in a launch.)"""
    dev = device()
    logits = torch.zeros((M, E), dtype=torch.float16, device=dev)
    best = torch.arange(M, device=dev) % E
    logits.scatter_(1, best[:, None], 1.0)
    w, e = moe.moe_route(logits, 1, normalize=False)
    assert torch.equal(e[:, 0], best)
    p = math.e / (math.e + E - 1)
    assert (w - p).abs().max().item() <= 5e-6 * p
    del logits, best, w, e
    torch.cuda.empty_cache()


# ------------------------------------------------------------------ expert layers
def experts_of(E, K, N, bits, group, dtype, g):
    """(gate, up, down) for the operator, and a function that gives one expert's in float64."""
    ws = [normal(shape, 0.05, dtype, g).to(device()) for shape in ((E, N, K), (E, N, K), (E, K, N))]
    if bits == 4:
        qs = [quant.quantize_q4(w, group) for w in ws]
        return qs, lambda e: tuple(weights_of(sliced(q, e)) for q in qs)
    return ws, lambda e: tuple(w[e].cpu().double() for w in ws)


@gpu
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize(
    "M,K,N,E,k,bits,group,act,normalize",
    [
        (1, 8, 8, 1, 1, 16, 0, "silu", True), (1, 256, 136, 8, 2, 16, 0, "silu", True), (1, 264, 392, 8, 2, 4, 32, "gelu", True),
        (2, 136, 72, 4, 4, 16, 0, "relu", False), (7, 200, 328, 16, 4, 4, 64, "silu", False), (16, 264, 136, 60, 6, 16, 0, "silu", True),
        (16, 392, 264, 8, 2, 4, 128, "silu", True), (17, 72, 200, 4, 2, 16, 0, "tanh", True), (33, 136, 264, 128, 8, 16, 0, "silu", False),
        (40, 264, 136, 8, 3, 4, 32, "silu", True), (64, 128, 64, 512, 16, 16, 0, "silu", True), (64, 136, 72, 2, 1, 4, 64, "gelu", True),
        (64, 8, 8, 1, 1, 16, 0, "silu", False), (64, 136, 1032, 1, 1, 4, 32, "silu", True),
        (1, 72, 4264, 4, 4, 16, 0, "silu", True), (12, 136, 1032, 32, 2, 4, 64, "silu", False), (2, 200, 1544, 16, 8, 4, 32, "gelu", True),
        (64, 136, 4296, 1, 1, 4, 32, "silu", True), (40, 264, 1160, 8, 3, 4, 32, "silu", True),
        (100, 72, 136, 8, 2, 16, 0, "silu", True), (130, 72, 136, 8, 2, 4, 128, "silu", True),
    ],
)
def test_moe_mlp(M, K, N, E, k, bits, group, act, normalize, dtype):
    g = gen(M + K + N)
    x, logits = normal((M, K), 1.0, dtype, g), normal((M, E), 1.5, torch.float32, g)
    ws, one = experts_of(E, K, N, bits, group, dtype, g)
    y = moe.moe_mlp_fwd(x.to(device()), logits.to(device()), *ws, k, normalize=normalize, act_fn=act)
    ref, bound = moe64(x.double(), logits, k, normalize, act, dtype, one)
    hold(y, ref, bound, dtype, 2)


@gpu
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("M,bits", [(1, 4), (2, 4), (1, 16), (2, 16), (3, 16), (4, 16)])
def test_hidden_states_of_a_few_tokens_keep_more_than_16_bits(M, bits, dtype):
    """Only y is rounded: its 2-norm is off by what one rounding costs (at most 0.6 u), not by two roundings' 0.8 u."""
    dev, K, N, E = device(), 1032, 392, 4
    g = gen(M)
    x, logits = normal((M, K), 1.0, dtype, g), normal((M, E), 1.0, torch.float32, g)
    ws, one = experts_of(E, K, N, bits, 64, dtype, g)
    ref, bound = moe64(x.double(), logits, 2, True, "silu", dtype, one)
    hold(moe.moe_mlp_fwd(x.to(dev), logits.to(dev), *ws, 2), ref, bound, dtype, 1)
    if bits == 4:
        y, off = mlp64(x.double(), *(v for w in one(1) for v in (w, None)), "silu", dtype)
        hold(quant.q4_mlp_fwd(x.to(dev), *(v for w in ws for v in (sliced(w, 1), None))), y, off + U[dtype] * y.abs() + SUB[dtype], dtype, 1)
    else:
        ws[2][:, 9, 17] = math.inf  # the rest of a hidden state can be 0: infinite, not NaN
        y = moe.moe_mlp_fwd(x.to(dev), logits.to(dev), *ws, 1).cpu()
        assert torch.isinf(y[:, 9]).all()
        y[:, 9] = 0
        assert torch.isfinite(y).all()


@gpu
@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("M", [1, 16, 50])
def test_moe_mlp_with_masked_experts(M, bits):
    """Rows that leave fewer experts than top_k, rows that leave none, and everything on one expert."""
    dev, dtype, E, K, N = device(), torch.bfloat16, 8, 136, 72
    g = gen(M)
    x, logits = normal((M, K), 1.0, dtype, g), normal((M, E), 1.5, torch.float32, g)
    ws, one = experts_of(E, K, N, bits, 32, dtype, g)
    logits[:, 1:] = logits[:, 1:].masked_fill(torch.rand((M, E - 1), generator=g) < 0.7, -math.inf)
    if M > 2:
        logits[2] = -math.inf
    y = moe.moe_mlp_fwd(x.to(dev), logits.to(dev), *ws, 3)
    ref, bound = moe64(x.double(), logits, 3, True, "silu", dtype, one)
    hold(y, ref, bound, dtype, 2)
    if M > 2:
        assert (y[2] == 0).all()
    logits[:, 1:] = -math.inf
    y = moe.moe_mlp_fwd(x.to(dev), logits.to(dev), *ws, 3)
    ref, bound = moe64(x.double(), logits, 1, True, "silu", dtype, one)
    hold(y, ref, bound, dtype, 2)
    assert (moe.moe_mlp_fwd(x.to(dev), torch.full((M, E), -math.inf, device=dev), *ws, 3) == 0).all()


@gpu
@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("M,E,k", [(17, 40, 2), (64, 64, 2), (64, 512, 3), (48, 6, 2)])
def test_moe_mlp_with_one_crowded_expert(M, E, k, bits):
    """An expert that every token chose beside many that one or two did: its tokens are more than the kernels take at once."""
    dev, dtype, K, N = device(), torch.float16, 72, 136
    g = gen(M + E)
    x, logits = normal((M, K), 1.0, dtype, g), normal((M, E), 1.0, torch.float32, g)
    logits[:, 3] += 20
    logits[5, 3] = -math.inf
    ws, one = experts_of(E, K, N, bits, 128, dtype, g)
    y = moe.moe_mlp_fwd(x.to(dev), logits.to(dev), *ws, k, normalize=False)
    ref, bound = moe64(x.double(), logits, k, False, "silu", dtype, one)
    hold(y, ref, bound, dtype, 2)


@gpu
@pytest.mark.parametrize("M,E", [(16, 4), (40, 4), (40, 20)])
def test_what_is_not_finite_stays_with_its_token_and_its_expert(M, E):
    dev, dtype, K, N = device(), torch.float16, 136, 72
    g = gen(0)
    x, logits = normal((M, K), 1.0, dtype, g).to(dev), normal((M, E), 1.5, torch.float32, g).to(dev)
    (gate, up, down), _ = experts_of(E, K, N, 16, 0, dtype, g)
    y = moe.moe_mlp_fwd(x, logits, gate, up, down, 2)
    experts = moe.moe_route(logits, 2).experts
    for ruined in range(3):
        ws = [t.clone() for t in (gate, up, down)]
        ws[ruined][3] = math.nan
        out = moe.moe_mlp_fwd(x, logits, *ws, 2)
        chose = (experts == 3).any(1)
        assert chose.any() and (~chose).any()
        assert torch.equal(out[~chose], y[~chose]) and torch.isnan(out[chose]).all()
    bad = x.clone()
    bad[5] = math.nan
    out = moe.moe_mlp_fwd(bad, logits, gate, up, down, 2)
    keep = torch.arange(M, device=dev) != 5
    assert torch.equal(out[keep], y[keep]) and torch.isnan(out[5]).all()
    # a token whose logits are not finite, in the way softmax has it
    wrong = logits.clone()
    wrong[7, 1] = math.nan
    out = moe.moe_mlp_fwd(x, wrong, gate, up, down, 2)
    keep = torch.arange(M, device=dev) != 7
    assert torch.equal(out[keep], y[keep]) and torch.isnan(out[7]).all()


@gpu
@pytest.mark.parametrize("bits", [16, 4])
def test_moe_mlp_rows_stand_alone_and_repeat(bits):
    """Other tokens of the batch change nothing but rounding (the sums' order may differ), leading dimensions and strides
    nothing at all, and neither does another call."""
    dev, dtype, E, K, N, M = device(), torch.bfloat16, 8, 264, 136, 12
    g = gen(9)
    x, logits = normal((M, K), 1.0, dtype, g).to(dev), normal((M, E), 1.5, torch.float32, g).to(dev)
    ws, one = experts_of(E, K, N, bits, 64, dtype, g)
    y = moe.moe_mlp_fwd(x, logits, *ws, 2)
    assert torch.equal(moe.moe_mlp_fwd(x.T.contiguous().T, logits.T.contiguous().T, *ws, 2), y)
    assert torch.equal(moe.moe_mlp_fwd(x.reshape(3, 4, K), logits.reshape(3, 4, E), *ws, 2), y.reshape(3, 4, K))
    assert torch.equal(moe.moe_mlp_fwd(x, logits, *ws, 2), y)
    assert moe.moe_mlp_fwd(x[:0], logits[:0], *ws, 2).shape == (0, K)
    for m in (0, 7):
        alone = moe.moe_mlp_fwd(x[m], logits[m], *ws, 2)
        ref, bound = moe64(x[m : m + 1].cpu().double(), logits[m : m + 1].cpu(), 2, True, "silu", dtype, one)
        hold(alone, ref, bound, dtype, 2)
    if bits == 16:  # weights in another order of their elements
        turned = [w.transpose(1, 2).contiguous().transpose(1, 2) for w in ws]
        assert torch.equal(moe.moe_mlp_fwd(x, logits, *turned, 2), y)
    for dt in HALF:  # logits of the activations' type
        low = logits.to(dt)
        assert torch.equal(moe.moe_mlp_fwd(x, low, *ws, 2), moe.moe_mlp_fwd(x, low.float(), *ws, 2))


@gpu
def test_moe_refusals():
    dev, dtype, g = device(), torch.float16, gen(2)
    ws, _ = experts_of(4, 72, 136, 16, 0, dtype, g)
    qs, _ = experts_of(4, 72, 136, 4, 32, dtype, g)
    x, logits = normal((3, 72), 1.0, dtype, g).to(dev), torch.zeros(3, 4, device=dev)
    call = moe.moe_mlp_fwd
    with pytest.raises(TypeError, match="either all"):
        call(x, logits, ws[0], qs[1], ws[2], 2)
    with pytest.raises(TypeError):
        call(x.float(), logits, *ws, 2)
    with pytest.raises(TypeError):
        call(x.bfloat16(), logits, *qs, 2)
    with pytest.raises(ValueError, match="token rows"):
        call(x, logits[:2], *ws, 2)
    with pytest.raises(ValueError, match="W_gate"):
        call(x, torch.zeros(3, 5, device=dev), *ws, 2)
    with pytest.raises(ValueError, match="W_up"):
        call(x, logits, ws[0], ws[1][:, :128], ws[2], 2)
    with pytest.raises(ValueError, match="W_down"):
        call(x, logits, ws[0], ws[1], ws[0], 2)
    with pytest.raises(ValueError, match="codes"):
        call(x, torch.zeros(3, 5, device=dev), *qs, 2)
    for k in (0, 5):
        with pytest.raises(ValueError, match="top_k"):
            call(x, logits, *ws, k)
    with pytest.raises(NotImplementedError):
        call(x, logits, *ws, 2, act_fn="softsign")
    with pytest.raises(RuntimeError, match="no backward"):
        call(x, logits, ws[0].clone().requires_grad_(True), ws[1], ws[2], 2)
    with pytest.raises(RuntimeError, match="traced"):
        torch.jit.trace(lambda t: call(t, logits, *ws, 2), (x,))


# ------------------------------------------------------------------ every kernel that the rules on sizes can choose
# The shapes below were picked from the rules in csrc/experts.hip for 256 CUs: a tile is 16 rows, a block 128 columns of the reduction
# (64 of 16-bit weights).  The references are computed on the GPU, in float64.
def weights64(q):
    """weights_of, looked up where the codes are."""
    codes, scales = q.codes.reshape(-1), q.scales.reshape(-1).double()
    KB, g = q.codes.shape[-5], q.group_size
    r = torch.arange(q.rows, device=codes.device).unsqueeze(1)
    c = torch.arange(q.cols, device=codes.device).unsqueeze(0)
    block = (r // 16) * KB + c // 128
    nibble = torch.where(c % 2 == 0, (c % 8) // 2, 4 + (c % 8) // 2)
    byte = block * 1024 + ((c % 32) // 8) * 256 + (r % 16) * 16 + ((c % 128) // 32) * 4 + nibble // 2
    n = ((codes[byte].int() >> (4 * (nibble % 2))) & 15) - 8
    at = block * (16 * 128 // g) + ((r % 16) // 4) * (4 * 128 // g) + ((c % 128) // g) * 4 + r % 4
    return n.double() * scales[at]


def drawn(shape, std, dtype, g):
    return torch.empty(shape, device=g.device).normal_(0.0, std, generator=g).to(dtype)


def on_gpu(seed):
    return torch.Generator(device=device()).manual_seed(seed)


def hold_on_gpu(got, y, bound, dtype, roundings):
    hold(got, y.cpu(), bound.cpu(), dtype, roundings)


@gpu
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize(
    "M,R,C",
    [
        # up to four tokens: one tile and up to 16, 17 to 127, 128 or more blocks (there split over workgroups too); more tiles
        # than CUs and up to 8 blocks, more
        (1, 1544, 264), (1, 2824, 264), (4, 4360, 136), (3, 16392, 72), (2, 520, 4360), (4, 1160, 4120),
        # 5 to 16: one tile and fewer than 32 blocks, 32 or more; two tiles and up to 8 blocks, more; four tiles
        (7, 1160, 264), (9, 4360, 136), (16, 1000, 4360), (12, 1160, 4360), (5, 1160, 8200),
        # 17 to 64, two, three and four token tiles: a short reduction in no more tiles than CUs, more tiles, a long reduction in parts
        (20, 520, 264), (40, 520, 264), (60, 520, 264), (20, 520, 4360), (40, 520, 4360), (60, 520, 4360), (20, 4360, 264), (40, 4360, 264),
        (60, 4360, 264),
    ],
)
def test_q4_linear_on_every_kernel(M, R, C, group, dtype):
    g = on_gpu(M + R)
    x, q, b = drawn((M, R), 1.0, dtype, g), quant.quantize_q4(drawn((C, R), 0.02, dtype, g), group), drawn((C,), 0.5, dtype, g)
    ref, bound = linear64(x.double(), weights64(q), b.double(), dtype)
    hold_on_gpu(quant.q4_linear_fwd(x, q, b), ref, bound, dtype, 1)


@gpu
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize(
    "M,K,N",
    [
        # up to four tokens and 5 to 16, up to four tiles a CU and more
        (2, 72, 264), (3, 72, 16424), (11, 72, 264), (9, 72, 16424),
        # 17 to 64: no more tiles than CUs, up to 12 blocks and more; up to two a CU, up to 12 blocks and more; more still
        *((M, K, N) for M in (20, 40, 60) for K, N in ((136, 264), (1672, 264), (136, 4360), (1672, 4360), (1672, 8200))),
    ],
)
def test_q4_mlp_on_every_kernel(M, K, N, group, dtype):
    g = on_gpu(M + K)
    x = drawn((M, K), 1.0, dtype, g)
    qs = [quant.quantize_q4(drawn(shape, 0.02, dtype, g), group) for shape in ((N, K), (N, K), (K, N))]
    bs = [drawn((n,), 0.1, dtype, g) for n in (N, N, K)]
    args = [v for pair in zip(qs, bs) for v in pair]
    ref, bound = mlp64(x.double(), *(weights64(v) if isinstance(v, quant.Q4Weight) else v.double() for v in args), "silu", dtype)
    hold_on_gpu(quant.q4_mlp_fwd(x, *args), ref, bound + U[dtype] * ref.abs() + SUB[dtype], dtype, 2)


@gpu
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("bits,group", [(16, 0), (4, 32), (4, 64), (4, 128)])
@pytest.mark.parametrize(
    "M,K,N,E,k",
    [
        # one token, its routing inside gate/up (up to 256 experts) and ahead of it, with few and many blocks of its experts together
        (1, 136, 520, 8, 8), (1, 72, 136, 200, 6), (1, 72, 136, 300, 6), (1, 136, 2056, 16, 16),
        # small batches
        (3, 136, 520, 200, 4), (8, 136, 392, 100, 2), (14, 136, 392, 8, 2), (16, 72, 1032, 32, 8),
        # 17 to 64 tokens: few for each expert (one token tile an entry), more (two)
        (50, 136, 264, 40, 2), (50, 136, 264, 4, 2), (64, 72, 1544, 200, 3), (33, 264, 1544, 6, 3),
        # on either side of 12 tokens for each
        (64, 72, 136, 85, 16), (64, 72, 136, 86, 16),
    ],
)
def test_moe_mlp_on_every_kernel(M, K, N, E, k, bits, group, dtype):
    g = on_gpu(M + K + N)
    x, logits = drawn((M, K), 1.0, dtype, g), drawn((M, E), 1.5, torch.float32, g)
    ws = [drawn(shape, 0.05, dtype, g) for shape in ((E, N, K), (E, N, K), (E, K, N))]
    if bits == 4:
        ws = [quant.quantize_q4(w, group) for w in ws]
        one = lambda e: tuple(weights64(sliced(w, e)).cpu() for w in ws)
    else:
        one = lambda e: tuple(w[e].double().cpu() for w in ws)
    ref, bound = moe64(x.double().cpu(), logits.cpu(), k, True, "silu", dtype, one)
    hold(moe.moe_mlp_fwd(x, logits, *ws, k), ref, bound, dtype, 2)


@gpu
@pytest.mark.parametrize("dtype", HALF)
def test_weights_so_large_that_their_reduction_is_split(dtype):
    """48 MB and more: four tiles a workgroup and three parts (4 bits, 12 tokens), one tile and three parts (16 bits, 9 tokens)."""
    g = on_gpu(1)
    M, R, C = 12, 23432, 4104
    x, q = drawn((M, R), 1.0, dtype, g), quant.quantize_q4(drawn((C, R), 0.02, dtype, g), 128)
    ref, bound = linear64(x.double(), weights64(q), None, dtype)
    y = quant.q4_linear_fwd(x, q)
    hold_on_gpu(y, ref, bound, dtype, 1)
    # the same without a workspace, in one part
    whole = torch.empty_like(y)
    rc = _cabi.lib().gmlp_q4_linear_fwd(x.data_ptr(), q.codes.data_ptr(), q.scales.data_ptr(), None, whole.data_ptr(), M, R, C, 128,
                                        HALF.index(dtype), None, 0, _cabi.stream_ptr(device()))
    assert rc == 0
    hold_on_gpu(whole, ref, bound, dtype, 1)
    M, K, N, E = 9, 1032, 11656, 2
    x, logits = drawn((M, K), 1.0, dtype, g), drawn((M, E), 1.5, torch.float32, g)
    ws = [drawn(shape, 0.02, dtype, g) for shape in ((E, N, K), (E, N, K), (E, K, N))]
    ref, bound = moe64(x.double().cpu(), logits.cpu(), 2, True, "silu", dtype, lambda e: tuple(w[e].double().cpu() for w in ws))
    hold(moe.moe_mlp_fwd(x, logits, *ws, 2), ref, bound, dtype, 2)


@gpu
@pytest.mark.parametrize("bits,E", [(16, 40), (4, 160)])
def test_experts_beyond_4_gib(bits, E):
    """The last expert's weights lie past 32-bit byte offsets; one token and 20, whose plan has entries of 16."""
    dtype, K, N = torch.bfloat16, 4096, 14336
    g = on_gpu(2)
    if bits == 16:
        ws = [drawn(shape, 0.02, dtype, g) for shape in ((E, N, K), (E, N, K), (E, K, N))]
        one = [w[E - 1].double() for w in ws]
    else:
        ws = []
        for rows, cols in ((N, K), (N, K), (K, N)):
            codes = torch.randint(0, 256, (E, rows // 16, cols // 128, 4, 16, 4, 4), generator=g, dtype=torch.uint8, device=g.device)
            scales = (0.002 + 0.003 * torch.rand((E, rows // 16, cols // 128, 4, 2, 4), generator=g, device=g.device)).to(dtype)
            ws.append(quant.Q4Weight(codes, scales, rows, cols, 64))
        one = [weights64(sliced(w, E - 1)) for w in ws]
    for M in (1, 20):
        x, logits = drawn((M, K), 1.0, dtype, g), drawn((M, E), 1.5, torch.float32, g)
        logits[:, E - 1] += 20
        ref, bound = mlp64(x.double(), *(v for w in one for v in (w, None)), "silu", dtype)
        y = moe.moe_mlp_fwd(x, logits, *ws, 1)
        hold_on_gpu(y, ref, bound + (U[dtype] + 1e-6) * ref.abs() + SUB[dtype], dtype, 2)
    del ws, one
    torch.cuda.empty_cache()


@gpu
@pytest.mark.parametrize("M", [1, 2, 30])
@pytest.mark.parametrize("E", [8, 100, 200, 300])
def test_logits_of_every_type(M, E):
    """16-bit logits route as their values in float32 do."""
    dtype, K, N, k = torch.bfloat16, 72, 136, 3
    g = on_gpu(E)
    x, logits = drawn((M, K), 1.0, dtype, g), drawn((M, E), 1.5, torch.float32, g)
    ws = [drawn(shape, 0.05, dtype, g) for shape in ((E, N, K), (E, N, K), (E, K, N))]
    for kind in HALF:
        low = logits.to(kind)
        assert torch.equal(moe.moe_mlp_fwd(x, low, *ws, k), moe.moe_mlp_fwd(x, low.float(), *ws, k))


@gpu
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("M,K,E", [(2, 4104, 8), (8, 2056, 64), (12, 4104, 256), (20, 1160, 12), (40, 1160, 8), (60, 4104, 128)])
def test_moe_logits_on_every_kernel(M, K, E, dtype):
    g = on_gpu(M + K)
    x, w = drawn((M, K), 1.0, dtype, g), drawn((E, K), 0.1, dtype, g)
    y, mass = x.double() @ w.double().T, x.double().abs() @ w.double().abs().T
    assert ((moe.moe_logits(x, w).double() - y).abs() <= (K + 16) * 2.0**-23 * mass).all()


# ------------------------------------------------------------------ streams and graphs
def _calls(bits):
    dev, dtype, g = device(), torch.bfloat16, gen(4)
    E, K, N, M = 16, 264, 392, 5
    ws, _ = experts_of(E, K, N, bits, 64, dtype, g)
    x, logits = normal((M, K), 1.0, dtype, g).to(dev), normal((M, E), 1.5, torch.float32, g).to(dev)
    if bits == 16:
        return x, logits, lambda: [moe.moe_mlp_fwd(x, logits, *ws, 3), *moe.moe_route(logits, 3)]
    one = [sliced(q, 2) for q in ws]
    return x, logits, lambda: [moe.moe_mlp_fwd(x, logits, *ws, 3), quant.q4_mlp_fwd(x, one[0], None, one[1], None, one[2], None),
                               quant.q4_linear_fwd(x, one[0])]


@gpu
@pytest.mark.parametrize("bits", [16, 4])
def test_operators_run_on_the_current_stream(bits):
    x, logits, call = _calls(bits)
    ref = call()
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        held = x.clone()
        x.fill_(math.nan)
        x.copy_(held)  # on the side stream: a call on another stream would read NaN, or race
        out = call()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(ref, out))


@gpu
@pytest.mark.parametrize("bits", [16, 4])
def test_operators_replay_in_a_graph(bits):
    x, logits, call = _calls(bits)
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    g = gen(8)
    for _ in range(4):  # other inputs and another routing each time
        x.copy_(normal(x.shape, 1.0, x.dtype, g))
        logits.copy_(normal(logits.shape, 1.5, logits.dtype, g))
        graph.replay()
        torch.cuda.synchronize()
        ref = call()
        assert all(torch.equal(a, b) for a, b in zip(ref, out))
        torch.cuda.synchronize()


# ------------------------------------------------------------------ modules
def test_modules_on_the_cpu():
    from triton_gated_mlp import FusedGatedMLP, GatedMoE, Q4GatedMLP

    m = GatedMoE(64, 72, 12, 3, hidden_act="gelu")
    assert {n: tuple(p.shape) for n, p in m.named_parameters()} == {
        "gate_proj": (12, 72, 64), "up_proj": (12, 72, 64), "down_proj": (12, 64, 72), "router.weight": (12, 64)}
    assert not m.quantized and "top_k=3" in repr(m)
    for bad in (0, 13):
        with pytest.raises(ValueError, match="top_k"):
            GatedMoE(64, 72, 12, bad)
    with pytest.raises(KeyError):
        GatedMoE(64, 72, 12, 3, hidden_act="softsign")
    with pytest.raises(RuntimeError, match="AMD GPU"):
        with torch.no_grad():
            m(torch.zeros(2, 64))
    with pytest.raises(RuntimeError, match="AMD GPU"):
        Q4GatedMLP.from_float(FusedGatedMLP(64, 72).half())
    # the batch from which experts run one by one, by their size
    assert GatedMoE(8, 8, 2, 1).long_batch() > 10**7
    with torch.device("meta"):
        assert GatedMoE(4096, 14336, 8, 2).long_batch() == 113 and GatedMoE(8192, 28672, 8, 2).long_batch() == 65


@gpu
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("M,K,E", [(1, 8, 4), (1, 2048, 64), (5, 264, 60), (16, 136, 8), (33, 1000, 128), (64, 264, 12), (100, 136, 16)])
def test_moe_logits(M, K, E, dtype):
    dev, g = device(), gen(M + K)
    x, w = normal((M, K), 1.0, dtype, g), normal((E, K), 0.1, dtype, g)
    out = moe.moe_logits(x.to(dev), w.to(dev))
    assert out.dtype == torch.float32
    y, mass = x.double() @ w.double().T, x.double().abs() @ w.double().abs().T
    assert ((out.cpu().double() - y).abs() <= (K + 16) * 2.0**-23 * mass).all()
    assert moe.moe_logits(x.to(dev)[:0], w.to(dev)).shape == (0, E)


@gpu
def test_moe_logits_refusals():
    dev = device()
    x, w = torch.zeros(2, 64, dtype=torch.float16, device=dev), torch.zeros(8, 64, dtype=torch.float16, device=dev)
    with pytest.raises(ValueError, match="W_router"):
        moe.moe_logits(x, w[:, :56])
    with pytest.raises(NotImplementedError):
        moe.moe_logits(x, w[:6])
    with pytest.raises(TypeError):
        moe.moe_logits(x, w.float())
    with pytest.raises(RuntimeError, match="no backward"):
        moe.moe_logits(x, w.clone().requires_grad_(True))


@gpu
@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("E,router", [(12, torch.bfloat16), (6, torch.float32)])
def test_gated_moe_module(E, router, bits):
    """Few tokens, the same tokens through the experts one by one, and a saved and loaded copy."""
    from triton_gated_mlp import GatedMoE

    dev, dtype, K, N, k = device(), torch.bfloat16, 136, 264, 2
    torch.manual_seed(3)
    m = GatedMoE(K, N, E, k, hidden_act="gelu").to(dev, dtype)
    m.router.to(router)
    x = torch.randn(2, 9, K, device=dev).to(dtype)
    with pytest.raises(RuntimeError, match="no backward"):
        m(x)
    with torch.no_grad():
        if bits == 4:
            m.quantize_(64)
            one = lambda e: tuple(weights_of(p.of(e)) for p in (m.gate_proj, m.up_proj, m.down_proj))
        else:
            one = lambda e: tuple(p[e].cpu().double() for p in (m.gate_proj, m.up_proj, m.down_proj))
        assert m.quantized == (bits == 4)
        y = m(x)
        rows = x.reshape(-1, K)
        logits = m.route_logits(rows)
        assert torch.allclose(logits.cpu().double(), rows.cpu().double() @ m.router.weight.cpu().double().T, atol=1e-4, rtol=0)
        ref, bound = moe64(rows.cpu().double(), logits.cpu(), k, True, "gelu", dtype, one)
        hold(y, ref, bound, dtype, 2)
        # each expert's output is rounded as well: three roundings, u in the mean square, and the weights' 1e-6
        out = m._one_by_one(rows, logits).cpu().double()
        assert ((out - ref).norm() / ref.norm()).item() <= 1.02 * U[dtype]
        m.long_batch = lambda: 1
        assert torch.equal(m(x).cpu().double().reshape(out.shape), out)
        other = GatedMoE(K, N, E, k, hidden_act="gelu").to(dev, dtype)
        other.router.to(router)
        if bits == 4:
            other.quantize_(64)
        other.load_state_dict(m.state_dict())
        assert torch.equal(other(x), y)


@gpu
@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("E,router", [(8, None), (6, None), (8, torch.float32)])
def test_gated_moe_module_without_rows(E, router, bits):
    from triton_gated_mlp import GatedMoE

    m = GatedMoE(64, 72, E, 2).to(device(), torch.float16)
    if router is not None:
        m.router.to(router)
    with torch.no_grad():
        m = m.quantize_(32) if bits == 4 else m
        for shape in ((0, 64), (2, 0, 64)):
            y = m(torch.zeros(shape, dtype=torch.float16, device=device()))
            assert y.shape == shape and y.dtype == torch.float16


def _on_four_bits(E, K, N, dtype):
    """A GatedMoE as quantize_ leaves it, without a GPU."""
    from triton_gated_mlp import GatedMoE
    from triton_gated_mlp.experts import _Q4Buffers

    m = GatedMoE(K, N, E, 2).to(dtype)
    for name, rows, cols in (("gate_proj", N, K), ("up_proj", N, K), ("down_proj", K, N)):
        tiles, blocks = -(-rows // 16), -(-cols // 128)
        codes = torch.randint(0, 256, (E, tiles, blocks, 4, 16, 4, 4), generator=gen(rows), dtype=torch.uint8)
        scales = torch.full((E, tiles, blocks, 4, 2, 4), 0.01, dtype=dtype)
        delattr(m, name)
        setattr(m, name, _Q4Buffers(quant.Q4Weight(codes, scales, rows, cols, 64)))
    return m


@pytest.mark.parametrize(
    "K,N,E,bits,streamed,own",
    [
        # a number of rows at which streaming measured the faster way, and one at which passes of their own did
        (4096, 14336, 8, 16, 96, 192), (2048, 5632, 8, 16, 256, 512), (2048, 1024, 64, 16, 1024, 3072), (1024, 2816, 16, 16, 768, 1536),
        (4096, 14336, 8, 4, 512, 1024), (2048, 5632, 8, 4, 512, 1536), (2048, 1024, 64, 4, 2048, 6144), (1024, 2816, 16, 4, 1536, 3072),
        (8192, 28672, 4, 4, 256, 512),
    ],
)
def test_the_way_of_a_batch_goes_by_its_experts_size_and_type(K, N, E, bits, streamed, own):
    from triton_gated_mlp import GatedMoE
    from triton_gated_mlp.experts import _Q4Buffers

    with torch.device("meta"):
        m = GatedMoE(K, N, E, 2)
        if bits == 4:
            for name, rows, cols in (("gate_proj", N, K), ("up_proj", N, K), ("down_proj", K, N)):
                delattr(m, name)
                setattr(m, name, _Q4Buffers(quant.Q4Weight(torch.empty(1, dtype=torch.uint8), torch.empty(1), rows, cols, 128)))
    assert streamed < m.long_batch() <= own


# (70 rows: the float32 GEMM's logits; 3 rows: that of a float32 router, of a number of experts that is no multiple of 4, and moe_logits)
ROUTERS = [(70, 8, None), (3, 8, torch.float32), (3, 6, None), (3, 8, None)]


@pytest.mark.parametrize("rows,E,router", ROUTERS)
def test_layers_of_four_bit_experts_refuse_what_autograd_would_record(rows, E, router):
    """The router's weight and x are the tensors that are left to differentiate for."""
    import torch.autograd.forward_ad as fw

    m = _on_four_bits(E, 64, 72, torch.float16)
    if router is not None:
        m.router.to(router)
    x = torch.zeros(rows, 64, dtype=torch.float16)
    for one_by_one in (False, True):
        if one_by_one:
            m.long_batch = lambda: 1
        m.router.requires_grad_(True)
        with pytest.raises(RuntimeError, match="no backward"):
            m(x)
        with pytest.raises(RuntimeError, match="no backward"):
            m.route_logits(x)
        m.router.requires_grad_(False)
        with pytest.raises(RuntimeError, match="no backward"):
            m(x.clone().requires_grad_(True))
        with fw.dual_level(), torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
            m(fw.make_dual(x, x))
        with torch.no_grad(), pytest.raises(RuntimeError, match="functorch"):
            torch.vmap(m)(x[None])
        with pytest.raises(RuntimeError, match="AMD GPU"):  # nothing to record: it gets as far as the kernels
            m(x)


@gpu
@pytest.mark.parametrize("rows,E,router", ROUTERS)
def test_layers_of_four_bit_experts_run_where_autograd_records_nothing(rows, E, router):
    m = _on_four_bits(E, 64, 72, torch.float16)
    if router is not None:
        m.router.to(router)
    m = m.to(device())
    x = normal((rows, 64), 1.0, torch.float16, gen(rows)).to(device())
    with pytest.raises(RuntimeError, match="no backward"):
        m(x)
    with torch.no_grad():
        y = m(x)
    m.router.requires_grad_(False)
    assert torch.equal(m(x), y) and not m(x).requires_grad


@gpu
@pytest.mark.parametrize("bits", [16, 4])
def test_masked_experts_of_a_long_batch_are_not_run(bits, monkeypatch):
    """As the streaming kernels have it: an expert that every token's mask leaves out, rows whose mask leaves fewer than top_k
    and a row whose mask leaves nothing."""
    from triton_gated_mlp import GatedMoE, experts

    dev, dtype, E, K, N, M, k = device(), torch.bfloat16, 6, 72, 136, 80, 3
    torch.manual_seed(1)
    g = gen(1)
    m = GatedMoE(K, N, E, k).to(dev, dtype)
    x, logits = normal((M, K), 1.0, dtype, g), normal((M, E), 1.5, torch.float32, g)
    logits[:, 1:] = logits[:, 1:].masked_fill(torch.rand((M, E - 1), generator=g) < 0.6, -math.inf)
    logits[:, 4] = -math.inf
    logits[2] = -math.inf
    ran = []
    for module, name in ((experts._fwd, "mlp_fwd"), (experts._quant, "q4_mlp_fwd")):
        def recorded(rows, *rest, call=getattr(module, name), **named):
            ran.append(rows.shape[0])
            return call(rows, *rest, **named)
        monkeypatch.setattr(module, name, recorded)
    with torch.no_grad():
        if bits == 4:
            m.quantize_(32)
            one = lambda e: tuple(weights_of(p.of(e)) for p in (m.gate_proj, m.up_proj, m.down_proj))
        else:
            one = lambda e: tuple(p[e].cpu().double() for p in (m.gate_proj, m.up_proj, m.down_proj))
        out = m._one_by_one(x.to(dev), logits.to(dev)).cpu().double()
        w, experts_of_rows = route64(logits, k, True)
        assert ran == [int(((experts_of_rows == e) & (w > 0)).sum()) for e in range(E) if e != 4]
        ref, _ = moe64(x.double(), logits, k, True, "silu", dtype, one)
        assert (out[2] == 0).all() and ((out - ref).norm() / ref.norm()).item() <= 1.02 * U[dtype]
        assert (m._one_by_one(x.to(dev), torch.full((M, E), -math.inf, device=dev)) == 0).all()
        assert len(ran) == E - 1
        # a token whose logits are not finite, in the way softmax has it, beside rows that stay as they are
        logits[7, 1] = math.nan
        wrong = m._one_by_one(x.to(dev), logits.to(dev)).cpu().double()
        keep = torch.arange(M) != 7
        assert ((wrong - ref)[keep].norm() / ref[keep].norm()).item() <= 1.02 * U[dtype] and torch.isnan(wrong[7]).all()


@gpu
@pytest.mark.parametrize("rows", [3, 70])
def test_q4_gated_mlp_module(rows):
    from triton_gated_mlp import FusedGatedMLP, Q4GatedMLP

    dev, dtype = device(), torch.float16
    torch.manual_seed(5)
    mlp = FusedGatedMLP(136, 264, bias=True, hidden_act="relu").to(dev, dtype).eval()
    q = Q4GatedMLP.from_float(mlp, 32)
    x = torch.randn(rows, 136, device=dev).to(dtype)
    with torch.no_grad():
        y = q(x)
    ws = [weights_of(p.weight()) for p in (q.gate_proj, q.up_proj, q.down_proj)]
    if rows > 64:
        ws = [w.to(dtype).double() for w in ws]
    bs = [layer.bias.detach().cpu().double() for layer in (mlp.gate_proj, mlp.up_proj, mlp.down_proj)]
    ref, bound = mlp64(x.cpu().double(), ws[0], bs[0], ws[1], bs[1], ws[2], bs[2], "relu", dtype)
    hold(y, ref, bound + U[dtype] * ref.abs() + SUB[dtype], dtype, 2)
    assert y.requires_grad is False and len(list(q.parameters())) == 0
    q2 = Q4GatedMLP.from_float(FusedGatedMLP(136, 264, bias=True, hidden_act="relu").to(dev, dtype), 32)
    q2.load_state_dict(q.state_dict())
    assert torch.equal(q2(x), y)
    # within the quantisation's error of the module it came from: at most half a step of 1/7 of a group's largest weight
    with torch.no_grad():
        assert ((mlp(x) - y).norm() / mlp(x).norm()).item() < 0.25


@gpu
@pytest.mark.parametrize("bits", ["4", "16"])
def test_the_decode_example_runs(bits):
    from triton_gated_mlp import decode_example

    us = decode_example.main(["--tokens", "2", "--layers", "2", "--hidden", "1024", "--intermediate", "1408", "--expert", "512",
                              "--experts", "16", "--top-k", "4", "--bits", bits, "--steps", "5"])
    assert us > 0
