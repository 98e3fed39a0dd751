"""Routing that is trained: weights, experts, counts, the balance loss and the gradient of the logits.

Tolerances, in fp32 with e = 2^-24.  A probability is an exponential (2 units of its argument's rounding, |l - max| <= 20 here: 22 e) over
a sum of E of them, which adds E e at most: (E + 64) e of its size is never reached.  The loss is a mean of those, sums of
at most 2^10 terms a lane ahead of 64 bits: (E + 2200) e of it.  A gradient is a difference of two such terms of
magnitude p (slope + mean) |d_loss| and w (|dw| + mixed): (E + 128) e of their sum, and the rounding of its type.  (Where it is
0, of an expert that was not chosen, automatic differentiation in 64 bits leaves what its own roundings of 2^-53 leave of the row's
largest terms: a few hundred of them are 2^-44.)
"""

import ctypes
import math

import pytest
import torch

from test_experts import device, gen
from triton_gated_mlp import FusedGatedMLP, GatedMoE, _cabi
from triton_gated_mlp.ops import moe

gpu = pytest.mark.gpu
E24 = 2.0**-24
ROUND = {torch.float32: 2.0**-24, torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}
SMALL = {torch.float32: 2.0**-126, torch.float16: 2.0**-25, torch.bfloat16: 2.0**-126}


# ------------------------------------------------------------------ plain implementation in 64 bits
def choose(logits, k):
    """[rows, k]: the largest that is left, the lowest number among equals, one after the other."""
    picks = []
    for row in logits.tolist():
        left = list(range(len(row)))
        mine = []
        for _ in range(k):
            best = max(left, key=lambda e: (row[e], -e))
            mine.append(best)
            left.remove(best)
        picks.append(mine)
    return torch.tensor(picks, dtype=torch.int64).reshape(len(picks), k)


def balance64(logits, experts, normalize, mask):
    """weights, counts, loss, differentiable in the float64 logits; `experts` fixed."""
    M, E = logits.shape
    none = (logits == -math.inf).all(1, keepdim=True)
    safe = torch.where(none, 0.0, logits)
    p = torch.where(none, 0.0, torch.softmax(safe, 1))
    w = p.gather(1, experts)
    if normalize:
        w = torch.where(none, 0.0, w / torch.where(none, 1.0, w.sum(1, keepdim=True)))
    there = ~none[:, 0] if mask is None else ~none[:, 0] & mask
    counted = there[:, None] & (logits.detach().gather(1, experts) > -math.inf)
    counts = torch.zeros(E, dtype=torch.int64).index_add_(0, experts.reshape(-1), counted.reshape(-1).long())
    if int(there.sum()) == 0:
        return w, counts, (logits * 0).nan_to_num().sum() * 0
    share = counts.double() / counts.sum()
    return w, counts, E * (share * p[there].mean(0)).sum()


def case(M, E, k, dtype, seed, masked=0, padded=False):
    g = gen(seed)
    logits = (torch.randn((M, E), generator=g) + 0.7 * torch.randn((1, E), generator=g)).to(dtype)
    if masked:
        off = torch.rand((M, E), generator=g).argsort(1)[:, :masked]
        logits.scatter_(1, off, -math.inf)
    mask = torch.rand(M, generator=g) < 0.6 if padded else None
    return logits, mask, 0.1 * torch.randn((M, k), generator=g), torch.tensor(0.37)


def check(logits, mask, dw, dl, k, normalize):
    dtype, E = logits.dtype, logits.shape[1]
    x = logits.to(device()).requires_grad_()
    got = moe.moe_route_balanced(x, k, normalize, None if mask is None else mask.to(device()))
    route = moe.moe_route(x.detach(), k, normalize)
    assert torch.equal(got.experts, route.experts)
    if E <= 256:  # (beyond, the sums over a token's experts have another order)
        assert torch.equal(got.weights.detach(), route.weights)
    experts = got.experts.cpu()
    ref = logits.double().requires_grad_()
    w, counts, loss = balance64(ref, experts, normalize, mask)
    assert torch.equal(got.counts.cpu(), counts) and got.counts.dtype == torch.int64
    assert got.loss.shape == () and got.loss.dtype == torch.float32
    assert abs(got.loss.item() - loss.item()) <= (E + 2200) * E24 * abs(loss.item())
    assert ((got.weights.detach().cpu().double() - w.detach()).abs() <= (E + 64) * E24 * w.detach()).all()
    p = torch.softmax(logits.double(), 1).nan_to_num()
    share = counts.double() / max(1, int(counts.sum()))
    for use_w, use_l in ((True, True), (True, False), (False, True)):
        outs = ([got.weights] if use_w else []) + ([got.loss] if use_l else [])
        grads = ([dw.to(device())] if use_w else []) + ([dl.to(device())] if use_l else [])
        (d,) = torch.autograd.grad(outs, x, grads, retain_graph=True)
        assert d.dtype == dtype and d.shape == x.shape
        outs64 = ([w] if use_w else []) + ([loss] if use_l else [])
        (r,) = torch.autograd.grad(outs64, ref, [t.double() for t in (([dw] if use_w else []) + ([dl] if use_l else []))], retain_graph=True)
        r = r.nan_to_num()
        there = torch.ones(len(logits), dtype=torch.bool) if mask is None else mask
        T = max(1, int((there & (logits > -math.inf).any(1)).sum()))
        size = torch.zeros_like(p)
        if use_l:
            size += p * (share + (share * p).sum(1, keepdim=True)) * dl.double() * E / T
        if use_w:
            mixed = (w.detach() * dw.double().abs()).sum(1, keepdim=True)
            size.scatter_add_(1, experts, w.detach() * (dw.double().abs() + mixed))
            size += 0 if normalize else p * mixed
        off = (d.cpu().double() - r).abs()
        bound = (E + 128) * E24 * size + ROUND[dtype] * r.abs() * 1.01 + SMALL[dtype] + 2.0**-44 * size.amax(1, keepdim=True)
        assert (off <= bound).all(), f"off by {(off / bound).max().item():.3f} of the bound"
    return got


# ------------------------------------------------------------------ without a GPU
def test_refusals_of_the_c_interface():
    lib = _cabi.lib()
    raw = ctypes.create_string_buffer(64 * 1024)
    a = (ctypes.addressof(raw) + 63) & ~63
    need = lib.gmlp_moe_balance_workspace_bytes(4, 8)
    assert need > 0 and lib.gmlp_moe_balance_workspace_bytes(0, 8) == 0 and lib.gmlp_moe_balance_workspace_bytes(4, 513) == 0

    def fwd(logits=a, mask=None, w=a, e=a, c=a, loss=a, slope=a, M=4, E=8, k=2, dtype=2, ws=a, n=need):
        return lib.gmlp_moe_balance_fwd(logits, mask, w, e, c, loss, slope, M, E, k, 1, dtype, ws, n, None)

    for name in ("logits", "w", "e", "c", "loss", "slope", "ws"):
        assert fwd(**{name: None}) == -1 and "NULL" in lib.gmlp_last_error().decode()
    assert fwd(dtype=3) == -1 and fwd(M=0) == -2 and fwd(E=513) == -2 and fwd(k=9) == -2 and fwd(k=0) == -2 and fwd(E=64, k=17) == -2
    assert fwd(n=need - 1) == -1 and "workspace" in lib.gmlp_last_error().decode() and fwd(ws=a + 8) == -3

    def bwd(logits=a, w=a, e=a, slope=a, dw=a, dl=a, d=a, M=4, E=8, k=2, dtype=2):
        return lib.gmlp_moe_balance_bwd(logits, None, w, e, slope, dw, dl, d, M, E, k, 1, dtype, None)

    for name in ("logits", "w", "e", "slope", "d"):
        assert bwd(**{name: None}) == -1
    assert bwd(dtype=3) == -1 and bwd(M=0) == -2 and bwd(E=513) == -2 and bwd(k=9) == -2


def test_cpu_tensors_and_transforms_are_refused():
    import torch.autograd.forward_ad as fw

    x = torch.zeros(3, 8)
    with pytest.raises(RuntimeError, match="AMD GPU"):
        moe.moe_route_balanced(x, 2)
    with fw.dual_level(), torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
        moe.moe_route_balanced(fw.make_dual(x, x), 2)
    with pytest.raises(RuntimeError, match="functorch"):
        torch.vmap(lambda t: moe.moe_route_balanced(t, 2).loss)(x[None])


def test_the_plain_gradient_against_differences():
    """The oracle's own: central differences of weights and loss with the choices and the counts held."""
    logits, mask, dw, dl = case(5, 7, 3, torch.float64, 3, masked=2, padded=True)
    experts = choose(logits, 3)
    for normalize in (True, False):
        x = logits.clone().requires_grad_()
        value = lambda t: (lambda w, c, l: (w * dw).sum() + l * dl)(*balance64(t, experts, normalize, mask))
        (d,) = torch.autograd.grad(value(x), x)
        for i in range(5):
            for j in range(7):
                if logits[i, j] == -math.inf:
                    assert d[i, j] == 0 or d[i, j].isnan()
                    continue
                up, down = logits.clone(), logits.clone()
                up[i, j] += 1e-6
                down[i, j] -= 1e-6
                assert abs((value(up) - value(down)).item() / 2e-6 - d[i, j].item()) < 1e-8


# ------------------------------------------------------------------ on the GPU
@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("normalize", [True, False])
@pytest.mark.parametrize(
    "M,E,k,masked,padded",
    [
        (1, 1, 1, 0, False), (1, 8, 2, 0, False), (3, 16, 16, 0, True), (64, 8, 2, 3, True), (17, 60, 4, 0, False), (100, 65, 6, 30, True),
        (33, 128, 8, 0, True), (5, 130, 3, 129, False), (70, 256, 8, 100, False), (40, 300, 2, 0, True), (19, 512, 16, 200, True),
        (4099, 12, 2, 4, True), (6000, 64, 8, 0, False),
    ],
)
def test_balanced_routing(M, E, k, masked, padded, normalize, dtype):
    check(*case(M, E, k, dtype, M + E, masked, padded), k, normalize)


@gpu
@pytest.mark.parametrize("E", [8, 70, 300])
def test_ties_and_tokens_that_do_not_count(E):
    k = 4
    logits, mask, dw, dl = case(40, E, k, torch.float32, E, padded=True)
    logits[3] = 0.5  # ties: the lowest numbers
    logits[4] = -math.inf  # nothing is available
    logits[5, 2:] = -math.inf  # fewer than it chooses
    logits[6, 1], logits[6, 2] = 0.0, -0.0
    logits[7] = torch.finfo(torch.float32).min
    mask[3:7] = True
    got = check(logits, mask, dw, dl, k, True)
    assert got.experts[3].tolist() == list(range(k)) and (got.weights[4] == 0).all() and (got.weights[5, 2:] == 0).all()
    check(logits, None, dw, dl, k, False)
    # nobody counts
    for x, m in ((logits, torch.zeros(40, dtype=torch.bool)), (torch.full((40, E), -math.inf), None)):
        x = x.to(device()).requires_grad_()
        got = moe.moe_route_balanced(x, k, True, None if m is None else m.to(device()))
        assert got.loss.item() == 0 and (got.counts == 0).all()
        (d,) = torch.autograd.grad(got.loss, x)
        assert (d == 0).all()


@gpu
def test_what_is_not_finite():
    logits, _, dw, dl = case(20, 16, 2, torch.float32, 1)
    logits[3, 4], logits[9, 1] = math.nan, math.inf
    x = logits.to(device()).requires_grad_()
    got = moe.moe_route_balanced(x, 2)
    assert got.loss.isnan() and got.weights[3].isnan().all() and got.weights[9].isnan().all()
    (d,) = torch.autograd.grad(got.weights, x, dw.to(device()))
    rest = torch.ones(20, dtype=torch.bool, device=x.device)
    rest[[3, 9]] = False
    assert d[3].isnan().any() and d[rest].isfinite().all()
    # left out, they are in neither counts nor loss
    got = moe.moe_route_balanced(x, 2, token_mask=rest)
    good = moe.moe_route_balanced(x.detach()[rest], 2)
    assert torch.equal(got.counts, good.counts) and abs(got.loss.item() - good.loss.item()) < 1e-5
    (d,) = torch.autograd.grad(got.loss, x)
    assert d[rest].isfinite().all() and (d[~rest] == 0).all()


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("normalize", [True, False])
@pytest.mark.parametrize("E", [6, 40, 300])
def test_what_is_not_finite_in_a_token_left_out_reaches_no_gradient_of_the_loss(E, normalize, dtype):
    """A token that is in neither counts nor loss has a gradient of 0 for it, whatever its logits hold, and the others' are as without it."""
    logits, _, _, dl = case(20, E, 2, dtype, E)
    logits[3, 4], logits[9, 1], logits[12] = math.nan, math.inf, math.nan
    rest = torch.ones(20, dtype=torch.bool, device=device())
    rest[[3, 9, 12]] = False
    x = logits.to(device()).requires_grad_()
    (d,) = torch.autograd.grad(moe.moe_route_balanced(x, 2, normalize, token_mask=rest).loss, x, dl.to(device()))
    good = logits.to(device())[rest].requires_grad_()
    (g,) = torch.autograd.grad(moe.moe_route_balanced(good, 2, normalize).loss, good, dl.to(device()))
    # (the same counts in both, and nothing else of the other tokens is in a token's gradient)
    assert (d[~rest] == 0).all() and torch.equal(d[rest], g)


@gpu
def test_even_routing_has_loss_one():
    for M, E in ((64, 8), (4096, 128)):
        x = torch.full((M, E), -30.0)
        x[torch.arange(M), torch.arange(M) % E] = 30.0
        assert abs(moe.moe_route_balanced(x.to(device()), 1).loss.item() - 1) < 1e-5
        x = torch.full((M, E), -30.0)
        x[:, 3] = 30.0
        got = moe.moe_route_balanced(x.to(device()), 1)
        assert abs(got.loss.item() - E) < 1e-4 * E and got.counts[3] == M


@gpu
def test_shapes_strides_streams_and_repeats():
    g = gen(5)
    x = torch.randn((3, 7, 20), generator=g).to(device())
    mask = (torch.rand((3, 7), generator=g) < 0.5).to(device())
    view = x[..., 3:17].detach().requires_grad_()
    got = moe.moe_route_balanced(view, 3, token_mask=mask)
    assert got.weights.shape == got.experts.shape == (3, 7, 3) and got.counts.shape == (14,)
    flat = x[..., 3:17].reshape(21, 14).clone().requires_grad_()
    same = moe.moe_route_balanced(flat, 3, token_mask=mask.reshape(21))
    assert torch.equal(got.weights.reshape(21, 3), same.weights) and torch.equal(got.loss, same.loss) and torch.equal(got.counts, same.counts)
    dw = torch.randn((3, 7, 3), generator=g).to(device())
    (d,) = torch.autograd.grad((got.weights, got.loss), view, (dw, torch.ones((), device=x.device)))
    (f,) = torch.autograd.grad((same.weights, same.loss), flat, (dw.reshape(21, 3), torch.ones((), device=x.device)))
    assert d.shape == view.shape and torch.equal(d.reshape(21, 14), f)
    # a gradient that is broadcast, and one that is transposed
    (d,) = torch.autograd.grad(moe.moe_route_balanced(flat, 3).weights.sum(), flat)
    assert d.abs().max() < 1e-6  # normalised weights sum to 1
    strided = dw.reshape(21, 3).T.contiguous().T
    (d,) = torch.autograd.grad(moe.moe_route_balanced(flat, 3, token_mask=mask.reshape(21)).weights, flat, strided)
    (f,) = torch.autograd.grad(moe.moe_route_balanced(flat, 3, token_mask=mask.reshape(21)).weights, flat, dw.reshape(21, 3))
    assert torch.equal(d, f)
    # one token, no leading dimension; no tokens
    one = moe.moe_route_balanced(x[0, 0], 2, token_mask=torch.ones((), dtype=torch.bool, device=x.device))
    assert one.weights.shape == (2,) and one.counts.sum() == 2
    none = x[:0].detach().requires_grad_()
    got = moe.moe_route_balanced(none, 2)
    assert got.weights.shape == (0, 7, 2) and got.loss.item() == 0 and (got.counts == 0).all()
    (d,) = torch.autograd.grad(got.loss, none)
    assert d.shape == none.shape
    # another stream; bit for bit the same again
    big = torch.randn((5000, 64), generator=g).to(device())
    first = moe.moe_route_balanced(big, 4)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = moe.moe_route_balanced(big, 4)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(first, second))


@gpu
@pytest.mark.parametrize("M,E,k", [(1, 3, 2), (64, 8, 2), (3000, 60, 4), (20000, 300, 3)])
def test_what_a_step_keeps_for_its_gradient(M, E, k):
    """Logits, mask, weights, experts and a slope for each expert, in tensors that hold nothing else."""
    x = torch.randn((M, E), device=device()).requires_grad_()
    mask = torch.ones(M, dtype=torch.bool, device=x.device)
    kept = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: kept.append(t) or t, lambda t: t):
        got = moe.moe_route_balanced(x, k, token_mask=mask)
    assert sorted(tuple(t.shape) for t in kept) == sorted([(M, E), (M,), (M, k), (M, k), (E,)])
    assert all(t.untyped_storage().nbytes() == t.numel() * t.element_size() for t in kept)
    del kept
    torch.autograd.grad((got.weights.sum(), got.loss), x)


@gpu
def test_what_autograd_is_refused():
    x = torch.randn(6, 8, device=device()).requires_grad_()
    got = moe.moe_route_balanced(x, 2)
    assert not got.experts.requires_grad and not got.counts.requires_grad and got.weights.requires_grad and got.loss.requires_grad
    (d,) = torch.autograd.grad(got.loss, x, create_graph=True)
    with pytest.raises(RuntimeError, match="no second derivative"):
        torch.autograd.grad(d.sum(), x)
    got = moe.moe_route_balanced(x, 2)
    with torch.no_grad():
        got.weights.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        got.loss.backward()
    with torch.no_grad():
        assert not moe.moe_route_balanced(x, 2).loss.requires_grad
    for call, error in [
        (lambda: moe.moe_route_balanced(x.double(), 2), TypeError), (lambda: moe.moe_route_balanced(x, 9), ValueError),
        (lambda: moe.moe_route_balanced(x, 0), ValueError), (lambda: moe.moe_route_balanced(x, 2, token_mask=torch.ones(5, dtype=torch.bool, device=x.device)), ValueError),
        (lambda: moe.moe_route_balanced(x, 2, token_mask=torch.ones(6, device=x.device)), TypeError),
        (lambda: moe.moe_route_balanced(x, 2, token_mask=torch.ones(6, dtype=torch.bool)), RuntimeError),
        (lambda: moe.moe_route_balanced(torch.zeros(2, 513, device=x.device), 2), NotImplementedError),
        (lambda: moe.moe_route_balanced(torch.zeros(2, 64, device=x.device), 17), NotImplementedError),
    ]:
        with pytest.raises(error):
            call()


@gpu
def test_a_training_step_under_capture_is_refused_and_inference_replays(monkeypatch):
    x = torch.randn(50, 8, device=device())
    mask = torch.ones(50, dtype=torch.bool, device=device())
    with monkeypatch.context() as m:
        m.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
        with pytest.raises(RuntimeError, match="autograd graph"):
            moe.moe_route_balanced(x.clone().requires_grad_(), 2)
    moe.moe_route_balanced(x, 2, token_mask=mask)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = moe.moe_route_balanced(x, 2, token_mask=mask)
    for seed in range(4):
        x.copy_(torch.randn((50, 8), generator=gen(seed)))
        mask.copy_(torch.rand(50, generator=gen(9 + seed)) < 0.5)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, moe.moe_route_balanced(x, 2, token_mask=mask)))


@gpu
def test_a_router_and_its_experts_are_trained_and_served_in_8_bits():
    """One step of a layer of FusedGatedMLP experts: gradients against the same layer in float64; then the experts serve in 8 bits."""
    K, N, E, k, M = 64, 128, 4, 2, 96
    torch.manual_seed(1)
    dtype = torch.bfloat16
    router = torch.nn.Linear(K, E, bias=False).to(device())
    experts = [FusedGatedMLP(K, N, bias=False).to(device()).to(dtype) for _ in range(E)]
    x = torch.randn(M, K, device=device()).to(dtype)
    target = torch.randn(M, K, device=device())
    routing = moe.moe_route_balanced(router(x.float()), k)
    y = torch.zeros(M, K, device=device())
    for e, expert in enumerate(experts):
        t, j = torch.nonzero(routing.experts == e, as_tuple=True)
        y = y.index_add(0, t, expert(x[t]).float() * routing.weights[t, j, None])
    loss = (y * target).mean() + 0.1 * routing.loss
    loss.backward()
    assert routing.counts.sum() == M * k and torch.equal(routing.counts, torch.bincount(routing.experts.reshape(-1), minlength=E))
    # the same in float64
    w64 = router.weight.detach().double().cpu().requires_grad_()
    x64 = x.double().cpu()
    w, counts, balance = balance64(x64 @ w64.T, routing.experts.cpu(), True, None)
    y64 = torch.zeros(M, K, dtype=torch.float64)
    for e, expert in enumerate(experts):
        t, j = torch.nonzero(routing.experts.cpu() == e, as_tuple=True)
        g, u, d = (getattr(expert, n).weight.detach().double().cpu() for n in ("gate_proj", "up_proj", "down_proj"))
        out = (torch.nn.functional.silu(x64[t] @ g.T) * (x64[t] @ u.T)) @ d.T
        y64 = y64.index_add(0, t, out * w[t, j, None])
    ((y64 * target.double().cpu()).mean() + 0.1 * balance).backward()
    # (experts' outputs are rounded to bfloat16 twice: 2^-7 of the terms' size at most)
    assert (router.weight.grad.cpu().double() - w64.grad).norm() <= 2.0**-7 * w64.grad.norm() + 1e-6
    assert all(p.grad is not None and p.grad.isfinite().all() for expert in experts for p in expert.parameters())
    layer = GatedMoE(K, N, E, k).to(device()).to(dtype)
    with torch.no_grad():
        layer.router = router
        for name in ("gate_proj", "up_proj", "down_proj"):
            getattr(layer, name).copy_(torch.stack([getattr(expert, name).weight for expert in experts]))
        served = layer.quantize_(bits=8)(x).double().cpu()
    # (8-bit rows: a step is 1/127 of the largest of some 4 root mean squares, its rounding 0.29 steps: 0.9 % of each operand, three products)
    assert (served - y64.detach()).norm() <= 0.04 * y64.detach().norm()
