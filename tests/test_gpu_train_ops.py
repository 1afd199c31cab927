"""Routing with its losses, and the GLU with an 8-bit checkpoint, against plain 64-bit implementations, their
gradients against the formulas' and against differences; then both in a training step of a layer."""
import pytest
import torch

import ep_moe
import mxfp4_grouped as M
import nf4_grouped
import nf4_qlora as Q
import synth

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U32 = 2.0 ** -24                                                     # one fp32 rounding


def gen(seed):
    return torch.Generator().manual_seed(seed)


# ------------------------------------------------------------------------------------------------ routing
def route64(logits, k, mode, norm, mask):
    """The definition in 64 bits, differentiable (CPU)."""
    lg = logits.detach().double().cpu().requires_grad_()
    dead = torch.isneginf(lg.detach()).all(1)
    keep = ~dead if mask is None else mask.cpu() & ~dead
    idx = torch.sort(lg.detach(), dim=1, descending=True, stable=True)[1][:, :k]
    live = torch.nonzero(~dead).reshape(-1)
    p = torch.softmax(lg[live], 1)
    sel = torch.softmax(torch.gather(lg[live], 1, idx[live]), 1) if mode == 1 or norm else torch.gather(p, 1, idx[live])
    w = torch.zeros(lg.shape[0], k, dtype=torch.float64).index_copy(0, live, sel)
    n = max(1, int(keep.sum()))
    counts = torch.zeros(lg.shape[1], dtype=torch.int64)
    counts.index_add_(0, idx[keep].reshape(-1), torch.ones(int(keep.sum()) * k, dtype=torch.int64))
    balance = lg.shape[1] * (counts.double() / (n * k) * p[keep[live]].sum(0) / n).sum()
    z = torch.logsumexp(lg[keep], 1).square().sum() / n
    return lg, idx, w, counts, balance, z


def check_routing(logits, k, mode, norm, mask, seed=0):
    T, E = logits.shape
    lg, idx, w, counts, balance, z = route64(logits, k, mode, norm, mask)
    x = logits.detach().requires_grad_()
    r = ep_moe.route_topk_train(x, k, mode, norm, token_mask=mask)
    assert torch.equal(r.idx.cpu(), idx) and torch.equal(r.counts.cpu().long(), counts)
    # a probability: expf of a difference (its rounding: |difference| <= 64 here), a sum of E terms, a division
    rel = (64 + E + 16) * 2 * U32
    assert ((r.weights.cpu().double() - w).abs() <= rel * w + 1e-30).all()
    assert abs(float(r.balance_loss.detach()) - float(balance.detach())) <= (rel + (T + E) * U32) * abs(float(balance.detach()))
    assert abs(float(r.z_loss.detach()) - float(z.detach())) <= (2 * rel + T * U32) * max(abs(float(z.detach())), 1e-6)
    g = gen(seed + 77)
    g_w, g_b, g_z = torch.randn(T, k, generator=g), torch.randn((), generator=g) * T, torch.randn((), generator=g) * T / 10
    want, = torch.autograd.grad((w * g_w.double()).sum() + balance * g_b.double() + z * g_z.double(), lg)
    got, = torch.autograd.grad((r.weights, r.balance_loss, r.z_loss), x, (g_w.to(DEV), g_b.to(DEV), g_z.to(DEV)))
    assert got.dtype == logits.dtype
    # each term is a probability times a sum of at most E + k + 2 others: bounded by the terms' own magnitudes
    n = max(1, int(counts.sum()) // k)
    lse = torch.logsumexp(lg.detach(), 1).abs()
    lse = torch.where(torch.isfinite(lse), lse, torch.zeros_like(lse))
    push = abs(float(g_b)) * E * counts.double().max() / (n * n * k)
    size = (g_w.double().abs() * w.detach()).sum(1) + g_w.double().abs().amax(1) + 2 * push + 2 * abs(float(g_z)) * lse / n
    tol = 4 * rel * size[:, None] + want.abs() * (torch.finfo(logits.dtype).eps / 2)
    if logits.dtype == torch.float16:
        tol = tol + 2.0 ** -25                                        # half a step of its subnormals
    bad = (got.cpu().double() - want).abs() > tol
    assert not bad.any(), (int(bad.sum()), float(((got.cpu().double() - want).abs() - tol).max()))


@pytest.mark.parametrize("mode,norm", [(0, False), (0, True), (1, False)])
@pytest.mark.parametrize("T,E,k", [(1, 1, 1), (1, 8, 2), (3, 32, 32), (64, 128, 8), (128, 33, 4), (129, 64, 6), (300, 60, 4),
                                   (1000, 256, 8), (2000, 257, 3), (700, 512, 10), (500, 1000, 7), (400, 1024, 32), (9000, 8, 2)])
def test_routing_shapes(T, E, k, mode, norm):
    check_routing((2 * torch.randn(T, E, generator=gen(T + E))).to(DEV), k, mode, norm, None)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("masked", [0.0, 0.3, 0.95])
def test_routing_types_ties_and_masks(dtype, masked):
    T, E, k = 777, 96, 5
    logits = (torch.randint(-6, 7, (T, E), generator=gen(5)).float() / 4).to(dtype)         # many ties
    logits[:, 7] = 0.0
    logits[:, 9] = -0.0
    mask = (torch.rand(T, generator=gen(6)) >= masked).to(DEV)
    check_routing(logits.to(DEV), k, 0, False, mask)
    check_routing(logits.to(DEV), k, 1, False, mask)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("E,k", [(48, 17), (64, 32), (100, 24), (256, 16), (256, 17), (256, 32), (512, 20), (1000, 32)])
def test_routing_many_choices(dtype, E, k):
    """k around and above the switch to two maxima a lane: distinct logits, few values, neighbours that are all large."""
    T = 150
    distinct = torch.stack([torch.randperm(E, generator=gen(90 + i)) for i in range(T)]).float() / 16 - E / 32
    ties = torch.randint(-3, 4, (T, E), generator=gen(91)).float()
    block = torch.randn(T, E, generator=gen(92))
    block[:, E // 2:E // 2 + 33] += 6                       # the choices lie side by side
    for logits in (distinct, ties, block):
        check_routing(logits.to(dtype).to(DEV), k, 0, False, None)
        check_routing(logits.to(dtype).to(DEV), k, 1, False, None)


@pytest.mark.parametrize("T", [6, 500])
def test_routing_excluded_experts_and_dead_tokens(T):
    E, k = 40, 6
    logits = torch.randn(T, E, generator=gen(7))
    logits[:, 10:20] = float("-inf")                       # experts that are switched off
    logits[1] = float("-inf")                              # a token with nothing to choose from
    logits[2, 3:] = float("-inf")                          # fewer choices than k
    logits[3] = torch.finfo(torch.float32).min             # a mask by the type's lowest value: an even choice
    check_routing(logits[:3].to(DEV), k, 0, False, None)
    check_routing(logits[:3].to(DEV), k, 0, True, None)
    x = logits.to(DEV).requires_grad_()
    r = ep_moe.route_topk_train(x, k)
    assert r.idx[1].tolist() == list(range(k)) and not r.weights[1].any()
    assert r.idx[3].tolist() == list(range(k)) and torch.equal(r.weights[3], torch.full((k,), 1 / E, device=DEV))
    r = ep_moe.route_topk_train(x, k, token_mask=torch.arange(T, device=DEV) != 3)
    (r.weights.sum() + r.balance_loss + r.z_loss).backward()
    assert torch.isfinite(x.grad).all() and not x.grad[1].any()
    assert int(r.counts.sum()) == (T - 2) * k


@pytest.mark.parametrize("E,k", [(3, 3), (16, 4), (32, 9), (33, 20), (200, 18)])
def test_routing_rows_with_little_to_choose_from(E, k):
    """Fewer finite logits than choices, one, none; ties of everything; also where a lane holds one expert."""
    logits = torch.randn(64, E, generator=gen(70 + E))
    for t in range(32):
        logits[t, torch.randperm(E, generator=gen(t))[t % (E + 1):]] = float("-inf")
    logits[32:40] = 1.25
    logits[40:44] = 0.0
    logits[41, ::2] = -0.0
    for mode in (0, 1):
        r = ep_moe.route_topk_train(logits.to(DEV), k, mode)
        c = ep_moe.route_topk_train(logits, k, mode)
        assert torch.equal(r.idx.cpu(), c.idx) and torch.equal(r.counts.cpu(), c.counts)
        # sums of at most E terms, two more roundings and the exponentials' few units, on both sides
        assert ((r.weights.cpu() - c.weights).abs() <= 2 * (E + 16) * 2 * U32 * c.weights + 1e-30).all()


def test_routing_nothing_counts_and_no_tokens():
    x = torch.randn(5, 16, generator=gen(8)).to(DEV).requires_grad_()
    r = ep_moe.route_topk_train(x, 2, token_mask=torch.zeros(5, dtype=torch.bool, device=DEV))
    assert float(r.balance_loss.detach()) == 0 and float(r.z_loss.detach()) == 0 and not r.counts.any()
    (r.balance_loss + r.z_loss).backward()
    assert not x.grad.any()
    e = torch.empty(0, 16, device=DEV, requires_grad=True)
    r = ep_moe.route_topk_train(e, 2)
    assert r.idx.shape == (0, 2) and float(r.balance_loss) == 0 and not r.counts.any()
    (r.weights.sum() + r.balance_loss).backward()
    assert e.grad.shape == (0, 16)


@pytest.mark.parametrize("T", [20, 300])
def test_routing_nan_rows_keep_to_themselves(T):
    x = torch.randn(T, 24, generator=gen(9)).to(DEV)
    x[4, 5] = float("nan")
    mask = torch.arange(T, device=DEV) != 4
    clean = x.clone()
    clean[4] = 0
    x.requires_grad_(), clean.requires_grad_()
    a, b = (ep_moe.route_topk_train(v, 3, token_mask=mask) for v in (x, clean))
    others = mask.nonzero().reshape(-1)
    assert torch.equal(a.balance_loss, b.balance_loss) and torch.equal(a.z_loss, b.z_loss) and torch.equal(a.counts, b.counts)
    assert torch.equal(a.idx[others], b.idx[others]) and torch.equal(a.weights[others], b.weights[others])
    assert 5 not in a.idx[4].tolist() and len(set(a.idx[4].tolist())) == 3 and torch.isnan(a.weights[4]).all()
    (a.balance_loss + a.z_loss).backward()
    assert torch.isfinite(x.grad).all()
    assert torch.isnan(ep_moe.route_topk_train(x.detach(), 3).balance_loss)
    for bits in (0x7fc00000, -0x400000):                     # either sign, beside nothing but -inf: a NaN row, not an empty one
        y = torch.randn(T, 24, generator=gen(9)).to(DEV)
        y[4] = float("-inf")
        y[4, 7] = torch.tensor(bits, dtype=torch.int32).view(torch.float32)
        assert torch.isnan(y[4, 7])
        r = ep_moe.route_topk_train(y, 3, 0, True)
        assert r.idx[4].tolist() == [0, 1, 2] and torch.isnan(r.weights[4]).all() and torch.isnan(r.balance_loss)
        assert torch.isfinite(r.weights[torch.arange(T, device=DEV) != 4]).all()


def test_routing_matches_route_topk_and_its_cpu_form():
    x = torch.randn(1000, 128, generator=gen(10)).to(DEV)
    for mode, norm in ((0, False), (0, True), (1, False)):
        r = ep_moe.route_topk_train(x, 8, mode, norm)
        idx, w = ep_moe.route_topk(x, 8, mode, norm)
        assert torch.equal(r.idx, idx)
        torch.testing.assert_close(r.weights, w, rtol=3e-5, atol=0)
        c = ep_moe.route_topk_train(x.cpu(), 8, mode, norm)
        assert torch.equal(r.idx.cpu(), c.idx) and torch.equal(r.counts.cpu(), c.counts)
        torch.testing.assert_close(r.balance_loss.cpu(), c.balance_loss, rtol=3e-5, atol=0)


def test_routing_gradient_against_differences():
    """Central differences of the 64-bit formulas (the selection does not change at this step)."""
    x = torch.randn(4, 12, generator=gen(11))
    g_w = torch.randn(4, 3, generator=gen(12)).double()

    def total(v):
        _, _, w, _, b, z = route64(v, 3, 0, False, None)
        return float(((w * g_w).sum() + 3 * b + 0.5 * z).detach())

    xd = x.to(DEV).requires_grad_()
    r = ep_moe.route_topk_train(xd, 3)
    got, = torch.autograd.grad((r.weights, r.balance_loss, r.z_loss), xd, (g_w.float().to(DEV), torch.tensor(3.0, device=DEV), torch.tensor(0.5, device=DEV)))
    h = 1e-5
    for t, e in [(0, 0), (1, 5), (2, 11), (3, int(r.idx[3, 0])), (0, int(r.idx[0, 2]))]:
        d = x.double().clone()
        d[t, e] += h
        up = total(d)
        d[t, e] -= 2 * h
        diff = (up - total(d)) / (2 * h)
        assert abs(diff - float(got[t, e])) <= 1e-5 * max(1.0, abs(diff)), (t, e)


def test_routing_partial_gradients_views_and_determinism():
    big = torch.randn(400, 200, generator=gen(13)).to(DEV)
    view = big[:, 30:126]
    base = ep_moe.route_topk_train(view.contiguous(), 4)
    again = ep_moe.route_topk_train(view, 4)
    for a, b in zip(base, again):
        assert torch.equal(a, b)
    t = view.t().contiguous().t()                               # column-major logits
    assert torch.equal(ep_moe.route_topk_train(t, 4).balance_loss, base.balance_loss)
    x = big.clone().requires_grad_()
    ep_moe.route_topk_train(x[:, 30:126], 4).z_loss.backward()
    assert not x.grad[:, :30].any() and x.grad[:, 30:126].any()
    x = view.contiguous().requires_grad_()
    r = ep_moe.route_topk_train(x, 4)
    g1, = torch.autograd.grad(r.weights.sum() * 2, x, retain_graph=True)
    g2, = torch.autograd.grad(r.balance_loss, x, retain_graph=True)
    g12, = torch.autograd.grad(r.weights.sum() * 2 + r.balance_loss, x)
    torch.testing.assert_close(g1 + g2, g12, rtol=1e-5, atol=1e-7)
    # a broadcast incoming gradient
    r = ep_moe.route_topk_train(x, 4)
    ga, = torch.autograd.grad(r.weights, x, torch.ones(1, 1, device=DEV).expand(400, 4))
    r = ep_moe.route_topk_train(x, 4)
    gb, = torch.autograd.grad(r.weights, x, torch.ones(400, 4, device=DEV))
    assert torch.equal(ga, gb)


def test_gradients_are_not_differentiable_twice():
    x = torch.randn(8, 16, device=DEV, requires_grad=True)
    r = ep_moe.route_topk_train(x, 2)
    g, = torch.autograd.grad(r.balance_loss, x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()
    gu = torch.randn(4, 64, device=DEV, dtype=torch.bfloat16, requires_grad=True)
    out = Q.glu_train(gu)
    g, = torch.autograd.grad(out, gu, torch.ones_like(out), create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


def test_routing_under_graphs_and_on_streams():
    x = torch.randn(512, 64, generator=gen(14)).to(DEV).requires_grad_()
    one = torch.ones((), device=DEV)

    def step():
        r = ep_moe.route_topk_train(x, 4)
        g, = torch.autograd.grad((r.balance_loss, r.z_loss), x, (one, one))
        return r.counts, r.balance_loss.detach(), g

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            want = step()
    torch.cuda.current_stream().wait_stream(side)
    del want
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step())
        graphs.append(g)
    with torch.no_grad():
        x.mul_(-1.5)
    torch.cuda.synchronize()
    graphs[0].replay()
    with torch.cuda.stream(side):
        graphs[1].replay()
    torch.cuda.synchronize()
    want = step()
    for o in outs:
        for a, b in zip(o, want):
            assert torch.equal(a, b)


# ------------------------------------------------------------------------------------------------ GLU with an 8-bit checkpoint
def parts(gu, act):
    h = gu.shape[1] // 2
    return (gu[:, :h], gu[:, h:]) if act == "silu" else (gu[:, 0::2], gu[:, 1::2])


def joined(g, u, act):
    return torch.cat((g, u), 1) if act == "silu" else torch.stack((g, u), 2).reshape(g.shape[0], -1)


def act64(g, u, act):
    if act == "silu":
        return g * torch.sigmoid(g) * u
    g, u = torch.clamp(g, max=7.0), torch.clamp(u, -7.0, 7.0)
    return (u + 1) * g * torch.sigmoid(1.702 * g)


def kept(v):
    """v [rows, h] (fp32) as the checkpoint holds it."""
    rows, h = v.shape
    b = torch.nn.functional.pad(v, (0, -h % 64)).reshape(rows, -1, 64)
    top = b.abs().amax(-1, keepdim=True)
    top = torch.where(top < 2.0 ** -100, torch.zeros_like(top), top)
    # a tensor over a tensor is one division; torch evaluates 127.0 / top as 127 * (1 / top), two roundings (127 / 7.875 then
    # comes out one step above the nearest fp32 number, and half the block's maximum, 63.5 steps, on the other side)
    q = torch.where(top > 0, torch.round(b.double() * (torch.full_like(top, 127.0) / top).double()), torch.zeros_like(b, dtype=torch.float64))
    return (q * (top / 127.0).double()).reshape(rows, -1)[:, :h]


def check_glu(gu, act, g_out, bias=None, row_expert=None):
    x = gu.to(DEV).requires_grad_()
    out = Q.glu_train(x, act, bias=bias.to(DEV) if bias is not None else None, row_expert=row_expert.to(DEV) if bias is not None else None)
    grad, = torch.autograd.grad(out, x, g_out.to(DEV))
    full = gu.float() + (bias[row_expert.long()].float() if bias is not None else 0.0)
    g, u = parts(full, act)
    ref = act64(g.double(), u.double(), act)
    # one rounding to bf16; in the logistic function 2^x (2 units of 2^-23), its reciprocal (1), the sum and two products
    # (half each), and the exponent's own roundings: two constants and two products of half a unit of 2^-23 to one of
    # 2^-24 each, 1.5 * 2^-23 |1.702 gate| together.  A logistic value below 2^-126 is flushed to zero (ftz), which
    # leaves up to 2^-126 times the rest of the product
    gd, ud = g.abs().double(), u.abs().double()
    slack = (5 + 2.6 * gd) * 2.0 ** -23
    assert ((out.detach().cpu().double() - ref).abs() <= ref.abs() * (2.0 ** -8 + slack) + 2.0 ** -126 * (1 + gd * (ud + 1))).all()
    kg, ku = (kept(v).requires_grad_() for v in (g, u))
    want = torch.autograd.grad(act64(kg, ku, act), (kg, ku), g_out.double())
    # the derivative's two terms may cancel: the fp32 steps count against their sizes
    sg = torch.sigmoid(kg.detach() * (1.0 if act == "silu" else 1.702))
    size = g_out.double().abs() * (ku.detach().abs() + 1) * sg * (1 + 1.702 * kg.detach().abs()) if act != "silu" else \
        g_out.double().abs() * ku.detach().abs() * sg * (1 + kg.detach().abs())
    slack = (8 + 4.5 * kg.detach().abs()) * 2.0 ** -23
    for got, ref, sz in zip(parts(grad.cpu().double(), act), want, (size, g_out.double().abs() * kg.detach().abs() * sg)):
        flushed = 2.0 ** -126 * (1 + g_out.double().abs() * (1 + ku.detach().abs()) * (1 + 1.702 * kg.detach().abs()))
        bad = (got - ref).abs() > ref.abs() * 2.0 ** -8 + sz * slack + flushed
        assert not bad.any(), (int(bad.sum()), float((got - ref).abs()[bad].max()))


@pytest.mark.parametrize("act", ["silu", "gpt_oss"])
@pytest.mark.parametrize("rows,h", [(1, 1), (1, 8), (3, 63), (2, 64), (5, 65), (7, 72), (33, 100), (4, 127), (300, 768), (65, 2880)])
def test_glu_shapes(act, rows, h):
    g = gen(rows + h)
    check_glu((3 * torch.randn(rows, 2 * h, generator=g)).to(torch.bfloat16), act, torch.randn(rows, h, generator=g).to(torch.bfloat16))


@pytest.mark.parametrize("act", ["silu", "gpt_oss"])
def test_glu_ranges_and_clamps(act):
    """Blocks of very different size beside each other, values at and beyond the clamps, zero and tiny blocks."""
    g = gen(15)
    rows, h = 48, 192
    gu = torch.randn(rows, 2 * h, generator=g) * torch.exp2(torch.randint(-20, 5, (rows, 1), generator=g).float())
    gu[0] = 0
    gu[1] = 1e-35
    gu[2, ::3] = 7.0
    gu[3, ::3] = -7.0
    gu[4] = torch.linspace(-12, 12, 2 * h)
    gu[5] = 80.0
    gu[6] = -80.0
    check_glu(gu.to(torch.bfloat16), act, torch.randn(rows, h, generator=g).to(torch.bfloat16))


def test_glu_bias_by_expert():
    g = gen(16)
    gu = torch.randn(40, 2 * 96, generator=g).to(torch.bfloat16)
    bias = (2 * torch.randn(5, 2 * 96, generator=g)).to(torch.bfloat16)
    who = torch.randint(0, 5, (40,), generator=g).to(torch.int32)
    check_glu(gu, "gpt_oss", torch.randn(40, 96, generator=g).to(torch.bfloat16), bias, who)
    gu = torch.randn(9, 2 * 13, generator=g).to(torch.bfloat16)
    check_glu(gu, "gpt_oss", torch.randn(9, 13, generator=g).to(torch.bfloat16), bias[:, :26].contiguous(), who[:9])
    nf4_grouped.last_status(DEV)
    Q.glu_train(gu.to(DEV), "gpt_oss", bias=bias[:, :26].to(DEV), row_expert=torch.full((9,), 5, device=DEV))
    assert nf4_grouped.last_status(DEV) == 1


@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
def test_glu_nonfinite_blocks_do_not_become_finite(bad):
    gu = torch.randn(4, 2 * 128, generator=gen(17)).to(torch.bfloat16)
    clean = gu.clone()
    gu[2, 70] = bad                                        # the gate's second block
    go = torch.ones(4, 128, dtype=torch.bfloat16, device=DEV)
    grads = []
    for v in (gu, clean):
        x = v.to(DEV).requires_grad_()
        grads.append(torch.autograd.grad(Q.glu_train(x, "silu"), x, go)[0])
    a, b = grads
    assert not torch.isfinite(a[2, 64:128]).any()
    keep = torch.ones(4, 256, dtype=torch.bool)
    keep[2, 64:128] = keep[2, 192:256] = False
    assert torch.equal(a.cpu()[keep], b.cpu()[keep])


def test_glu_gradient_against_differences():
    """Of the formula at kept values: inputs that the checkpoint holds exactly (whole steps of their block)."""
    rows, h = 2, 64
    g = gen(18)
    codes = torch.randint(-127, 128, (rows, 2, 64), generator=g).float()
    codes[:, :, 0] = 127
    step = 2.0 ** -5
    for act in ("silu", "gpt_oss"):
        v = codes * step
        gu = joined(v[:, 0], v[:, 1], act).to(torch.bfloat16)
        assert torch.equal(gu.float(), joined(v[:, 0], v[:, 1], act))
        x = gu.to(DEV).requires_grad_()
        grad, = torch.autograd.grad(Q.glu_train(x, act), x, torch.ones(rows, h, dtype=torch.bfloat16, device=DEV))
        d = 1e-6
        gd, ud = v[:, 0].double(), v[:, 1].double()
        want = joined((act64(gd + d, ud, act) - act64(gd - d, ud, act)) / (2 * d), (act64(gd, ud + d, act) - act64(gd, ud - d, act)) / (2 * d), act)
        assert ((grad.cpu().double() - want).abs() <= want.abs() * 2.0 ** -8 + 1e-5).all()


def test_glu_views_no_grad_and_broadcast_gradient():
    big = torch.randn(30, 300, generator=gen(19)).to(torch.bfloat16).to(DEV)
    x = big.clone().requires_grad_()
    out = Q.glu_train(x[:, 20:212], "silu")
    g, = torch.autograd.grad(out, x, torch.ones(1, 1, dtype=torch.bfloat16, device=DEV).expand(30, 96))
    y = big[:, 20:212].contiguous().requires_grad_()
    out2 = Q.glu_train(y, "silu")
    g2, = torch.autograd.grad(out2, y, torch.ones(30, 96, dtype=torch.bfloat16, device=DEV))
    assert torch.equal(out, out2) and torch.equal(g[:, 20:212], g2) and not g[:, :20].any()
    with torch.no_grad():
        assert torch.equal(Q.glu_train(y, "silu"), out2)
    odd = torch.empty(30 * 192 + 1, dtype=torch.bfloat16, device=DEV)[1:].reshape(30, 192).copy_(y.detach())       # not 16-byte aligned
    assert torch.equal(Q.glu_train(odd, "silu"), out2)
    assert Q.glu_train(big[:0, :64], "gpt_oss").shape == (0, 32)
    with pytest.raises(ValueError, match="frozen"):
        Q.glu_train(y, "gpt_oss", bias=torch.zeros(1, 192, dtype=torch.bfloat16, device=DEV, requires_grad=True),
                    row_expert=torch.zeros(30, dtype=torch.int32, device=DEV))
    with pytest.raises(TypeError):
        Q.glu_train(y.detach().float(), "silu")


def test_glu_keeps_eight_bits():
    rows, h = 4096, 1024
    x = torch.randn(rows, 2 * h, device=DEV, dtype=torch.bfloat16, requires_grad=True)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    out = Q.glu_train(x, "silu")
    kept_bytes = torch.cuda.memory_allocated() - before - out.numel() * 2
    assert rows * 2 * h <= kept_bytes <= rows * 2 * h * 17 / 16 + 4096


def test_glu_under_graphs_and_on_streams():
    """Two captured forward-and-backward passes of the same buffers, replayed on two streams with other inputs."""
    x = torch.randn(300, 256, generator=gen(21)).to(torch.bfloat16).to(DEV).requires_grad_()
    go = torch.randn(300, 128, generator=gen(22)).to(torch.bfloat16).to(DEV)

    def step():
        out = Q.glu_train(x, "gpt_oss")
        return out.detach(), torch.autograd.grad(out, x, go)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step())
        graphs.append(g)
    with torch.no_grad():
        x.mul_(-0.75)
    go.mul_(2)
    torch.cuda.synchronize()
    graphs[0].replay()
    with torch.cuda.stream(side):
        graphs[1].replay()
    torch.cuda.synchronize()
    want = step()
    for o in outs:
        assert torch.equal(o[0], want[0]) and torch.equal(o[1], want[1])


# ------------------------------------------------------------------------------------------------ together
def test_w4a4_train_is_the_quantised_product_with_the_plain_gradient():
    E, N, K = 3, 64, 128
    g = gen(23)
    wb, ws = synth.mxfp4_stack(E, N, K, g, device=DEV)
    x = torch.randn(20, K, generator=g).to(torch.bfloat16).to(DEV).requires_grad_()
    go = torch.randn(20, N, generator=g).to(torch.bfloat16).to(DEV)
    sizes, ids = [5, 0, 15], [2, 1, 0]
    y = Q.gemm_mxfp4_grouped_w4a4_train(x, wb, ws, sizes, ids)
    assert torch.equal(y, M.gemm_mxfp4_grouped_w4a4(*M.quantize_mxfp4(x), wb, ws, sizes, ids))
    got, = torch.autograd.grad(y, x, go)
    assert torch.equal(got, M.dgrad_mxfp4_grouped(go, wb, ws, sizes, ids))
    half = x.detach().half().requires_grad_()
    got, = torch.autograd.grad(Q.gemm_mxfp4_grouped_w4a4_train(half, wb, ws, sizes, ids), half, go)
    assert got.dtype == torch.float16


@pytest.mark.parametrize("fmt,rows_fmt", [("nf4", "bf16"), ("mxfp4", "bf16"), ("mxfp4", "mxfp4")])
def test_layer_training_step(fmt, rows_fmt):
    """Router with its losses, the experts' products on 4-bit stacks, the GLU from its checkpoint, the weighted sum:
    the gradients of hidden rows and logits against the same layer in 64-bit tensor operations on the decoded stacks
    (the products' and the activation's roundings to bf16 apart, hence the bound)."""
    T, E, k, K, h = 48, 6, 2, 128, 64
    g = gen(20)
    act = "silu" if fmt == "nf4" else "gpt_oss"
    if fmt == "nf4":
        gu, dn = synth.nf4_stack(E, 2 * h, K, g, scale=0.08, device=DEV), synth.nf4_stack(E, K, h, g, scale=0.08, device=DEV)
        dec = [torch.stack([nf4_grouped.dequant_ref(b[e], a[e], b.shape[1], b.shape[2] * 2) for e in range(E)]).double() for b, a in (gu, dn)]
    else:
        gu, dn = synth.mxfp4_stack(E, 2 * h, K, g, device=DEV, e_lo=121, e_hi=122), synth.mxfp4_stack(E, K, h, g, device=DEV, e_lo=121, e_hi=122)
        dec = [M.dequant_stack_cuda(b, s).double() for b, s in (gu, dn)]
    x0 = torch.randn(T, K, generator=g).to(torch.bfloat16).to(DEV)
    l0 = torch.randn(T, E, generator=g).to(DEV)
    go = torch.randn(T, K, generator=g).to(DEV)

    def layer(x, logits, wide):
        if wide:
            r = ep_moe._route_train_ops(logits, k, 0, True, None)
        else:
            r = ep_moe.route_topk_train(logits, k, 0, True)
        order = torch.argsort(r.idx.reshape(-1), stable=True)
        sizes, ids = r.counts.tolist(), list(range(E))
        a = x[order // k]
        if wide:
            e = r.idx.reshape(-1)[order]
            gate, up = parts(torch.einsum("tk,tnk->tn", a, dec[0][e]), act)
            y = torch.einsum("tk,tnk->tn", act64(gate, up, act), dec[1][e])
        elif fmt == "nf4":
            y = Q.ffn_4bit_grouped_train(a, *gu, *dn, sizes, ids, act=act)
        else:
            y = Q.ffn_mxfp4_grouped_train(a, *gu, *dn, sizes, ids, act=act, rows=rows_fmt)
        w = r.weights.reshape(-1)[order]
        out = torch.zeros(T, K, dtype=torch.float64 if wide else torch.float32, device=DEV).index_add(0, order // k, y.to(w.dtype)[:, :] * w[:, None] if not wide else y * w.double()[:, None])
        return out, r.balance_loss, r.z_loss

    res = []
    for wide in (False, True):
        x = (x0.double() if wide else x0.clone()).requires_grad_()
        l = l0.clone().requires_grad_()
        out, bal, z = layer(x, l, wide)
        loss = (out * go.to(out.dtype)).sum() + 0.1 * bal + 0.01 * z
        loss.backward()
        res.append((out.detach().double(), x.grad.double(), l.grad.double()))
    # bf16 roundings on the way (rows, two products, activation, two gradients): each at most 2^-8 relative and
    # independent over the sums; MXFP4 rows: half a step of e2m1, up to 1/4 of a value, about 1/8 in the mean
    limit = 2.0 ** -8 * 6 if rows_fmt == "bf16" else 0.25
    for a, b in zip(*res):
        assert float((a - b).norm() / b.norm()) <= limit
    assert nf4_grouped.last_status(DEV) == 0
