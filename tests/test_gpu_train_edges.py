"""Calls of the training operators at the edges of what their documentation allows."""
import pytest
import torch

import ep_moe
import nf4_qlora as Q
import synth
from mxfp4_pack_ref import dequant_mxfp4
from test_gpu_train_ops import check_routing

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def gen(seed):
    return torch.Generator().manual_seed(seed)


def stack64(stack, e):
    blocks, scales = (t[e].cpu() for t in stack)
    return dequant_mxfp4(blocks.reshape(blocks.shape[0], -1, 16), scales).double()


# ------------------------------------------------------------------------------------------------ products
@pytest.mark.parametrize("N", [1, 7, 8, 20, 61, 130])
@pytest.mark.parametrize("product", ["gemm_mxfp4_grouped_train", "gemm_mxfp4_grouped_w4a4_train"])
def test_gradient_of_any_width(product, N):
    """What the forward pass takes has a gradient: exact products added in fp32 (at most N steps of 2^-23 of the sum of
    magnitudes), one rounding to bf16."""
    E, K, sizes, ids = 3, 128, [5, 0, 15], [2, 1, 0]
    g = gen(N)
    stack = synth.mxfp4_stack(E, N, K, g, device=DEV)
    x = torch.randn(20, K, generator=g).to(torch.bfloat16).to(DEV).requires_grad_()
    go = torch.randn(20, N, generator=g).to(torch.bfloat16).to(DEV)
    for tables in ((sizes, ids), (torch.tensor(sizes, device=DEV), torch.tensor(ids, device=DEV))):
        y = getattr(Q, product)(x, *stack, *tables)
        grad, = torch.autograd.grad(y, x, go)
        assert y.shape == (20, N) and grad.shape == x.shape and grad.dtype == x.dtype
        first = 0
        for n, e in zip(sizes, ids):
            w, rows = stack64(stack, e), go[first:first + n].cpu().double()
            ref, mags = rows @ w, rows.abs() @ w.abs()
            assert ((grad[first:first + n].cpu().double() - ref).abs() <= ref.abs() * 2.0 ** -8 + mags * N * 2.0 ** -23).all()
            first += n


@pytest.mark.parametrize("kernel", [True, False])
@pytest.mark.parametrize("product", ["gemm_4bit_grouped_train", "gemm_mxfp4_grouped_train", "gemm_mxfp4_grouped_w4a4_train"])
def test_rows_without_an_expert_have_no_gradient(product, kernel):
    """A padding group and rows behind the last one: zeros, whatever the gradient's memory held before."""
    nf4 = "4bit" in product
    if not kernel and not nf4:
        pytest.skip("only the NF4 gradient has the loop")
    g = gen(12)
    stack = (synth.nf4_stack if nf4 else synth.mxfp4_stack)(2, 64, 128, g, device=DEV)
    more = dict(dgrad_kernel=kernel) if nf4 else {}
    x = torch.randn(300, 128, generator=g).to(torch.bfloat16).to(DEV).requires_grad_()
    go = torch.randn(300, 64, generator=g).to(torch.bfloat16).to(DEV)
    want = torch.zeros_like(x)
    first = 0
    for n, e in ((100, 1), (50, -1), (90, 0)):
        if e >= 0:
            part = x.detach()[first:first + n].clone().requires_grad_()
            want[first:first + n] = torch.autograd.grad(getattr(Q, product)(part, *stack, [n], [e], **more), part, go[first:first + n])[0]
        first += n
    sizes, ids = [100, 50, 90], [1, -1, 0]
    for tables in ((torch.tensor(sizes, device=DEV), torch.tensor(ids, device=DEV)), (sizes + [60], ids + [-1]),
                   (torch.tensor(sizes, device=DEV), torch.tensor(ids))):
        y = getattr(Q, product)(x, *stack, *tables, **more)
        stale = [torch.full((300, 128), float("nan"), dtype=torch.bfloat16, device=DEV) for _ in range(4)]
        del stale
        assert torch.equal(torch.autograd.grad(y, x, go)[0], want)


@pytest.mark.parametrize("on_device", [False, True])
def test_ffn_with_factors_and_padding_groups(on_device):
    """Rows of padding groups hold unwritten memory between the products: none of it reaches a gradient."""
    E, K, h, N, r = 3, 128, 64, 128, 4
    g = gen(15)
    gu, dn = synth.nf4_stack(E, 2 * h, K, g, scale=0.08, device=DEV), synth.nf4_stack(E, N, h, g, scale=0.08, device=DEV)
    factors = [0.1 * torch.randn(*s, generator=g) for s in ((E, r, K), (E, 2 * h, r), (E, r, h), (E, N, r))]
    x, go = (torch.randn(n, d, generator=g).to(torch.bfloat16) for n, d in ((40, K), (40, N)))
    sizes, ids = [10, 14, 16], [1, -1, 2]
    keep = torch.cat((torch.arange(10), torch.arange(24, 40)))

    def grads(x, go, sizes, ids):
        leaves = [t.to(DEV).requires_grad_() for t in (x, *factors)]
        stale = [torch.full((40, n), float("nan"), dtype=torch.bfloat16, device=DEV) for n in (h, 2 * h, N, K) for _ in range(3)]
        del stale
        y = Q.ffn_4bit_grouped_train(leaves[0], *gu, *dn, sizes, ids, lora_gu=leaves[1:3], lora_dn=leaves[3:])
        return torch.autograd.grad(y, leaves, go.to(DEV))

    go[10:24] = 0                                             # the caller leaves the padding's result alone
    tables = (torch.tensor(sizes, device=DEV), torch.tensor(ids, device=DEV)) if on_device else (sizes, ids)
    got, want = grads(x, go, *tables), grads(x[keep], go[keep], [10, 16], [1, 2])
    assert not got[0][10:24].any()
    for a, b in zip((got[0][keep.to(DEV)], *got[1:]), want):
        assert torch.isfinite(a).all() and float((a.double() - b.double()).norm()) <= 1e-5 * float(b.double().norm())


@pytest.mark.parametrize("product", ["gemm_4bit_grouped_train", "gemm_mxfp4_grouped_train", "gemm_mxfp4_grouped_w4a4_train"])
def test_products_of_no_rows(product):
    stack = (synth.nf4_stack if "4bit" in product else synth.mxfp4_stack)(2, 20, 128, gen(13), device=DEV)
    for sizes, ids in (([], []), ([0, 0], [1, 0]), (torch.zeros(2, dtype=torch.int64, device=DEV), torch.tensor([0, 1], device=DEV))):
        x = torch.empty(0, 128, dtype=torch.bfloat16, device=DEV, requires_grad=True)
        y = getattr(Q, product)(x, *stack, sizes, ids)
        y.sum().backward()
        assert y.shape == (0, 20) and x.grad.shape == (0, 128)


def test_ffn_gradient_with_an_odd_result_width():
    E, K, h, N, sizes, ids = 2, 64, 32, 61, [3, 6], [1, 0]
    g = gen(2)
    gu, dn = synth.mxfp4_stack(E, 2 * h, K, g, device=DEV), synth.mxfp4_stack(E, N, h, g, device=DEV)
    x0 = torch.randn(9, K, generator=g).to(torch.bfloat16).to(DEV)
    for rows in ("bf16", "mxfp4"):
        x = x0.clone().requires_grad_()
        y = Q.ffn_mxfp4_grouped_train(x, *gu, *dn, sizes, ids, rows=rows)
        y.float().square().sum().backward()
        assert y.shape == (9, N) and torch.isfinite(x.grad).all() and x.grad.abs().amax(1).all()


PRODUCTS = ["gemm_4bit_grouped_train", "gemm_mxfp4_grouped_train", "gemm_mxfp4_grouped_w4a4_train"]


@pytest.mark.parametrize("product", PRODUCTS)
def test_second_derivatives_of_products_are_refused_where_they_exist(product):
    g = gen(3)
    stack = (synth.nf4_stack if "4bit" in product else synth.mxfp4_stack)(2, 64, 128, g, device=DEV)
    x = torch.randn(6, 128, generator=g).to(torch.bfloat16).to(DEV).requires_grad_()
    y = getattr(Q, product)(x, *stack, [2, 4], [1, 0])
    want, = torch.autograd.grad(y.float().square().sum(), x, retain_graph=True)
    grad, = torch.autograd.grad(y.float().square().sum(), x, create_graph=True)
    assert torch.equal(grad, want)
    with pytest.raises(RuntimeError, match=product):          # a penalty beside a term that has a gradient of its own
        (grad.float().square().sum() + x.float().sum()).backward()
    # an incoming gradient that is a constant: the product's own gradient is one too
    x.grad = None                                             # the sum's part got there before the refusal
    y = getattr(Q, product)(x, *stack, [2, 4], [1, 0])
    grad, = torch.autograd.grad(y, x, torch.ones_like(y), create_graph=True)
    (grad.float().square().sum() + x.float().sum()).backward()
    assert torch.equal(x.grad, torch.ones_like(x))


def test_the_loop_of_the_nf4_gradient_stays_differentiable():
    g = gen(4)
    stack = synth.nf4_stack(2, 64, 128, g, device=DEV)
    x = torch.randn(6, 128, generator=g).to(torch.bfloat16).to(DEV).requires_grad_()
    y = Q.gemm_4bit_grouped_train(x, *stack, [2, 4], [1, 0], dgrad_kernel=False)
    go = torch.randn(6, 64, generator=g).to(torch.bfloat16).to(DEV).requires_grad_()
    grad, = torch.autograd.grad(y, x, go, create_graph=True)
    grad.float().sum().backward()
    assert go.grad is not None and go.grad.abs().sum() > 0


# ------------------------------------------------------------------------------------------------ routing
@pytest.mark.parametrize("mode,norm", [(0, False), (1, False)])
@pytest.mark.parametrize("offset", [100.0, -3000.0, 1e4, -1e5, 1e6])
def test_routing_far_from_zero(offset, mode, norm):
    """Logits with a common offset: probabilities and gradients depend on their differences, and so does the error."""
    for T, E, k in ((40, 32, 4), (300, 256, 8), (70, 1000, 20)):
        logits = 2 * torch.randn(T, E, generator=gen(T)) + offset
        logits[3] = float("-inf")
        logits[5, 1:] = float("-inf")
        check_routing(logits.to(DEV), k, mode, norm, None)


@pytest.mark.parametrize("T", [10, 300])
@pytest.mark.parametrize("mode,norm", [(0, False), (0, True), (1, False)])
def test_routing_rows_with_a_nan_as_route_topk_weighs_them(T, mode, norm):
    x = torch.randn(T, 24, generator=gen(9))
    x[4, 5], x[6, 3], x[7, [1, 2]] = float("nan"), float("inf"), float("inf")
    x[8, 5] = float("-inf")
    r = ep_moe.route_topk_train(x.to(DEV), 3, mode, norm)
    c = ep_moe.route_topk_train(x, 3, mode, norm)
    idx, w = ep_moe.route_topk(x.to(DEV), 3, mode, norm)
    assert torch.equal(r.idx, idx) and torch.equal(r.idx.cpu(), c.idx)
    for other in (w, c.weights.to(DEV)):
        # a sum of 24 exponentials (1 + |x| <= 16 units of 2^-24 each), a division, at either side
        torch.testing.assert_close(r.weights, other, rtol=2 * (24 + 16 + 8) * 2.0 ** -23, atol=0, equal_nan=True)
    assert torch.isnan(r.weights[4]).all() == (mode == 0)


@pytest.mark.parametrize("T", [10, 300])
def test_routing_gradient_of_chosen_weights_beside_a_nan(T):
    """Mode 1 weighs the chosen logits alone: without a gradient of the losses a NaN that was not chosen has no part in it."""
    x = torch.randn(T, 24, generator=gen(10))
    x[4, 5] = float("nan")
    g_w = torch.randn(T, 3, generator=gen(11))
    grads = []
    for dev in (DEV, "cpu"):
        v = x.to(dev).requires_grad_()
        grads.append(torch.autograd.grad(ep_moe.route_topk_train(v, 3, 1).weights, v, g_w.to(dev))[0].cpu())
    assert torch.isfinite(grads[0]).all()
    # w (g - sum w g): three products and their sum, each half a step of 2^-23, weights good to (3 + 16) steps
    assert ((grads[0] - grads[1]).abs() <= 2 * (19 + 4) * 2.0 ** -23 * 4 * g_w.abs().amax()).all()
    v = x.to(DEV).requires_grad_()
    r = ep_moe.route_topk_train(v, 3, 1)
    grad, = torch.autograd.grad((r.weights, r.z_loss), v, (g_w.to(DEV), torch.ones((), device=DEV)))
    assert torch.isnan(grad[4]).all() and torch.isfinite(grad[torch.arange(T) != 4]).all()


def test_a_masked_batch_through_a_layer():
    """The groups of a padded batch are made from the ids of all tokens; the losses' counts leave the padding out."""
    T, E, k, K, h = 60, 5, 2, 128, 64
    g = gen(8)
    gu, dn = synth.nf4_stack(E, 2 * h, K, g, scale=0.08, device=DEV), synth.nf4_stack(E, K, h, g, scale=0.08, device=DEV)
    x = torch.randn(T, K, generator=g).to(torch.bfloat16).to(DEV)
    logits = torch.randn(T, E, generator=g)
    logits[7] = float("-inf")
    mask = torch.rand(T, generator=g) < 0.7
    r = ep_moe.route_topk_train(logits.to(DEV), k, token_mask=mask.to(DEV))
    c = ep_moe.route_topk_train(logits, k, token_mask=mask)
    assert torch.equal(r.counts.cpu(), c.counts) and int(r.counts.sum()) == k * int((mask & (torch.arange(T) != 7)).sum())
    order = torch.argsort(r.idx.reshape(-1), stable=True)
    sizes = torch.bincount(r.idx.reshape(-1), minlength=E)
    assert int(sizes.sum()) == T * k and not torch.equal(sizes.int(), r.counts)
    y = Q.ffn_4bit_grouped_train(x[order // k], *gu, *dn, sizes, torch.arange(E, device=DEV))
    for p in range(0, T * k, 7):
        one = Q.ffn_4bit_grouped_train(x[order[p] // k][None], *gu, *dn, [1], [int(r.idx.reshape(-1)[order[p]])])
        # the same sums in another order and a rounding to bf16 after each of three steps, at either side
        assert float((y[p].double() - one[0].double()).norm() / one[0].double().norm()) <= 6 * 2.0 ** -8


def test_routing_logits_of_the_largest_size():
    """Differences beyond the exponential's range, sizes up to the type's largest: one expert takes all, without a NaN."""
    big = torch.finfo(torch.float32).max
    logits = torch.randn(6, 64, generator=gen(7))
    logits[0, 9], logits[1, 9], logits[2] = big, 1e30, -big
    logits[3, :32], logits[4] = 3e38, -1e30
    logits[4, 11] = -1e29
    x = logits.to(DEV).requires_grad_()
    r = ep_moe.route_topk_train(x, 4)
    r.weights.backward(torch.ones_like(r.weights))
    want = logits.double().requires_grad_()
    p = torch.softmax(want, 1)
    p.gather(1, r.idx.cpu()).sum().backward()
    # d = p_e ([e chosen] - sum of the chosen p): two factors up to 1, each off by the rounding of a sum of 64 exponentials and
    # of its parts (half a step of 2^-23 a term, a handful of units for exponential and reciprocal), well within 72 steps
    assert ((x.grad.cpu().double() - want.grad).abs() <= 2 * 72 * 2.0 ** -23).all()
    assert torch.isfinite(torch.autograd.grad(ep_moe.route_topk_train(x, 4).balance_loss, x)[0]).all()


# ------------------------------------------------------------------------------------------------ second derivatives
def test_second_derivatives_are_refused_beside_other_terms():
    """A penalty on a gradient, beside a term whose gradient is a graph: the part through the kernel must not go missing."""
    x = torch.randn(8, 16, generator=gen(5)).to(DEV).requires_grad_()
    r = ep_moe.route_topk_train(x, 2)
    for out in (r.balance_loss, r.z_loss, r.weights):
        want, = torch.autograd.grad(out, x, torch.ones_like(out), retain_graph=True)
        grad, = torch.autograd.grad(out, x, torch.ones_like(out), create_graph=True)
        assert torch.equal(grad, want)
        with pytest.raises(RuntimeError, match="route_topk_train"):
            (grad.square().sum() + x.sum()).backward()
    gu = torch.randn(4, 64, generator=gen(6)).to(torch.bfloat16).to(DEV).requires_grad_()
    out = Q.glu_train(gu)
    want, = torch.autograd.grad(out, gu, torch.ones_like(out), retain_graph=True)
    grad, = torch.autograd.grad(out, gu, torch.ones_like(out), create_graph=True)
    assert torch.equal(grad, want)
    with pytest.raises(RuntimeError, match="glu_train"):
        (grad.float().square().sum() + gu.float().sum()).backward()


# ------------------------------------------------------------------------------------------------ GLU
@pytest.mark.parametrize("mode", [torch.no_grad, torch.inference_mode])
@pytest.mark.parametrize("act", ["silu", "gpt_oss"])
def test_glu_without_gradients_makes_no_checkpoint(mode, act):
    rows, h = 4096, 1024
    x = torch.randn(rows, 2 * h, device=DEV, dtype=torch.bfloat16, requires_grad=True)
    want = Q.glu_train(x, act).detach()
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    with mode():
        out = Q.glu_train(x, act)
    assert torch.cuda.max_memory_allocated() - before <= 2 * rows * h + 4096          # the result and nothing beside it
    assert torch.equal(out, want) and not out.requires_grad


@pytest.mark.parametrize("act", ["silu", "gpt_oss"])
def test_glu_codes_are_nearest(act):
    """Every value is held by a code that no other code is nearer than: off by at most half a step of the block's maximum / 127.
    127 / max is rounded once (2^-24), so a value may pass half way by 127 * 2^-24 steps; many lie there exactly."""
    import _gnf4b
    rows, h = 257, 200
    nb = -(-h // 64)
    gu = torch.randn(rows, 2 * h, generator=gen(14)).to(torch.bfloat16)
    gu[:40, ::3] = gu[:40].float().abs().amax(1, keepdim=True).to(torch.bfloat16) / 2                  # 63.5 steps
    gu[40] = torch.linspace(-4, 4, 2 * h).to(torch.bfloat16)
    x = gu.to(DEV)
    out = torch.empty(rows, h, dtype=torch.bfloat16, device=DEV)
    codes = torch.empty(rows, nb, 2, 64, dtype=torch.int8, device=DEV)
    steps = torch.empty(rows, nb, 2, dtype=torch.float32, device=DEV)
    assert _gnf4b.load().gnf4b_glu_ckpt8_fwd(x.data_ptr(), rows, h, 0 if act == "silu" else 1, None, None, 0, out.data_ptr(), codes.data_ptr(),
                                             steps.data_ptr(), None, torch.cuda.current_stream().cuda_stream) == 0
    gate, up = (gu[:, :h], gu[:, h:]) if act == "silu" else (gu[:, 0::2], gu[:, 1::2])
    v = torch.nn.functional.pad(torch.stack((gate, up), 1).double(), (0, nb * 64 - h)).reshape(rows, 2, nb, 64).transpose(1, 2)
    top = v.abs().amax(-1, keepdim=True)
    assert torch.equal(steps.cpu(), (top[..., 0].float() / 127.0))
    code = codes.cpu().double()
    assert code.abs().max() == 127 and ((v * 127 - code * top).abs() <= top * (0.5 + 127 * 2.0 ** -24)).all()
    assert ((v * 254 / top) % 2 == 1).sum() > 500                     # of the inputs: values half way between two codes
