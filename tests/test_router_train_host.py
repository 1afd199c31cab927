"""route_topk_train on CPU tensors (its tensor-operation form) against a plain loop in 64 bits and against differences,
and the refusals of the training operators: no GPU needed."""
import ctypes
import math

import pytest
import torch

import _gnf4b
import ep_moe
import nf4_qlora


def plain(logits, k, mode, norm, mask):
    """One token at a time, in Python floats."""
    T, E = logits.shape
    rows = logits.double().tolist()
    idx, w, counts, n, mean_p, z = [], [], [0] * E, 0, [0.0] * E, 0.0
    for t in range(T):
        l = rows[t]
        order = sorted(range(E), key=lambda e: (-l[e], e))[:k]
        top = max(l)
        idx.append(order)
        if top == -math.inf:
            w.append([0.0] * k)
            continue
        ex = [math.exp(v - top) for v in l]
        tot = sum(ex)
        sel = [ex[e] for e in order]
        w.append([s / (sum(sel) if mode == 1 or norm else tot) for s in sel])
        if mask is not None and not mask[t]:
            continue
        n += 1
        z += (top + math.log(tot)) ** 2
        for e in order:
            counts[e] += 1
        for e in range(E):
            mean_p[e] += ex[e] / tot
    bal = E * sum(c / (n * k) * p / n for c, p in zip(counts, mean_p)) if n else 0.0
    return idx, w, counts, bal, z / n if n else 0.0


@pytest.mark.parametrize("mode,norm", [(0, False), (0, True), (1, False)])
@pytest.mark.parametrize("T,E,k", [(1, 1, 1), (5, 8, 2), (17, 33, 33), (9, 64, 6)])
def test_cpu_form_against_plain_loop(T, E, k, mode, norm):
    g = torch.Generator().manual_seed(T * 100 + E)
    logits = torch.randn(T, E, generator=g)
    logits[0, : E // 2] = float("-inf")
    if T > 3:
        logits[2] = float("-inf")
    if E > 4:
        logits[-1, 1] = logits[-1, 3] = logits[-1].max() + 1            # a tie
    mask = torch.rand(T, generator=g) < 0.7 if T > 1 else None
    r = ep_moe.route_topk_train(logits, k, mode, norm, token_mask=mask)
    idx, w, counts, bal, z = plain(logits, k, mode, norm, mask)
    assert r.idx.tolist() == idx and r.counts.tolist() == counts
    torch.testing.assert_close(r.weights.double(), torch.tensor(w, dtype=torch.float64), rtol=2e-6, atol=1e-7)
    assert abs(float(r.balance_loss) - bal) <= 1e-5 * max(1, abs(bal)) and abs(float(r.z_loss) - z) <= 1e-5 * max(1, abs(z))


def test_cpu_gradient_is_finite_beside_dead_and_masked_rows():
    logits = torch.randn(6, 5)
    logits[1] = float("-inf")
    logits[2, 3] = float("-inf")
    logits[4] = float("nan")
    logits.requires_grad_()
    r = ep_moe.route_topk_train(logits, 2, token_mask=torch.tensor([1, 1, 1, 1, 0, 1], dtype=torch.bool))
    (r.balance_loss + r.z_loss).backward()
    assert torch.isfinite(logits.grad[[0, 1, 2, 3, 5]]).all() and not logits.grad[1].any()


def test_refusals():
    x = torch.zeros(4, 8)
    for bad in (dict(k=0), dict(k=9), dict(k=2, mode=2)):
        with pytest.raises(ValueError):
            ep_moe.route_topk_train(x, **bad)
    with pytest.raises(ValueError):
        ep_moe.route_topk_train(torch.zeros(8), 2)
    with pytest.raises(TypeError):
        ep_moe.route_topk_train(x.double(), 2)
    for mask in (torch.ones(4), torch.ones(5, dtype=torch.bool), torch.ones(4, 1, dtype=torch.bool)):
        with pytest.raises(ValueError):
            ep_moe.route_topk_train(x, 2, token_mask=mask)
    with pytest.raises(RuntimeError, match="CUDA"):
        nf4_qlora.glu_train(torch.zeros(2, 8, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="act is"):
        nf4_qlora.glu_train(torch.zeros(2, 8, dtype=torch.bfloat16), "relu")
    with pytest.raises(ValueError, match="rows is"):
        nf4_qlora.ffn_mxfp4_grouped_train(x, x, x, x, x, [4], [0], rows="fp8")


def test_c_entry_points_check_before_they_launch():
    lib = _gnf4b.load()
    buf = ctypes.create_string_buffer(1024)
    p = (ctypes.addressof(buf) + 63) // 64 * 64

    def fwd(dtype=0, T=4, stride=8, E=8, k=2, mode=0, norm=0, lg=p, counts=p, idx=p):
        return lib.gnf4b_route_train_fwd(lg, dtype, T, stride, E, k, mode, norm, None, idx, p, p, counts, p, p, p, None, 0, None)

    assert fwd(dtype=3) == -1 and fwd(T=-1) == -1 and fwd(mode=2) == -1 and fwd(norm=2) == -1
    assert fwd(E=0) == -2 and fwd(k=0) == -2 and fwd(k=9) == -2 and fwd(stride=-8) == -2
    assert fwd(E=2048, stride=2048) == -6 and fwd(E=64, k=33) == -6 and fwd(T=1 << 31) == -6
    assert fwd(lg=None) == -1 and fwd(counts=None) == -1 and fwd(idx=None) == -1

    def bwd(T=4, k=2, grad=p, w=p):
        return lib.gnf4b_route_train_bwd(p, 0, T, 8, 8, k, 0, 0, None, p, w, p, p, p, None, None, None, grad, None)

    assert bwd(T=-1) == -1 and bwd(k=9) == -2 and bwd(grad=None) == -1 and bwd(w=None) == -1 and bwd(T=0) == 0
    f = lib.gnf4b_glu_ckpt8_fwd
    assert f(p, -1, 8, 0, None, None, 0, p, p, p, None, None) == -1 and f(p, 1, 8, 2, None, None, 0, p, p, p, None, None) == -1
    assert f(p, 1, 0, 0, None, None, 0, p, p, p, None, None) == -2
    assert f(p, 1, 8, 0, p, p, 1, p, p, p, None, None) == -1 and f(p, 1, 8, 1, p, None, 1, p, p, p, None, None) == -1
    assert f(p, 1, 8, 0, None, None, 0, p, p, None, None, None) == -1 and f(p, 1, 8, 0, None, None, 0, None, p, p, None, None) == -1
    assert f(p, 1, 8, 0, None, None, 0, p, p + 4, p, None, None) == -1 and f(p, 1 << 60, 8, 0, None, None, 0, p, p, p, None, None) == -6
    assert f(None, 0, 8, 0, None, None, 0, None, None, None, None, None) == 0
    b = lib.gnf4b_glu_ckpt8_bwd
    assert b(p, p, p, -1, 8, 0, p, None) == -1 and b(p, p, p, 1, 8, 3, p, None) == -1 and b(p, p, p, 1, 0, 0, p, None) == -2
    assert b(p, None, p, 1, 8, 0, p, None) == -1 and b(p, p, p + 4, 1, 8, 0, p, None) == -1 and b(p, p, p, 0, 8, 0, p, None) == 0
