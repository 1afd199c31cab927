"""Calls of the training operators at the edges of what their documentation allows."""
import pytest
import torch

import mxfp4_grouped as M
import nf4_qlora as Q
import synth
from mxfp4_pack_ref import dequant_mxfp4

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
