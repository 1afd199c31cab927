"""The low-rank delta beside padding groups (expert id -1): their rows have no delta and no part in any gradient.  No GPU needed."""
import pytest
import torch

import nf4_qlora as Q


@pytest.mark.parametrize("form", [Q.lora_delta_grouped, Q._lora_delta_grouped_loop])
def test_padding_groups_stay_out(form):
    E, r, K, N = 3, 2, 8, 5
    g = torch.Generator().manual_seed(1)
    sizes, ids = [4, 3, 0, 5], [1, -1, 0, 2]
    x = torch.randn(12, K, generator=g)
    A, B = torch.randn(E, r, K, generator=g), torch.randn(E, N, r, generator=g)
    go = torch.randn(12, N, generator=g)
    x[5], go[6] = float("nan"), float("nan")                  # of the padding group: memory that nobody wrote
    leaves = [t.clone().requires_grad_() for t in (x, A, B)]
    d = form(*leaves, sizes, ids, 0.5)
    grads = torch.autograd.grad(d, leaves, go)
    assert not d[4:7].any() and not grads[0][4:7].any()
    keep = [0, 1, 2, 3, 7, 8, 9, 10, 11]
    clean = [x[keep].clone().requires_grad_(), *(t.clone().requires_grad_() for t in (A, B))]
    want = form(*clean, [4, 5], [1, 2], 0.5)
    want_grads = torch.autograd.grad(want, clean, go[keep])
    # the same short sums, at most in another order: a few steps of 2^-23 of sums of up to 8 terms of order one
    for a, b in ((d[keep], want), (grads[0][keep], want_grads[0]), (grads[1], want_grads[1]), (grads[2], want_grads[2])):
        torch.testing.assert_close(a, b, rtol=1e-5, atol=1e-5)
