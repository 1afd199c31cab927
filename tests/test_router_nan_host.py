"""route_topk_train on CPU tensors: rows with a NaN or an infinity get the weights that route_topk gives.  No GPU needed."""
import pytest
import torch

import ep_moe


@pytest.mark.parametrize("mode,norm", [(0, False), (0, True), (1, False)])
def test_cpu_form_gives_the_weights_of_route_topk(mode, norm):
    x = torch.randn(8, 12, generator=torch.Generator().manual_seed(1))
    x[1, 5] = float("nan")
    x[2, 3] = float("inf")
    x[3, [1, 2]] = float("inf")
    x[4] = float("nan")
    x[5, 4] = float("-inf")
    r = ep_moe.route_topk_train(x, 3, mode, norm)
    idx, w = ep_moe.route_topk(x, 3, mode, norm)
    assert torch.equal(r.idx, idx) and torch.equal(torch.isnan(r.weights), torch.isnan(w))
    # a softmax of at most 12 terms on either side, and a second division
    torch.testing.assert_close(r.weights, w, rtol=32 * 2.0 ** -24, atol=0, equal_nan=True)
    assert torch.isnan(r.weights[1]).all() == (mode == 0)
