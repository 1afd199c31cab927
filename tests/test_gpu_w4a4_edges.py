"""Calls of the product of two MXFP4 operands at the edges of what its documentation allows."""
import pytest
import torch

import mxfp4_grouped as M
import nf4_grouped

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def gen(seed):
    return torch.Generator().manual_seed(seed)


def packed(rows, K, seed, lo=120, hi=130):
    g = gen(seed)
    return (torch.randint(0, 256, (*rows, K // 2), dtype=torch.uint8, generator=g).to(DEV),
            torch.randint(lo, hi, (*rows, K // 32), dtype=torch.uint8, generator=g).to(DEV))


def test_rows_without_a_stack_are_refused():
    wb, ws = packed((2, 16), 64, 1)
    xb, xs = packed((5,), 64, 2)
    ids = torch.zeros(1, dtype=torch.int32, device=DEV)
    off = torch.tensor([0, 5], dtype=torch.int32, device=DEV)
    for tables in (dict(sizes=[5], expert_ids=[0]), dict(sizes=None, expert_ids=ids, group_offsets=off),
                   dict(sizes=torch.tensor([5], device=DEV), expert_ids=ids)):
        with pytest.raises(ValueError, match="no experts"):
            M.gemm_mxfp4_grouped_w4a4(xb, xs, wb[:0], ws[:0], **tables)
    assert M.gemm_mxfp4_grouped_w4a4(xb[:0], xs[:0], wb[:0], ws[:0], [], []).shape == (0, 16)
