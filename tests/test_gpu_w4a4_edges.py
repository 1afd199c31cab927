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


def test_odd_strides_of_dimensions_of_one():
    """A stack of one row, or of one expert, cut out of wider memory: the stride that is not used may be anything."""
    K, T = 128, 7
    xb, xs = packed((T,), K, 3)
    big, bs = packed((4, 6), 2 * K, 4)
    flat, fs = big.reshape(-1), bs.reshape(-1)
    for shape, strides in (((4, 1, K // 2), (96, 72, 1)), ((4, 1, K // 2), (96, 5, 1)), ((1, 6, K // 2), (1000, 80, 1)),
                           ((1, 1, K // 2), (9, 7, 1))):
        wb = flat.as_strided(shape, strides)
        ws = fs.as_strided((*shape[:2], K // 32), (9, 5, 1))
        sizes, ids = [3, 4], [shape[0] - 1, 0]
        want = M.gemm_mxfp4_grouped_w4a4(xb, xs, wb.clone(memory_format=torch.contiguous_format),
                                         ws.clone(memory_format=torch.contiguous_format), sizes, ids)
        assert torch.equal(M.gemm_mxfp4_grouped_w4a4(xb, xs, wb, ws, sizes, ids), want)
    assert nf4_grouped.last_status(DEV) == 0
