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


def test_two_host_threads_at_once():
    """Each thread on its own stream, over products of very different tiles, the quantiser, the router and the GLU."""
    import threading

    import ep_moe
    import nf4_qlora

    K, E, N = 1312, 3, 300
    wb, ws = packed((E, N), K, 5)
    batches = []
    for i, sizes in enumerate(([1, 1], [400, 3], [17, 0, 60], [130], [1, 300])):
        x = torch.randn(sum(sizes), K, generator=gen(20 + i)).to(torch.bfloat16).to(DEV)
        batches.append((x, sizes, [(i + j) % E for j in range(len(sizes))]))

    def one(x, sizes, ids):
        y = M.gemm_mxfp4_grouped_w4a4(*M.quantize_mxfp4(x), wb, ws, sizes, ids)
        logits = y.float().clamp(-4, 4).requires_grad_()
        r = ep_moe.route_topk_train(logits, 5)
        grad, = torch.autograd.grad((r.weights, r.z_loss), logits, (torch.ones_like(r.weights), torch.ones_like(r.z_loss)))
        gu = y.clamp(-4, 4).requires_grad_()
        out = nf4_qlora.glu_train(gu, "silu")
        return y, r.idx, r.balance_loss.detach(), grad, out.detach(), torch.autograd.grad(out, gu, torch.ones_like(out))[0]

    want = [one(*b) for b in batches]
    torch.cuda.synchronize()
    wrong = []

    def work(first):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for i in range(60):
                    b = (first + i * (1 + first)) % len(batches)
                    got = one(*batches[b])
                    torch.cuda.current_stream().synchronize()
                    if not all(torch.equal(p, q) for p, q in zip(got, want[b])):
                        wrong.append((first, i, b))
        except Exception as e:                          # a thread's exception would be lost
            wrong.append(repr(e))

    threads = [threading.Thread(target=work, args=(t,)) for t in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not wrong and nf4_grouped.last_status(DEV) == 0
