"""The CTA-pair form of the product of two MXFP4 operands.  Every case asks the library's own plan first that pairs are what it
would take, so that a moved threshold cannot leave the form untested."""
import ctypes

import pytest
import torch

import _gnf4b
import mxfp4_grouped as M
import nf4_grouped
from mxfp4_pack_ref import dequant_mxfp4

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def gen(seed):
    return torch.Generator().manual_seed(seed)


def takes_pairs(T, G, N, K, max_rows=-1):
    lib = _gnf4b.load()
    sms, smem = ctypes.c_int32(), ctypes.c_int32()
    plan = (ctypes.c_int32 * 9)()
    assert lib.gnf4b_device_info(ctypes.byref(sms), ctypes.byref(smem)) == 0
    assert lib.gnf4b_w4a4_plan(T, G, N, K, max_rows, sms.value, smem.value, plan) == 0
    return plan[0] == 1


def packed(rows, K, seed, lo=120, hi=130):
    g = gen(seed)
    return (torch.randint(0, 256, (*rows, K // 2), dtype=torch.uint8, generator=g).to(DEV),
            torch.randint(lo, hi, (*rows, K // 32), dtype=torch.uint8, generator=g).to(DEV))


def values64(blocks, scales):
    """Packed rows as fp64 numbers (the table decode, exact in fp32)."""
    return dequant_mxfp4(blocks.reshape(*blocks.shape[:-1], -1, 16), scales).double()


def check(out, xb, xs, wb, ws, sizes, ids):
    """One rounding to bf16 is 2^-8 of the value; K exact products added in fp32 are off by at most K steps of 2^-23 of the sum of
    magnitudes (a step may be cut off instead of rounded)."""
    K, first = 2 * xb.shape[1], 0
    for n, e in zip(sizes, ids):
        if n and e >= 0:
            rows = slice(first, first + n)
            ref = values64(xb[rows], xs[rows]) @ values64(wb[e], ws[e]).t()
            mags = values64(xb[rows] & 0x77, xs[rows]) @ values64(wb[e] & 0x77, ws[e]).t()
            off = (out[rows].double() - ref).abs() - (ref.abs() * 2.0 ** -8 + mags * K * 2.0 ** -23)
            assert off.isfinite().all() and not (off > 0).any(), (n, e, int((off > 0).sum()), float(off.max()))
        first += n


SIZES = [[400], [401, 1, 0, 17], [511], [513], [1000, 16, 33], [1, 385, 0, 64, 770]]


@pytest.mark.parametrize("sizes", SIZES)
@pytest.mark.parametrize("N", [2, 61, 128, 200, 256, 320, 384, 1000, 1001])
def test_shapes(N, sizes):
    """Widths that leave the second CTA's tile empty (up to 128 behind the last 256), partly filled or odd."""
    E, K = 3, 1312
    assert takes_pairs(sum(sizes), len(sizes), N, K, max(sizes))
    wb, ws = packed((E, N), K, 1)
    xb, xs = packed((sum(sizes),), K, 2)
    ids = [(2 * i + 1) % E for i in range(len(sizes))]
    check(M.gemm_mxfp4_grouped_w4a4(xb, xs, wb, ws, sizes, ids), xb, xs, wb, ws, sizes, ids)
    assert nf4_grouped.last_status(DEV) == 0


@pytest.mark.parametrize("K", [1344, 1568, 1792, 2048, 2080, 2880, 2912, 4128, 5152])
def test_lengths(K):
    """Whole and broken last stages and spans of scales; scale rows on 16 bytes, on 8, on none; rows on and off 128 bytes."""
    E, N, sizes, ids = 2, 300, [450, 0, 5, 384], [1, 0, 0, 1]
    assert takes_pairs(sum(sizes), 4, N, K, max(sizes))
    wb, ws = packed((E, N), K, 3)
    xb, xs = packed((sum(sizes),), K, 4)
    check(M.gemm_mxfp4_grouped_w4a4(xb, xs, wb, ws, sizes, ids), xb, xs, wb, ws, sizes, ids)
    assert nf4_grouped.last_status(DEV) == 0


@pytest.mark.parametrize("N,G", [(8192, 12), (3001, 33)])
def test_many_items_per_pair(N, G):
    """Several turns of the stage ring, the scale ring and the accumulator on every pair."""
    E, K = 4, 1312
    sizes = [384 + 29 * (i % 7) if i % 5 else 3 + i for i in range(G)]
    ids = [(3 * i) % E for i in range(G)]
    assert takes_pairs(sum(sizes), G, N, K, max(sizes))
    wb, ws = packed((E, N), K, 5)
    xb, xs = packed((sum(sizes),), K, 6)
    check(M.gemm_mxfp4_grouped_w4a4(xb, xs, wb, ws, sizes, ids), xb, xs, wb, ws, sizes, ids)
    assert nf4_grouped.last_status(DEV) == 0


def test_hundreds_of_items_per_pair():
    G, K, N = 200, 1344, 40960
    sizes = [(1, 3, 2)[i % 3] for i in range(G)]
    ids = [i % 2 for i in range(G)]
    T = sum(sizes)
    assert takes_pairs(T, G, N, K, 400) and G * (N // 256) > 256 * 74
    wb, ws = packed((2, N), K, 7)
    xb, xs = packed((T,), K, 8)
    off = torch.tensor([0, *torch.tensor(sizes).cumsum(0).tolist()], dtype=torch.int32, device=DEV)
    out = M.gemm_mxfp4_grouped_w4a4(xb, xs, wb, ws, None, torch.tensor(ids, device=DEV), group_offsets=off, max_rows=400)
    expert = torch.tensor(ids).repeat_interleave(torch.tensor(sizes)).to(DEV)
    order = torch.argsort(expert, stable=True)
    check(out[order], xb[order], xs[order], wb, ws, torch.bincount(expert).tolist(), [0, 1])
    assert nf4_grouped.last_status(DEV) == 0


def test_row_counts_unknown_to_the_host():
    """Device tables, no hint: any group may be long, so pairs also take batches of short ones; more groups than one table."""
    E, K, N, G = 5, 1312, 264, 700
    sizes = [(i * 7) % 3 for i in range(G)]
    sizes[650] = 290
    ids = [(i * 3) % E for i in range(G)]
    T = sum(sizes)
    assert takes_pairs(T, G, N, K)
    wb, ws = packed((E, N), K, 9)
    xb, xs = packed((T,), K, 10)
    off = torch.tensor([0, *torch.tensor(sizes).cumsum(0).tolist()], dtype=torch.int32, device=DEV)
    out = M.gemm_mxfp4_grouped_w4a4(xb, xs, wb, ws, None, torch.tensor(ids, device=DEV), group_offsets=off)
    check(out, xb, xs, wb, ws, sizes, ids)
    again = M.gemm_mxfp4_grouped_w4a4(xb, xs, wb, ws, torch.tensor(sizes, device=DEV), torch.tensor(ids, device=DEV))
    assert torch.equal(out, again) and nf4_grouped.last_status(DEV) == 0


def test_padding_bad_ids_and_rows_outside():
    """A padding group, an id outside the stack and rows behind the last group: output rows left as they were."""
    K, N, T = 1312, 136, 1200
    assert takes_pairs(T, 4, N, K)
    wb, ws = packed((2, N), K, 11)
    xb, xs = packed((T,), K, 12)
    off = torch.tensor([0, 400, 430, 820, 1100], dtype=torch.int32, device=DEV)
    ids = torch.tensor([1, -1, 7, 0], dtype=torch.int32, device=DEV)
    out = torch.full((T, N), 77.0, dtype=torch.bfloat16, device=DEV)
    nf4_grouped.last_status(DEV)
    rc = _gnf4b.load().gnf4b_gemm_grouped_w4a4(xb.data_ptr(), xs.data_ptr(), T, wb.data_ptr(), wb.stride(0), wb.stride(1), ws.data_ptr(),
                                               ws.stride(0), ws.stride(1), off.data_ptr(), ids.data_ptr(), 4, 2, N, K, -1, out.data_ptr(),
                                               nf4_grouped._status_ptr(torch.device(DEV)), torch.cuda.current_stream().cuda_stream)
    assert rc == 0 and nf4_grouped.last_status(DEV) == _gnf4b.ST_BAD_EXPERT
    assert (out[400:820] == 77).all() and (out[1100:] == 77).all()
    check(out, xb, xs, wb, ws, [400, 30, 390, 280], [1, -1, -1, 0])


def test_a_marked_block_stays_in_its_row():
    K, N, sizes, ids = 1312, 200, [390, 400], [1, 0]
    assert takes_pairs(790, 2, N, K, 400)
    wb, ws = packed((2, N), K, 13)
    xb, xs = packed((790,), K, 14)
    clean = M.gemm_mxfp4_grouped_w4a4(xb, xs, wb, ws, sizes, ids)
    xs[389, 40], xs[390, 0] = 255, 255
    out = M.gemm_mxfp4_grouped_w4a4(xb, xs, wb, ws, sizes, ids)
    bad = torch.zeros(790, dtype=torch.bool, device=DEV)
    bad[389:391] = True
    assert torch.isnan(out[bad]).all() and torch.equal(out[~bad], clean[~bad])


def test_streams_graphs_and_chains():
    """Products one after the other (the next launch begins while this one ends), two graphs of the same buffers on two streams."""
    K, N, E, T = 1312, 1344, 3, 1000
    assert takes_pairs(T, 3, N, K, 600) and takes_pairs(T, 3, K, N, 600)
    wb, ws = packed((E, N), K, 15, 116, 122)
    vb, vs = packed((E, K), N, 16, 116, 122)
    xb, xs = packed((T,), K, 17, 122, 126)
    off = torch.tensor([0, 400, 401, 1000], dtype=torch.int32, device=DEV)
    ids = torch.tensor([2, 0, 1], dtype=torch.int32, device=DEV)

    def chain():
        b, s = xb, xs
        for w in ((wb, ws), (vb, vs), (wb, ws)):
            y = M.gemm_mxfp4_grouped_w4a4(b, s, *w, None, ids, group_offsets=off, max_rows=600)
            b, s = M.quantize_mxfp4(y)
        return y

    def slowly():
        b, s = xb, xs
        for w in ((wb, ws), (vb, vs), (wb, ws)):
            y = M.gemm_mxfp4_grouped_w4a4(b, s, *w, None, ids, group_offsets=off, max_rows=600)
            torch.cuda.synchronize()
            b, s = M.quantize_mxfp4(y)
            torch.cuda.synchronize()
        return y

    want = slowly()
    assert torch.isfinite(want).all() and torch.equal(chain(), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = chain()
    assert torch.equal(chain(), want)
    side.synchronize()
    assert torch.equal(other, want)
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(chain())
        graphs.append(g)
    off.copy_(torch.tensor([0, 16, 600, 1000], dtype=torch.int32))
    torch.cuda.synchronize()
    graphs[0].replay()
    with torch.cuda.stream(side):
        graphs[1].replay()
    torch.cuda.synchronize()
    want = slowly()
    assert torch.equal(outs[0], want) and torch.equal(outs[1], want)
    assert nf4_grouped.last_status(DEV) == 0
