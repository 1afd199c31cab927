"""MXFP4 quantiser, and the grouped product whose two operands are MXFP4, against plain 64-bit implementations."""
import numpy as np
import pytest
import torch

import mxfp4_grouped as M
import nf4_grouped
from mxfp4_pack_ref import dequant_mxfp4, quantize_pack_mxfp4

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def gen(seed):
    return torch.Generator().manual_seed(seed)


def values64(blocks, scales):
    """Packed rows as fp64 numbers, on the CPU (the framework's table decode, exact in fp32)."""
    b = blocks.cpu()
    return dequant_mxfp4(b.reshape(*b.shape[:-1], -1, 16), scales.cpu()).double()


def pack_ref(x):
    """quantize_pack_mxfp4 with its exponent taken exactly: its fp32 log2 can be off at the borders of an octave."""
    xb = x.double().reshape(*x.shape[:-1], x.shape[-1] // 32, 32)
    top = xb.abs().amax(-1).clamp_min(float(torch.tensor(1e-20)))
    m, p = torch.frexp(top / 4.0)
    e = torch.where(m <= 0.75, p - 1, p)
    v = torch.ldexp(xb, -e[..., None])
    table = torch.tensor(M.FP4_VALUES, dtype=torch.float64)
    codes = (v[..., None] - table).abs().argmin(-1).to(torch.uint8)
    return (codes[..., 0::2] | (codes[..., 1::2] << 4)).reshape(*x.shape[:-1], x.shape[-1] // 2), (e + 127).to(torch.uint8)


def packed(rows, K, seed, lo=120, hi=130):
    g = gen(seed)
    return (torch.randint(0, 256, (*rows, K // 2), dtype=torch.uint8, generator=g).to(DEV),
            torch.randint(lo, hi, (*rows, K // 32), dtype=torch.uint8, generator=g).to(DEV))


def product64(xb, xs, wb, ws, sizes, ids):
    x, out, first = values64(xb, xs), [], 0
    for n, e in zip(sizes, ids):
        out.append(x[first:first + n] @ values64(wb[e], ws[e]).t())
        first += n
    return torch.cat(out), first


# one rounding to bf16 is 2^-8 of the value; the fp32 accumulation of K exact products is off by at most K rounding
# steps of 2^-24 of the sum of magnitudes (the tensor core may truncate, hence a whole step each)
def check_product(out, ref, mags, K):
    tol = ref.abs() * 2.0 ** -8 + mags * K * 2.0 ** -23
    bad = (out.cpu().double() - ref).abs() > tol
    assert not bad.any(), (int(bad.sum()), float(((out.cpu().double() - ref).abs() - tol).max()))


# ------------------------------------------------------------------------------------------------ quantiser
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("shape", [(1, 32), (3, 64), (7, 2880), (129, 96), (2, 3, 160), (5000, 512)])
def test_quantize_bytes(dtype, shape):
    x = (torch.randn(*shape, generator=gen(1)) * torch.exp2(torch.randint(-9, 10, shape, generator=gen(2)).float())).to(dtype)
    b, s = M.quantize_mxfp4(x.to(DEV))
    rb, rs = pack_ref(x)
    assert b.shape == (*shape[:-1], shape[-1] // 2) and s.shape == (*shape[:-1], shape[-1] // 32)
    assert torch.equal(s.cpu(), rs)
    assert torch.equal(b.cpu(), rb)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_quantize_ties_and_borders(dtype):
    ties = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 0.0, -0.0])
    eps = torch.finfo(dtype).eps
    near = torch.cat([ties, ties * (1 + eps), ties * (1 - eps / 2)])
    near = torch.cat([near, -near])                                       # 96 values
    rows = [near * 2.0 ** k for k in (-12, -3, 0, 2, 9)]
    rows += [torch.cat([r.new_tensor([6.0 * (1 + eps)]), r[1:]]) for r in rows[2:3]]
    x = torch.stack(rows).to(dtype)
    b, s = M.quantize_mxfp4(x.to(DEV))
    rb, rs = pack_ref(x)
    assert torch.equal(s.cpu(), rs) and torch.equal(b.cpu(), rb)
    # the block exponent's own border, each number the only one of its block
    tops = torch.cat([torch.tensor([1.5, 6.0, 3.0, 0.75]) * f for f in (1 - eps / 2, 1.0, 1 + eps)]).to(dtype)
    x = torch.zeros(tops.numel(), 32, dtype=dtype)
    x[:, 5] = tops
    b, s = M.quantize_mxfp4(x.to(DEV))
    rb, rs = pack_ref(x)
    assert torch.equal(s.cpu(), rs) and torch.equal(b.cpu(), rb)


def test_quantize_equals_the_reference_packer():
    x = torch.randn(37, 256, generator=gen(3)).to(torch.bfloat16)
    b, s = M.quantize_mxfp4(x.to(DEV))
    rb, rs = quantize_pack_mxfp4(x)
    assert torch.equal(s.cpu(), rs) and torch.equal(b.cpu(), rb.reshape(37, -1))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_quantize_zero_tiny_and_huge(dtype):
    fi = torch.finfo(dtype)
    x = torch.zeros(6, 64, dtype=dtype)
    x[1, 3] = fi.smallest_normal
    x[2, 7] = fi.max
    x[2, 40] = -fi.max
    x[3] = fi.min
    x[4, 1] = fi.smallest_normal * 2.0 ** -7 if dtype != torch.float16 else 2.0 ** -24
    x[5] = 1e-4
    b, s = M.quantize_mxfp4(x.to(DEV))
    rb, rs = pack_ref(x)
    assert torch.equal(s.cpu(), rs) and torch.equal(b.cpu(), rb)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_quantize_nonfinite_blocks_are_marked(dtype, bad):
    x = torch.randn(3, 96, generator=gen(4)).to(dtype)
    clean_b, clean_s = M.quantize_mxfp4(x.to(DEV))
    x[1, 40] = bad
    b, s = M.quantize_mxfp4(x.to(DEV))
    assert s[1, 1] == 255 and not torch.isfinite(M.dequantize_mxfp4(b, s)[1, 32:64]).any()
    s[1, 1], b[1, 16:32] = clean_s[1, 1], clean_b[1, 16:32]
    assert torch.equal(b, clean_b) and torch.equal(s, clean_s)            # the neighbours are what they were


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_quantize_views(dtype):
    big = torch.randn(40, 200, generator=gen(5)).to(dtype).to(DEV)
    for view in (big[:, 8:72], big[:, 3:67], big[::3, 16:112], big[5], big[5, 8:40], big[:1, 64:128], big[:32, :64].t(),
                 big[:1, :64].expand(6, 64), big[0:0, :64]):
        view = view[..., :view.shape[-1] // 32 * 32]
        b, s = M.quantize_mxfp4(view)
        rb, rs = pack_ref(view.cpu())
        assert torch.equal(s.cpu(), rs) and torch.equal(b.cpu(), rb), view.shape


@pytest.mark.parametrize("shape", [(64,), (0, 32), (2, 0, 96), (1, 1, 1, 32), (3, 2, 2, 64)])
def test_quantize_and_back_any_rank(shape):
    x = torch.randn(*shape, generator=gen(31)).to(torch.bfloat16)
    b, s = M.quantize_mxfp4(x.to(DEV))
    assert b.shape == (*shape[:-1], shape[-1] // 2) and s.shape == (*shape[:-1], shape[-1] // 32)
    back = M.dequantize_mxfp4(b, s)
    assert back.shape == x.shape
    if x.numel():
        rb, rs = M.quantize_mxfp4(x.reshape(-1, shape[-1]).to(DEV))
        assert torch.equal(b.reshape(rb.shape), rb) and torch.equal(back.reshape(-1, shape[-1]), M.dequantize_mxfp4(rb, rs))
    with pytest.raises(ValueError):
        M.dequantize_mxfp4(b, s[..., :-1])
    with pytest.raises(ValueError):
        M.dequantize_mxfp4(b[None], s)


def test_dequantize_every_byte_and_exponent():
    b = torch.arange(256, dtype=torch.uint8).reshape(16, 16).repeat(256, 1)          # every byte under every exponent
    s = torch.arange(256, dtype=torch.uint8).repeat_interleave(16)[:, None]
    ref = dequant_mxfp4(b.reshape(-1, 1, 16), s)
    got = M.dequantize_mxfp4(b.to(DEV), s.to(DEV), torch.float32).cpu()
    assert torch.equal(got.view(torch.int32), ref.view(torch.int32))
    assert torch.equal(M.dequantize_mxfp4(b.to(DEV), s.to(DEV)).cpu().view(torch.int16), ref.to(torch.bfloat16).view(torch.int16))
    assert torch.equal(M.dequantize_mxfp4(b.to(DEV), s.to(DEV), torch.float16).cpu().view(torch.int16), ref.half().view(torch.int16))


@pytest.mark.parametrize("act", ["silu", "gpt_oss"])
@pytest.mark.parametrize("rows,h", [(1, 32), (5, 96), (33, 768), (260, 2880)])
def test_glu_quantize_is_glu_then_quantize(act, rows, h):
    import ep_moe
    gu = (3 * torch.randn(rows, 2 * h, generator=gen(6))).to(torch.bfloat16).to(DEV)
    want = M.quantize_mxfp4(ep_moe.silu_glu(gu) if act == "silu" else M.glu_gpt_oss(gu))
    got = M.glu_quantize_mxfp4(gu, act)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    shifted = torch.empty(gu.numel() + 1, dtype=gu.dtype, device=DEV)[1:].reshape(rows, 2 * h).copy_(gu)    # not 16-byte aligned
    got = M.glu_quantize_mxfp4(shifted, act)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    if act == "gpt_oss":
        bias = torch.randn(3, 2 * h, generator=gen(7)).to(torch.bfloat16).to(DEV)
        who = torch.randint(0, 3, (rows,), generator=gen(8)).to(DEV)
        want = M.quantize_mxfp4(M.glu_gpt_oss(gu, bias, who))
        got = M.glu_quantize_mxfp4(gu, act, bias, who)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_glu_quantize_flags_a_bad_expert():
    gu = torch.randn(4, 64, generator=gen(9)).to(torch.bfloat16).to(DEV)
    bias = torch.zeros(2, 64, dtype=torch.bfloat16, device=DEV)
    nf4_grouped.last_status(DEV)
    M.glu_quantize_mxfp4(gu, "gpt_oss", bias, torch.tensor([0, 5, 1, -1], device=DEV))
    assert nf4_grouped.last_status(DEV) == 1
    assert nf4_grouped.last_status(DEV) == 0


# ------------------------------------------------------------------------------------------------ product
@pytest.mark.parametrize("K", [32, 64, 96, 256, 288, 768, 1056, 2880])
@pytest.mark.parametrize("N", [1, 8, 61, 128, 200])
def test_product_shapes(K, N):
    sizes, ids = [1, 0, 17, 3], [2, 0, 1, 2]
    wb, ws = packed((3, N), K, 10)
    xb, xs = packed((sum(sizes),), K, 11)
    out = M.gemm_mxfp4_grouped_w4a4(xb, xs, wb, ws, sizes, ids)
    ref, _ = product64(xb, xs, wb, ws, sizes, ids)
    mags, _ = product64(xb & 0x77, xs, wb & 0x77, ws, sizes, ids)
    check_product(out, ref, mags, K)
    assert nf4_grouped.last_status(DEV) == 0


@pytest.mark.parametrize("sizes", [[1], [15], [16], [17], [33], [64], [65], [127], [128], [129], [144], [200], [255], [256], [257],
                                   [513], [1000], [1, 300, 2, 129, 0, 64], [1] * 40, [700, 1]])
def test_product_group_sizes(sizes):
    K, N, E = 352, 192, 5
    ids = [(3 * i + 1) % E for i in range(len(sizes))]
    wb, ws = packed((E, N), K, 12)
    xb, xs = packed((sum(sizes),), K, 13)
    out = M.gemm_mxfp4_grouped_w4a4(xb, xs, wb, ws, sizes, ids)
    ref, _ = product64(xb, xs, wb, ws, sizes, ids)
    mags, _ = product64(xb & 0x77, xs, wb & 0x77, ws, sizes, ids)
    check_product(out, ref, mags, K)


@pytest.mark.parametrize("rows", [3, 20, 100, 190])
def test_product_many_items_per_sm(rows):
    """Several items, several turns of the stage ring and of the scale ring on every SM (and SM pair, from 128 rows on),
    an odd number of tiles."""
    G, E, K = 40, 6, 2080
    N = 1200 if rows > 50 else 5000
    sizes = [rows + (7 * i) % 90 if rows > 50 else rows for i in range(G)]
    ids = [(5 * i) % E for i in range(G)]
    wb, ws = packed((E, N), K, 40)
    xb, xs = packed((sum(sizes),), K, 41)
    out = M.gemm_mxfp4_grouped_w4a4(xb, xs, wb, ws, sizes, ids)
    w, m = ([values64(b, ws[e]).to(DEV) for e, b in enumerate(v)] for v in (wb, wb & 0x77))
    x, a = (values64(v, xs).to(DEV).split(sizes) for v in (xb, xb & 0x77))
    ref = torch.cat([v @ w[e].t() for v, e in zip(x, ids)]).cpu()
    mags = torch.cat([v @ m[e].t() for v, e in zip(a, ids)]).cpu()
    check_product(out, ref, mags, K)
    assert nf4_grouped.last_status(DEV) == 0


@pytest.mark.parametrize("max_rows", [None, 1, 7, 40, 300])
def test_product_device_tables_and_row_hints(max_rows):
    """max_rows shapes the tiles only: unknown, understated and overstated give the same bits."""
    sizes, ids, K, N = [3, 0, 40, 1, 290], [0, 3, 1, 2, 0], 544, 136
    wb, ws = packed((4, N), K, 14)
    xb, xs = packed((sum(sizes),), K, 15)
    want = M.gemm_mxfp4_grouped_w4a4(xb, xs, wb, ws, sizes, ids)
    off = torch.tensor([0] + list(np.cumsum(sizes)), dtype=torch.int32, device=DEV)
    got = M.gemm_mxfp4_grouped_w4a4(xb, xs, wb, ws, None, torch.tensor(ids, device=DEV), group_offsets=off, max_rows=max_rows)
    assert torch.equal(got, want)
    got = M.gemm_mxfp4_grouped_w4a4(xb, xs, wb, ws, torch.tensor(sizes, device=DEV), torch.tensor(ids, device=DEV))
    assert torch.equal(got, want)


def test_product_more_groups_than_one_table():
    G, K, N, E = 1500, 64, 72, 7
    sizes = [(i * 7) % 3 for i in range(G)]
    ids = [(i * 5) % E for i in range(G)]
    wb, ws = packed((E, N), K, 16)
    xb, xs = packed((sum(sizes),), K, 17)
    out = M.gemm_mxfp4_grouped_w4a4(xb, xs, wb, ws, sizes, ids)
    ref, _ = product64(xb, xs, wb, ws, sizes, ids)
    mags, _ = product64(xb & 0x77, xs, wb & 0x77, ws, sizes, ids)
    check_product(out, ref, mags, K)


def test_product_padding_bad_ids_and_rows_outside():
    """A padding group, an id outside the stack and rows behind the last group: output rows left as they were."""
    import _gnf4b
    K, N, T = 128, 64, 40
    wb, ws = packed((2, N), K, 18)
    xb, xs = packed((T,), K, 19)
    off = torch.tensor([0, 5, 9, 12, 30], dtype=torch.int32, device=DEV)
    ids = torch.tensor([1, -1, 7, 0], dtype=torch.int32, device=DEV)
    out = torch.full((T, N), 77.0, dtype=torch.bfloat16, device=DEV)
    nf4_grouped.last_status(DEV)
    rc = _gnf4b.load().gnf4b_gemm_grouped_w4a4(xb.data_ptr(), xs.data_ptr(), T, wb.data_ptr(), wb.stride(0), wb.stride(1), ws.data_ptr(),
                                               ws.stride(0), ws.stride(1), off.data_ptr(), ids.data_ptr(), 4, 2, N, K, -1, out.data_ptr(),
                                               nf4_grouped._status_ptr(torch.device(DEV)), torch.cuda.current_stream().cuda_stream)
    assert rc == 0 and nf4_grouped.last_status(DEV) == _gnf4b.ST_BAD_EXPERT
    assert (out[5:12] == 77).all() and (out[30:] == 77).all()
    for lo, hi, e in ((0, 5, 1), (12, 30, 0)):
        want = M.gemm_mxfp4_grouped_w4a4(xb[lo:hi], xs[lo:hi], wb, ws, [hi - lo], [e])
        assert torch.equal(out[lo:hi], want)


def test_product_bad_offsets_are_skipped():
    import _gnf4b
    K, N, T = 64, 32, 10
    wb, ws = packed((1, N), K, 20)
    xb, xs = packed((T,), K, 21)
    nf4_grouped.last_status(DEV)
    ids = torch.zeros(3, dtype=torch.int32, device=DEV)
    for offs in ([0, 4, 2, 10], [0, 4, 8, 11], [-3, 4, 8, 10]):
        M.gemm_mxfp4_grouped_w4a4(xb, xs, wb, ws, None, ids, group_offsets=torch.tensor(offs, dtype=torch.int32, device=DEV))
        assert nf4_grouped.last_status(DEV) == _gnf4b.ST_BAD_OFFSETS, offs


def test_product_views_of_stacks_and_rows():
    K, N, E = 192, 48, 4
    big, bs = packed((E, 3 * N), 2 * K, 22)
    xb, xs = packed((23,), 2 * K, 23)
    sizes, ids = [9, 14], [3, 1]
    views = [(big[:, N:2 * N, :K // 2], bs[:, N:2 * N, :K // 32]),              # row and column ranges
             (big[:, ::3, K // 2:], bs[:, ::3, K // 32:]),                      # every third row
             (big[:, :N, 5:5 + K // 2], bs[:, :N, 1:1 + K // 32]),              # unaligned columns: copied
             (big[:1, :N, :K // 2].expand(E, N, K // 2), bs[:1, :N, :K // 32].expand(E, N, K // 32)),
             (big[:, :N, :K // 2].transpose(0, 1).contiguous().transpose(0, 1), bs[:, :N, :K // 32].transpose(0, 1).contiguous().transpose(0, 1))]
    xv = (xb[:, 16:16 + K // 2], xs[:, 1:1 + K // 32])
    for wb, ws in views:
        out = M.gemm_mxfp4_grouped_w4a4(*xv, wb, ws, sizes, ids)
        want = M.gemm_mxfp4_grouped_w4a4(xv[0].contiguous(), xv[1].contiguous(), wb.contiguous(), ws.contiguous(), sizes, ids)
        assert torch.equal(out, want)
        ref, _ = product64(*xv, wb, ws, sizes, ids)
        mags, _ = product64(xv[0] & 0x77, xv[1], wb & 0x77, ws, sizes, ids)
        check_product(out, ref, mags, K)


def test_product_extreme_scales_and_nan():
    K, N = 256, 16
    wb, ws = packed((1, N), K, 24, 0, 20)              # 2^-127 .. : products far below the fp32 range are zeros
    xb, xs = packed((4,), K, 25, 0, 20)
    assert not M.gemm_mxfp4_grouped_w4a4(xb, xs, wb, ws, [4], [0]).any()
    wb, ws = packed((1, N), K, 26, 0, 40)              # tiny times huge
    xb, xs = packed((4,), K, 27, 215, 250)
    out = M.gemm_mxfp4_grouped_w4a4(xb, xs, wb, ws, [4], [0])
    ref, _ = product64(xb, xs, wb, ws, [4], [0])
    mags, _ = product64(xb & 0x77, xs, wb & 0x77, ws, [4], [0])
    check_product(out, ref, mags, K)
    xs[2, 3] = 255
    nan = M.gemm_mxfp4_grouped_w4a4(xb, xs, wb, ws, [4], [0])
    assert torch.isnan(nan[2]).all() and torch.equal(nan[[0, 1, 3]], out[[0, 1, 3]])
    x = torch.randn(5, K, generator=gen(28)).to(DEV)
    x[1, 70] = float("inf")
    nan = M.gemm_mxfp4_grouped_w4a4(*M.quantize_mxfp4(x), wb, ws, [5], [0])
    assert torch.isnan(nan[1]).all() and torch.isfinite(nan[[0, 2, 3, 4]]).all()


@pytest.mark.parametrize("max_rows,K,N,G", [(3, 64, 20480, 256), (3, 1344, 20480, 256), (400, 1344, 40960, 130)])
def test_product_hundreds_of_items_per_sm(max_rows, K, N, G):
    """More than 256 items for every SM (and SM pair, the last case)."""
    wb, ws = packed((2, N), K, 60)
    xb, xs = packed((2 * G,), K, 61)
    sizes = [(1, 3, 2)[i % 3] for i in range(G)]
    ids = [i % 2 for i in range(G)]
    T = sum(sizes)
    xb, xs = xb[:T].contiguous(), xs[:T].contiguous()
    off = torch.tensor([0, *torch.tensor(sizes).cumsum(0).tolist()], dtype=torch.int32, device=DEV)
    out = M.gemm_mxfp4_grouped_w4a4(xb, xs, wb, ws, None, torch.tensor(ids, device=DEV), group_offsets=off, max_rows=max_rows)
    expert = torch.tensor(ids).repeat_interleave(torch.tensor(sizes)).to(DEV)
    for e in range(2):                                     # all of an expert's rows as one group: the same sums
        rows = torch.nonzero(expert == e).reshape(-1)
        assert torch.equal(out[rows], M.gemm_mxfp4_grouped_w4a4(xb[rows], xs[rows], wb, ws, [len(rows)], [e]))


def test_product_beyond_32_bit_offsets():
    """A stack of more than 4 GiB: the last expert against its own copy."""
    E, N, K = 300, 4096, 7168
    wb = torch.randint(0, 256, (E, N, K // 2), dtype=torch.uint8, device=DEV)
    ws = torch.randint(120, 126, (E, N, K // 32), dtype=torch.uint8, device=DEV)
    xb, xs = packed((5,), K, 42)
    out = M.gemm_mxfp4_grouped_w4a4(xb, xs, wb, ws, [2, 3], [E - 1, 0])
    for lo, hi, e in ((0, 2, E - 1), (2, 5, 0)):
        assert torch.equal(out[lo:hi], M.gemm_mxfp4_grouped_w4a4(xb[lo:hi], xs[lo:hi], wb[e:e + 1].clone(), ws[e:e + 1].clone(), [hi - lo], [0]))


def test_quantize_beyond_32_bit_offsets():
    rows, K = 70000, 32 * 1000
    x = torch.zeros(rows, K, dtype=torch.bfloat16, device=DEV)
    x[-3:] = torch.randn(3, K, generator=gen(43)).to(torch.bfloat16).to(DEV)
    b, s = M.quantize_mxfp4(x)
    rb, rs = pack_ref(x[-3:].cpu())
    assert torch.equal(b[-3:].cpu(), rb) and torch.equal(s[-3:].cpu(), rs)
    del x
    v = M.dequantize_mxfp4(b, s)
    assert torch.equal(v[-3:].cpu().double(), values64(rb, rs)) and not v[:-3].any()


def test_product_empty_calls():
    wb, ws = packed((2, 16), 64, 29)
    xb, xs = packed((0,), 64, 30)
    assert M.gemm_mxfp4_grouped_w4a4(xb, xs, wb, ws, [], []).shape == (0, 16)
    assert M.gemm_mxfp4_grouped_w4a4(xb, xs, wb, ws, [0, 0], [0, 1]).shape == (0, 16)


def test_product_on_other_streams_and_under_graphs():
    """Two graphs captured from the same buffers replay on two streams; routing changes under replay."""
    K, N, E, T = 512, 256, 6, 96
    wb, ws = packed((E, N), K, 31)
    xb, xs = packed((T,), K, 32)
    off = torch.tensor([0, 30, 31, 96], dtype=torch.int32, device=DEV)
    ids = torch.tensor([4, 0, 5], dtype=torch.int32, device=DEV)
    call = lambda: M.gemm_mxfp4_grouped_w4a4(xb, xs, wb, ws, None, ids, group_offsets=off, max_rows=65)  # noqa: E731
    want = call()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert torch.equal(call(), want)
    side.synchronize()
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(call())
        graphs.append(g)
    off.copy_(torch.tensor([0, 64, 64, 96], dtype=torch.int32))
    torch.cuda.synchronize()
    other = torch.cuda.Stream()
    graphs[0].replay()
    with torch.cuda.stream(other):
        graphs[1].replay()
    torch.cuda.synchronize()
    want = call()
    assert torch.equal(outs[0], want) and torch.equal(outs[1], want)


@pytest.mark.parametrize("act", ["silu", "gpt_oss"])
def test_ffn_w4a4_is_its_parts(act):
    E, K, h, N = 4, 128, 96, 160
    gub, gus = packed((E, 2 * h), K, 33, 118, 124)
    dnb, dns = packed((E, N), h, 34, 118, 124)
    x = torch.randn(50, K, generator=gen(35)).to(torch.bfloat16).to(DEV)
    sizes, ids = [1, 20, 29], [3, 0, 2]
    gu = M.gemm_mxfp4_grouped_w4a4(*M.quantize_mxfp4(x), gub, gus, sizes, ids)
    import ep_moe
    hrow = ep_moe.silu_glu(gu) if act == "silu" else M.glu_gpt_oss(gu)
    want = M.gemm_mxfp4_grouped_w4a4(*M.quantize_mxfp4(hrow), dnb, dns, sizes, ids)
    assert torch.equal(M.ffn_mxfp4_grouped_w4a4(x, gub, gus, dnb, dns, sizes, ids, act=act), want)
    assert torch.equal(M.ffn_mxfp4_grouped_w4a4(M.quantize_mxfp4(x), gub, gus, dnb, dns, sizes, ids, act=act), want)
