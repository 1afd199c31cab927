"""Grouped W4A16 GEMM over native MXFP4 expert stacks on NVIDIA B200 -- the drop-in for
the reference module of the same name (pjordanandrsn/grouped-nf4-gemm,
kernel/mxfp4_grouped.py:134-172).

``out[t] = a[t] @ dequant_mxfp4(blocks[e(t)]).T`` for rows grouped by expert, one launch of
the sm_100a kernels in ``libgnf4b.so``.  Decode rules (ref :7-16): e2m1 codebook, element
2j in the LOW nibble of byte j, one e8m0 scale byte per 32 elements with value 2^(e-127).
The decode follows the ``ldexp`` semantics of ``mxfp4_pack_ref.dequant_mxfp4`` (a zero
element times the 0xFF scale stays zero).  Offsets are 64-bit throughout, so stacks beyond
2 GiB are fine (the reference's Triton kernel multiplies ``eid * stride`` in int32,
ref :65, 73).
"""
from __future__ import annotations

import torch

import _gnf4b
from nf4_grouped import (_call_on, _dispatch, _group_tables, _launch, _launch_ffn, _launch_host, _prefill_block_m,  # noqa: F401  (re-exported names)
                         _raw_stream, _require_cuda, _status_ptr, build_group_tiles)

# e2m1 codebook, index = (sign << 3) | magnitude (ref :34-35)
FP4_VALUES = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0,
              -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0]
MX_BLOCK = 32
E8M0_BIAS = 127

_LUT_CACHE: dict = {}


def _lut(device):
    key = str(device)
    if key not in _LUT_CACHE:
        _LUT_CACHE[key] = torch.tensor(FP4_VALUES, dtype=torch.float32, device=device)
    return _LUT_CACHE[key]


def gemm_mxfp4_grouped(a_cat, blocks, scales, sizes, expert_ids,
                       block_m: int | None = None, prefill_variant: int | None = None, *,
                       group_offsets=None, max_rows=None, path: int = 0, tables_ready: bool | None = None):
    """Single-launch grouped MXFP4 GEMM (ref :134-172).  ``a_cat [T,K]`` bf16/fp16 rows
    sorted by group; ``blocks [E,N,K//2]`` uint8; ``scales [E,N,K//32]`` uint8 (e8m0);
    ``sizes`` per-group row counts; ``expert_ids [G]`` list / CPU / CUDA int tensor.
    Returns ``[T,N]`` bf16 in the same row order.  ``block_m`` and ``prefill_variant`` are
    Triton knobs of the reference, accepted and ignored.  ``group_offsets`` / ``max_rows`` /
    ``path`` / ``tables_ready`` are the keyword-only additions described at ``nf4_grouped.gemm_4bit_grouped``."""
    E, N, _ = blocks.shape
    T, K = a_cat.shape
    assert scales.shape == (E, N, K // MX_BLOCK), (scales.shape, (E, N, K // MX_BLOCK))
    assert blocks.dtype == torch.uint8 and scales.dtype == torch.uint8
    _require_cuda(a_cat, "gemm_mxfp4_grouped",
                  "For a CPU-checkable decode of the same MXFP4 bytes, use "
                  "mxfp4_pack_ref.dequant_mxfp4(blocks, scales).")
    if blocks.shape[2] * 2 != K:
        raise ValueError(f"a_cat has K={K} but blocks pack K={blocks.shape[2] * 2}")
    return _dispatch(_gnf4b.FMT_MXFP4, _gnf4b.OP_FWD, a_cat, blocks, scales, sizes, expert_ids, N,
                     group_offsets=group_offsets, max_rows=max_rows, path=path, tables_ready=tables_ready)


def ffn_mxfp4_grouped(a_cat, blocks_gu, scales_gu, blocks_dn, scales_dn, sizes, expert_ids, *, act: str = "gpt_oss",
                      bias_gu=None, group_offsets=None, max_rows=None, tables_ready: bool | None = None,
                      fused: bool = True):
    """One MXFP4 expert FFN per row on CUDA tensors: ``act(a @ W_gu[e].T (+ bias_gu[e])) @ W_dn[e].T``.
    ``act="gpt_oss"``: gate and up interleaved in the gate_up columns, the clamped GLU of gpt-oss evaluated as the
    reference's chain of bf16 tensor operations (``kernel/mxfp4_pipelined.py:440-445, 453-461``); ``act="silu"``:
    SiLU(gate) * up over column halves.  ``bias_gu`` is an optional bf16 ``[E, N_gu]``.  Batch-1 decode (every group
    one row) runs as ONE kernel launch; the down bias and the router-weighted sum stay with the caller (fp32 there)."""
    if act not in ("gpt_oss", "silu"):
        raise ValueError("act is 'gpt_oss' or 'silu'")
    assert blocks_gu.dtype == torch.uint8 and scales_gu.dtype == torch.uint8
    assert blocks_dn.dtype == torch.uint8 and scales_dn.dtype == torch.uint8
    _require_cuda(a_cat, "ffn_mxfp4_grouped", "The CPU-checkable equivalent composes mxfp4_pack_ref.dequant_mxfp4 per expert.")
    return _launch_ffn(_gnf4b.FMT_MXFP4, _gnf4b.ACT_GPT_OSS_GLU if act == "gpt_oss" else _gnf4b.ACT_SILU_GLU, a_cat,
                       blocks_gu, scales_gu, blocks_dn, scales_dn, sizes, expert_ids, bias_gu=bias_gu,
                       group_offsets=group_offsets, max_rows=max_rows, tables_ready=tables_ready, fused=fused)


def glu_gpt_oss(gate_up, bias=None, row_expert=None):
    """The activation of gpt-oss between its expert GEMMs as one kernel: ``gate_up [rows, 2h]`` bf16 (gate and up
    interleaved) -> ``[rows, h]`` bf16; ``bias`` bf16 ``[E, 2h]`` is added first (row r takes ``bias[row_expert[r]]``)."""
    _require_cuda(gate_up, "glu_gpt_oss", "")
    gate_up = gate_up.contiguous()
    rows, two_h = gate_up.shape
    out = torch.empty(rows, two_h // 2, dtype=torch.bfloat16, device=gate_up.device)
    if bias is not None:
        bias = bias.contiguous()
        row_expert = row_expert.to(torch.int32).contiguous()
    lib = _gnf4b.load()
    with torch.cuda.device(gate_up.device):
        rc = lib.gnf4b_glu_gpt_oss(gate_up.data_ptr(), rows, two_h // 2, bias.data_ptr() if bias is not None else None,
                                   row_expert.data_ptr() if bias is not None else None, out.data_ptr(),
                                   torch.cuda.current_stream(gate_up.device).cuda_stream)
    _gnf4b.check(rc, "gnf4b_glu_gpt_oss")
    return out


def gemm_mxfp4_grouped_host(a_host, blocks, scales, sizes, expert_ids, out=None, *, path: int = 0,
                            return_status: bool = False):
    """``gemm_mxfp4_grouped`` with host activations, host group tables and a host result, the stack resident on
    the GPU: the calling convention of the reference's native CPU kernel
    (``gnf4_native/cpu_kernels.c:1097``).  See ``nf4_grouped.gemm_4bit_grouped_host``."""
    assert blocks.dtype == torch.uint8 and scales.dtype == torch.uint8
    return _launch_host(_gnf4b.FMT_MXFP4, _gnf4b.OP_FWD, a_host, blocks, scales, sizes, expert_ids,
                        blocks.shape[1], out, path=path, return_status=return_status)


def dgrad_mxfp4_grouped_host(grad_host, blocks, scales, sizes, expert_ids, out=None, *, return_status: bool = False):
    """``dgrad_mxfp4_grouped`` with host buffers (``gnf4_native/cpu_kernels.c:1386-1397``)."""
    return _launch_host(_gnf4b.FMT_MXFP4, _gnf4b.OP_DGRAD, grad_host, blocks, scales, sizes, expert_ids,
                        blocks.shape[2] * 2, out, return_status=return_status)


def dgrad_mxfp4_grouped(grad_out, blocks, scales, sizes, expert_ids, *, group_offsets=None, max_rows=None,
                        zero_rest: bool = False):
    """``grad_a[t,:] = grad_out[t,:] @ dequant_mxfp4(blocks[e(t)])`` in one launch, ``[T,K]``
    bf16.  The reference has this only as a per-expert Python loop on the GPU
    (kernel/mxfp4_qlora.py:105-122) and as a CPU kernel (gnf4_native/cpu_kernels.c:1386-1397).  Rows of no group or
    of a padding group (expert id -1) are not written, or zeros with ``zero_rest``."""
    E, N, half = blocks.shape
    _require_cuda(grad_out, "dgrad_mxfp4_grouped",
                  "The CPU-checkable equivalent is grad_out @ dequant_mxfp4(blocks, scales) per group.")
    if grad_out.dtype != torch.bfloat16:
        raise ValueError(f"dgrad_mxfp4_grouped cannot run this problem: grad_out dtype {grad_out.dtype} is not bfloat16")
    if grad_out.shape[1] != N:
        raise ValueError(f"grad_out has {grad_out.shape[1]} columns but the stack has N={N}")
    return _launch(_gnf4b.FMT_MXFP4, _gnf4b.OP_DGRAD, grad_out, blocks, scales, sizes, expert_ids, half * 2,
                   group_offsets=group_offsets, max_rows=max_rows, zero_rest=zero_rest)


def dequant_stack_cuda(blocks, scales):
    """Element decode of a whole MXFP4 stack by the CUDA library's decode routines ->
    ``[E,N,K]`` fp32, for bit-for-bit comparison with ``mxfp4_pack_ref.dequant_mxfp4``."""
    _require_cuda(blocks, "dequant_stack_cuda", "Use mxfp4_pack_ref.dequant_mxfp4 on CPU tensors.")
    E, N, half = blocks.shape
    if blocks.stride(2) != 1:
        blocks = blocks.contiguous()
    if scales.stride(2) != 1:
        scales = scales.contiguous()
    out = torch.empty(E, N, half * 2, dtype=torch.float32, device=blocks.device)
    lib = _gnf4b.load()
    with torch.cuda.device(blocks.device):
        rc = lib.gnf4b_dequant(_gnf4b.FMT_MXFP4, blocks.data_ptr(), blocks.stride(0), blocks.stride(1),
                               scales.data_ptr(), _gnf4b.S_E8M0, scales.stride(0), scales.stride(1),
                               E, N, half * 2, out.data_ptr(),
                               torch.cuda.current_stream(blocks.device).cuda_stream)
    _gnf4b.check(rc, "gnf4b_dequant")
    return out


# --------------------------------------------------------------------------- #
# both operands in MXFP4: quantiser, product, expert FFN
# --------------------------------------------------------------------------- #
_X_DTYPES = {torch.bfloat16: _gnf4b.X_BF16, torch.float16: _gnf4b.X_FP16, torch.float32: _gnf4b.X_FP32}


def quantize_mxfp4(x):
    """Rows to MXFP4 on the GPU: ``x [..., K]`` bf16 / fp16 / fp32 (K a multiple of 32) -> ``(blocks [..., K//2],
    scales [..., K//32])`` uint8, element 2j in the low nibble.  Per 32 elements the exponent is the least integer
    e >= -69 with max|x| <= 6 * 2^e and every element takes the nearest e2m1 value, the lower magnitude on a tie: byte
    for byte what ``mxfp4_pack_ref.quantize_pack_mxfp4`` gives (as ``[..., K//32, 16]``).  A block that holds an
    infinity or a NaN gets the exponent byte 255.  Rows may be a strided view; other layouts are copied first."""
    if not x.is_cuda:
        _require_cuda(x, "quantize_mxfp4", "The CPU counterpart is mxfp4_pack_ref.quantize_pack_mxfp4.")
    dtype = _X_DTYPES.get(x.dtype)
    if dtype is None:
        raise TypeError(f"quantize_mxfp4 takes bfloat16, float16 or float32, got {x.dtype}")
    shape = x.shape
    K = shape[-1] if shape else 0
    if K == 0 or K % MX_BLOCK:
        raise ValueError(f"the last dimension must be a positive multiple of {MX_BLOCK}, got shape {tuple(shape)}")
    dev = x.device
    if len(shape) == 2:
        rows = shape[0]
        blocks = torch.empty(rows, K // 2, dtype=torch.uint8, device=dev)
        scales = torch.empty(rows, K // MX_BLOCK, dtype=torch.uint8, device=dev)
    else:
        rows = x.numel() // K
        x = x.reshape(rows, K)
        blocks = torch.empty(*shape[:-1], K // 2, dtype=torch.uint8, device=dev)
        scales = torch.empty(*shape[:-1], K // MX_BLOCK, dtype=torch.uint8, device=dev)
    pitch, unit = x.stride()
    if unit != 1:
        x, pitch = x.contiguous(), K
    rc = _call_on(dev, _gnf4b.load().gnf4b_quantize_mxfp4, x.data_ptr(), dtype, rows, K, pitch if rows > 1 else K,
                  blocks.data_ptr(), scales.data_ptr())
    if rc:
        _gnf4b.check(rc, "gnf4b_quantize_mxfp4")
    return blocks, scales


def _check_packed(blocks, scales, what: str):
    bs, ss = blocks.shape, scales.shape
    n = len(bs)
    if blocks.dtype is torch.uint8 and scales.dtype is torch.uint8 and n == len(ss) and n and bs[-1] == 16 * ss[-1] > 0 \
            and (bs[0] == ss[0] if n == 2 else bs[:-1] == ss[:-1]) and scales.device == blocks.device:
        return
    if blocks.dtype != torch.uint8 or scales.dtype != torch.uint8:
        raise TypeError(f"{what}: blocks and scales must be uint8, got {blocks.dtype} and {scales.dtype}")
    if scales.device != blocks.device:
        raise ValueError(f"{what}: blocks and scales must live on the same device")
    raise ValueError(f"{what}: blocks {tuple(bs)} and scales {tuple(ss)} are not [..., K//2] and [..., K//32]")


def _packed_rows(t, align: int):
    """``t`` contiguous and its data aligned."""
    t = t.contiguous()
    return t.clone() if t.data_ptr() % align else t


def dequantize_mxfp4(blocks, scales, dtype=torch.bfloat16):
    """The values of packed rows, ``blocks [..., K//2]`` and ``scales [..., K//32]`` -> ``[..., K]`` in bf16 or fp32
    (exact) or fp16 (rounded once).  An exponent byte of 255 reads as 2^128, as in ``mxfp4_pack_ref.dequant_mxfp4``."""
    if not blocks.is_cuda:
        _require_cuda(blocks, "dequantize_mxfp4", "The CPU counterpart is mxfp4_pack_ref.dequant_mxfp4.")
    if dtype not in _X_DTYPES:
        raise TypeError(f"dequantize_mxfp4 returns bfloat16, float16 or float32, not {dtype}")
    _check_packed(blocks, scales, "dequantize_mxfp4")
    blocks, scales = _packed_rows(blocks, 4), scales.contiguous()
    out = torch.empty(*blocks.shape[:-1], 2 * blocks.shape[-1], dtype=dtype, device=blocks.device)
    rc = _call_on(blocks.device, _gnf4b.load().gnf4b_dequantize_mxfp4, blocks.data_ptr(), scales.data_ptr(), scales.numel(),
                  _X_DTYPES[dtype], out.data_ptr())
    if rc:
        _gnf4b.check(rc, "gnf4b_dequantize_mxfp4")
    return out


def glu_quantize_mxfp4(gate_up, act: str = "silu", bias=None, row_expert=None):
    """The activation between an expert's two products with its result packed in the same pass: ``gate_up [rows, 2h]``
    bf16 (h a multiple of 32) -> ``(blocks [rows, h//2], scales [rows, h//32])``, the bytes of ``ep_moe.silu_glu``
    (``act="silu"``) or ``glu_gpt_oss`` (``act="gpt_oss"``; optional ``bias`` bf16 ``[E, 2h]`` by ``row_expert``) followed
    by ``quantize_mxfp4``."""
    if act not in ("gpt_oss", "silu"):
        raise ValueError("act is 'gpt_oss' or 'silu'")
    _require_cuda(gate_up, "glu_quantize_mxfp4", "")
    if gate_up.dtype != torch.bfloat16:
        raise TypeError(f"gate_up must be bfloat16, got {gate_up.dtype}")
    if gate_up.dim() != 2 or gate_up.shape[1] == 0 or gate_up.shape[1] % (2 * MX_BLOCK):
        raise ValueError(f"gate_up must be [rows, 2h] with h a multiple of {MX_BLOCK}, got {tuple(gate_up.shape)}")
    rows, h = gate_up.shape[0], gate_up.shape[1] // 2
    dev = gate_up.device
    gate_up = gate_up.detach().contiguous()
    E = 0
    if bias is not None:
        if act != "gpt_oss" or row_expert is None:
            raise ValueError("bias goes with act='gpt_oss' and row_expert")
        if bias.dtype != torch.bfloat16 or bias.dim() != 2 or bias.shape[1] != 2 * h or bias.shape[0] == 0 or bias.device != dev:
            raise ValueError(f"bias must be a bfloat16 tensor [E, {2 * h}] on {dev}")
        if tuple(row_expert.shape) != (rows,) or row_expert.device != dev or row_expert.dtype not in (torch.int32, torch.int64):
            raise ValueError(f"row_expert must be an integer tensor of {rows} expert ids on {dev}")
        E = bias.shape[0]
        bias, row_expert = bias.detach().contiguous(), row_expert.to(torch.int32).contiguous()
    blocks = torch.empty(rows, h // 2, dtype=torch.uint8, device=dev)
    scales = torch.empty(rows, h // MX_BLOCK, dtype=torch.uint8, device=dev)
    rc = _call_on(dev, _gnf4b.load().gnf4b_glu_quantize_mxfp4, gate_up.data_ptr(), rows, h,
                  _gnf4b.ACT_SILU_GLU if act == "silu" else _gnf4b.ACT_GPT_OSS_GLU,
                  bias.data_ptr() if bias is not None else None, row_expert.data_ptr() if bias is not None else None, E,
                  blocks.data_ptr(), scales.data_ptr(), _status_ptr(dev))
    if rc:
        _gnf4b.check(rc, "gnf4b_glu_quantize_mxfp4")
    return blocks, scales


def _refuse_w4a4(a_blocks, a_scales, blocks, scales):
    if a_blocks.dim() != 2 or blocks.dim() != 3:
        raise ValueError(f"a_blocks must be [T, K//2] and blocks [E, N, K//2], got {tuple(a_blocks.shape)} and {tuple(blocks.shape)}")
    _check_packed(a_blocks, a_scales, "gemm_mxfp4_grouped_w4a4 (rows)")
    _check_packed(blocks, scales, "gemm_mxfp4_grouped_w4a4 (stack)")
    if blocks.device != a_blocks.device:
        raise ValueError("rows and stack must live on the same device")
    raise ValueError(f"the rows have K={2 * a_blocks.shape[1]} but the stack packs K={2 * blocks.shape[2]}")


def gemm_mxfp4_grouped_w4a4(a_blocks, a_scales, blocks, scales, sizes, expert_ids, *, group_offsets=None, max_rows=None):
    """Grouped product of MXFP4 rows with MXFP4 expert stacks: ``out[t] = dequant(a)[t] @ dequant(W[e(t)]).T``, both
    operands multiplied as they are packed, on the block-scaled tensor cores (fp32 accumulation, one rounding to bf16).

    ``a_blocks [T, K//2]`` / ``a_scales [T, K//32]`` uint8 rows sorted by group (``quantize_mxfp4`` makes them);
    ``blocks [E, N, K//2]`` / ``scales [E, N, K//32]`` and ``sizes``, ``expert_ids``, ``group_offsets``, ``max_rows`` as in
    ``gemm_mxfp4_grouped`` (``max_rows`` only shapes the tiles).  An exponent byte of 255 is NaN here, as in the OCP
    format.  Returns ``[T, N]`` bf16, rows that belong to no group not written.  A stack whose strides are not positive
    multiples of 16 bytes is copied first.

    A few one-row groups (one decoded token) are better served by ``gemm_mxfp4_grouped`` on the rows as they are: four
    experts with N = 5760, K = 2880 take 11.9 to 12.7 us there and 13.1 here, with the quantiser's 1.5 still to pay.  With
    32 one-row groups this product is ahead, 55 against 68 us, and with more rows per group by a factor of four."""
    if not a_blocks.is_cuda:
        _require_cuda(a_blocks, "gemm_mxfp4_grouped_w4a4",
                      "The CPU-checkable equivalent multiplies mxfp4_pack_ref.dequant_mxfp4 of both operands per group.")
    u8, index = torch.uint8, a_blocks.get_device()
    xb, xs, wb, ws = a_blocks.shape, a_scales.shape, blocks.shape, scales.shape
    if not (a_blocks.dtype is u8 and a_scales.dtype is u8 and blocks.dtype is u8 and scales.dtype is u8
            and len(xb) == len(xs) == 2 and len(wb) == len(ws) == 3 and xb[0] == xs[0] and wb[0] == ws[0] and wb[1] == ws[1]
            and wb[2] == xb[1] == 16 * xs[1] > 0 and ws[2] == xs[1]
            and a_scales.get_device() == blocks.get_device() == scales.get_device() == index):
        _refuse_w4a4(a_blocks, a_scales, blocks, scales)
    for table in (group_offsets, expert_ids, sizes):
        if isinstance(table, torch.Tensor) and table.is_cuda and table.get_device() != index:
            raise ValueError(f"a group table lives on {table.device}, the rows on {a_blocks.device}")
    T, half = xb
    E, N, _ = wb
    dev = a_blocks.device
    out = torch.empty(T, N, dtype=torch.bfloat16, device=dev)
    if T == 0 or N == 0:
        return out
    if E == 0:
        raise ValueError(f"the stack holds no experts, but there are {T} rows")
    x_p, w_p = a_blocks.data_ptr(), blocks.data_ptr()
    if x_p % 16 or not a_blocks.is_contiguous():
        a_blocks = _packed_rows(a_blocks, 16)
        x_p = a_blocks.data_ptr()
    a_scales = a_scales.contiguous()
    # the stack as TMA takes it: 16-byte aligned, positive strides in multiples of 16 bytes
    w_e, w_n, unit = blocks.stride()
    if unit != 1 or w_p % 16 or (E > 1 and (w_e <= 0 or w_e % 16)) or (N > 1 and (w_n <= 0 or w_n % 16)):
        blocks = _packed_rows(blocks, 16)
        w_p = blocks.data_ptr()
        w_e, w_n, _ = blocks.stride()
    s_e, s_n, unit = scales.stride()
    if unit != 1:
        scales = scales.contiguous()
        s_e, s_n, _ = scales.stride()
    prev = torch.cuda.current_device()
    if index != prev:
        torch.cuda.set_device(dev)                      # the C library launches on the current device
    try:
        stream_ptr = _raw_stream(dev)
        off_t, ids_t, G, max_rows = _group_tables(sizes, expert_ids, T, E, dev, group_offsets, max_rows, stream_ptr)
        if G == 0:
            return out
        rc = _gnf4b.load().gnf4b_gemm_grouped_w4a4(
            x_p, a_scales.data_ptr(), T, w_p, w_e, w_n, scales.data_ptr(), s_e, s_n,
            off_t if isinstance(off_t, int) else off_t.data_ptr(), ids_t if isinstance(ids_t, int) else ids_t.data_ptr(), G, E, N,
            2 * half, max_rows, out.data_ptr(), _status_ptr(dev), stream_ptr)
    finally:
        if index != prev:
            torch.cuda.set_device(prev)
    if rc:
        _gnf4b.check(rc, "gnf4b_gemm_grouped_w4a4")
    return out


def ffn_mxfp4_grouped_w4a4(a_cat, blocks_gu, scales_gu, blocks_dn, scales_dn, sizes, expert_ids, *, act: str = "gpt_oss",
                           bias_gu=None, row_expert=None, group_offsets=None, max_rows=None):
    """One MXFP4 expert FFN per row with the rows in MXFP4 too: quantise ``a_cat [T, K]``, gate_up product, activation
    packed as it is computed, down product -> ``[T, N_dn]`` bf16.  Stacks, groups and ``act`` as in ``ffn_mxfp4_grouped``;
    ``a_cat`` may also be the packed pair ``(blocks, scales)`` (quantise a token once, gather its bytes to its experts).
    ``bias_gu`` (bf16 ``[E, N_gu]``) goes with ``act="gpt_oss"`` only and is added per row, by ``row_expert [T]``, where
    ``ffn_mxfp4_grouped`` takes it by group.

    Four launches, the rows rounded to MXFP4 twice.  One decoded token is better served by ``ffn_mxfp4_grouped``, one launch:
    four gpt-oss experts 24 us against 29 in a graph, 24 against 46 in single calls.  With 32 one-row groups 92 us against
    115, with 64 rows per group 118 against 418."""
    if act not in ("gpt_oss", "silu"):
        raise ValueError("act is 'gpt_oss' or 'silu'")
    a_b, a_s = a_cat if isinstance(a_cat, (tuple, list)) else quantize_mxfp4(a_cat)
    if blocks_gu.shape[1] % 2 or blocks_dn.shape[0] != blocks_gu.shape[0] or blocks_dn.shape[2] * 4 != blocks_gu.shape[1]:
        raise ValueError(f"down stack {tuple(blocks_dn.shape)} does not follow gate_up {tuple(blocks_gu.shape)}")
    gu = gemm_mxfp4_grouped_w4a4(a_b, a_s, blocks_gu, scales_gu, sizes, expert_ids, group_offsets=group_offsets, max_rows=max_rows)
    h_b, h_s = glu_quantize_mxfp4(gu, act, bias_gu, row_expert)
    return gemm_mxfp4_grouped_w4a4(h_b, h_s, blocks_dn, scales_dn, sizes, expert_ids, group_offsets=group_offsets, max_rows=max_rows)
