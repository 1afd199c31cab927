"""Differentiable grouped 4-bit GEMMs for QLoRA-style training on top of the CUDA op.

Mirror of the reference's autograd layer (``kernel/nf4_qlora.py:32-305`` for NF4 and the
``_FusedGroupedMxfp4`` function of ``kernel/mxfp4_qlora.py:98-122`` for MXFP4): the packed base weight is
frozen, so the only gradient is the input gradient ``grad_out @ W`` -- one launch of the dgrad kernel -- and
nothing decoded survives from forward to backward.  The trainable part is the per-expert low-rank delta,
added to the projection BEFORE any activation (``act(Wx + BAx) != act(Wx) + d``).

Same names, argument meaning and defaults as the reference:

    gemm_4bit_grouped_train(a_cat, packed, absmax, sizes, expert_ids, weights_fn=None, dgrad_kernel=True)
    lora_delta_grouped(a_cat, lora_A, lora_B, sizes, expert_ids, scaling=1.0)
    fused_grouped_lora(a_cat, packed, absmax, sizes, expert_ids, lora_A=None, lora_B=None, weights_fn=None,
                       scaling=1.0, dgrad_kernel=True)

plus ``gemm_mxfp4_grouped_train`` (the reference's MXFP4 backward is a Python loop over experts; here it is
the same dgrad kernel with the MXFP4 decode), ``gemm_mxfp4_grouped_w4a4_train`` (rows in MXFP4 forward, straight-through
gradient) and the whole expert FFN for training: ``glu_train``, the activation between the two products that keeps its
input in 8 bits for the backward pass, and ``ffn_4bit_grouped_train`` / ``ffn_mxfp4_grouped_train`` around it.
"""
from __future__ import annotations

import torch

#: the batched low-rank delta pads every group to the widest one; beyond this ratio of padded to real rows
#: (a very hot expert) the per-expert loop is used instead (reference: ``_PAD_WASTE_LIMIT``)
_PAD_WASTE_LIMIT = 4.0


def _host_ints(v):
    return [int(x) for x in (v.tolist() if torch.is_tensor(v) else v)]


class _FirstOnly(torch.autograd.Function):
    """Identity behind a kernel's gradient: a second derivative through it is refused when it is asked for, instead of coming
    back without this term."""

    @staticmethod
    def forward(ctx, grad, what):
        ctx.what = what
        return grad.view_as(grad)

    @staticmethod
    def backward(ctx, _grad):
        raise RuntimeError(f"the gradient of {ctx.what} is a kernel's result: it cannot be differentiated a second time")


def first_derivative_only(grad, what: str):
    """``grad`` as a backward pass under ``create_graph=True`` returns it, see ``_FirstOnly``."""
    return _FirstOnly.apply(grad.detach().requires_grad_(), what)


def _product_gradient(dgrad, what, grad_out, packed, scales, sizes, expert_ids):
    """``dgrad(grad_out, ...)``.  The product is linear in its rows: its gradient depends on ``grad_out`` alone.  Rows that no
    expert takes have the gradient zero; with group tables in host memory and no padding group there are none."""
    on_host = not any(torch.is_tensor(t) and t.is_cuda for t in (sizes, expert_ids))
    grad = dgrad(grad_out, packed, scales, sizes, expert_ids, zero_rest=not on_host or min(_host_ints(expert_ids), default=0) < 0)
    return first_derivative_only(grad, what) if torch.is_grad_enabled() and grad_out.requires_grad else grad


class FusedGroupedNf4(torch.autograd.Function):
    """``out = gemm_4bit_grouped(a_cat, packed, absmax, sizes, expert_ids)`` with
    ``grad_a = dgrad_4bit_grouped(grad_out, ...)``.

    ``weights_fn`` (optional, zero arguments, returns ``(packed, absmax)``) is called at backward time
    instead of keeping the two tensors on the context: an offloading caller re-stages a layer by replacing
    storage, and a tensor held here would keep the evicted storage alive (ref ``:54-72``).
    ``dgrad_kernel=False`` takes the exact per-expert loop (decode one expert, one matmul per group) -- the
    form to use when a gradient has to be compared bit for bit with a dequantise-then-matmul trainer; the
    loop is also the fallback when the kernel cannot take the problem (``dgrad_eligible``) or the stack
    lives on another device.
    """

    @staticmethod
    def forward(ctx, a_cat, packed, absmax, sizes, expert_ids, weights_fn=None, dgrad_kernel=True):
        from nf4_grouped import gemm_4bit_grouped
        ctx.use_kernel = bool(dgrad_kernel)
        ctx.weights_fn = weights_fn
        ctx.stack = None if weights_fn is not None else (packed, absmax)
        ctx.sizes, ctx.expert_ids = sizes, expert_ids       # kept as given: no host read of device ids here
        return gemm_4bit_grouped(a_cat, packed, absmax, sizes, expert_ids)

    @staticmethod
    def backward(ctx, grad_out):
        if not ctx.needs_input_grad[0]:
            return (None,) * 7
        from nf4_grouped import dequant_ref, dgrad_4bit_grouped, dgrad_eligible
        packed, absmax = ctx.stack if ctx.weights_fn is None else ctx.weights_fn()
        grad_out = grad_out.contiguous()
        if ctx.use_kernel and packed.device == grad_out.device and dgrad_eligible(grad_out, packed, absmax) is None:
            return (_product_gradient(dgrad_4bit_grouped, "gemm_4bit_grouped_train", grad_out, packed, absmax, ctx.sizes, ctx.expert_ids),
                    *(None,) * 6)
        n_out, k_in = packed.shape[1], packed.shape[2] * 2
        grad_a = torch.zeros(grad_out.shape[0], k_in, dtype=grad_out.dtype, device=grad_out.device)
        first = 0
        for rows, e in zip(_host_ints(ctx.sizes), _host_ints(ctx.expert_ids)):
            if rows and e >= 0:                              # a padding group has no gradient
                w = dequant_ref(packed[e].to(grad_out.device), absmax[e].to(grad_out.device), n_out, k_in)
                grad_a[first:first + rows] = grad_out[first:first + rows] @ w.to(grad_out.dtype)
            first += rows
        return (grad_a,) + (None,) * 6


def gemm_4bit_grouped_train(a_cat, packed, absmax, sizes, expert_ids, weights_fn=None, dgrad_kernel=True):
    """``gemm_4bit_grouped`` that ``a_cat`` may require a gradient through (ref ``:161-171``)."""
    return FusedGroupedNf4.apply(a_cat, packed, absmax, sizes, expert_ids, weights_fn, dgrad_kernel)


def _dgrad_mxfp4(grad_out, blocks, scales, sizes, expert_ids, zero_rest):
    """``dgrad_mxfp4_grouped`` for any N: its kernel takes multiples of 8 (16-byte rows of ``grad_out``), other widths are
    filled up with columns of zeros against rows of zeros."""
    from mxfp4_grouped import dgrad_mxfp4_grouped
    fill = -blocks.shape[1] % 8
    if fill:
        grad_out = torch.nn.functional.pad(grad_out, (0, fill))
        blocks, scales = (torch.nn.functional.pad(t, (0, 0, 0, fill)) for t in (blocks, scales))
    return dgrad_mxfp4_grouped(grad_out.contiguous(), blocks, scales, sizes, expert_ids, zero_rest=zero_rest)


class FusedGroupedMxfp4(torch.autograd.Function):
    """The MXFP4 counterpart: forward ``gemm_mxfp4_grouped``, backward ``dgrad_mxfp4_grouped``."""

    @staticmethod
    def forward(ctx, a_cat, blocks, scales, sizes, expert_ids):
        from mxfp4_grouped import gemm_mxfp4_grouped
        ctx.stack = (blocks, scales)
        ctx.sizes, ctx.expert_ids = sizes, expert_ids
        return gemm_mxfp4_grouped(a_cat, blocks, scales, sizes, expert_ids)

    @staticmethod
    def backward(ctx, grad_out):
        if not ctx.needs_input_grad[0]:
            return (None,) * 5
        return (_product_gradient(_dgrad_mxfp4, "gemm_mxfp4_grouped_train", grad_out, *ctx.stack, ctx.sizes, ctx.expert_ids),
                *(None,) * 4)


def gemm_mxfp4_grouped_train(a_cat, blocks, scales, sizes, expert_ids):
    return FusedGroupedMxfp4.apply(a_cat, blocks, scales, sizes, expert_ids)


def _lora_delta_grouped_loop(a_cat, lora_A, lora_B, sizes, expert_ids, scaling=1.0):
    """One pair of matmuls per non-empty group: the fallback for skewed routing and the form the batched
    path is tested against.  ``None`` when there are no rows."""
    out, first = None, 0
    for rows, e in zip(_host_ints(sizes), _host_ints(expert_ids)):
        if rows and e >= 0:                                  # a padding group has no delta
            x = a_cat[first:first + rows].to(lora_A.dtype)
            d = scaling * ((x @ lora_A[e].t()) @ lora_B[e].t())
            if out is None:
                out = torch.zeros(a_cat.shape[0], lora_B.shape[1], dtype=d.dtype, device=a_cat.device)
            out[first:first + rows] = d
        first += rows
    return out


def lora_delta_grouped(a_cat, lora_A, lora_B, sizes, expert_ids, scaling=1.0):
    """``scaling * B_e (A_e x)`` for every row x of every group (``lora_A [E, r, K]``, ``lora_B [E, N, r]``)
    -> ``[T, N]``; ``None`` when all groups are empty (ref ``:174-248``).  ``scaling`` is LoRA's alpha / r.

    Batched: the non-empty groups are padded to the widest one and run as two ``bmm``s, so the autograd
    graph has two nodes per projection instead of two per expert; when padding would multiply the rows by
    more than ``_PAD_WASTE_LIMIT`` the per-expert loop is used."""
    size_list = _host_ints(sizes)
    on_device = torch.is_tensor(expert_ids) and expert_ids.device.type != "cpu"
    ids = None if on_device else _host_ints(expert_ids)
    live = [g for g, n in enumerate(size_list) if n > 0]
    if not live:
        return None
    rows = [size_list[g] for g in live]
    total, widest = sum(rows), max(rows)
    if len(live) * widest > _PAD_WASTE_LIMIT * total:
        return _lora_delta_grouped_loop(a_cat, lora_A, lora_B, sizes, expert_ids, scaling)
    dev = a_cat.device
    if on_device:
        experts = expert_ids.to(torch.int64)[torch.tensor(live, dtype=torch.int64, device=expert_ids.device)]
    else:
        experts = torch.tensor([ids[g] for g in live], dtype=torch.int64, device=dev)
    # row t of the live rows belongs to live group grp[t], at position pos[t] inside it
    counts = torch.tensor(rows, dtype=torch.int64, device=dev)
    starts = torch.cumsum(counts, 0) - counts
    grp = torch.repeat_interleave(torch.arange(len(live), device=dev), counts, output_size=total)
    pos = torch.arange(total, device=dev) - starts[grp]
    # live rows in a_cat: the groups are contiguous, empty groups take no rows, so they are rows [0, total)
    a_rows, none = a_cat[:total].to(lora_A.dtype), None
    if on_device or min(ids) < 0:
        # rows of a padding group (expert -1) have no delta: what they hold, and what comes back through them, stays out of
        # the factors' gradients whatever it is
        none = (experts < 0)[grp][:, None]
        experts = experts.clamp_min(0)
        a_rows = a_rows.masked_fill(none, 0)
    x = torch.zeros(len(live), widest, a_cat.shape[1], dtype=lora_A.dtype, device=dev)
    x[grp, pos] = a_rows
    low = torch.bmm(x, lora_A[experts].transpose(1, 2))                        # [G, widest, r]
    d = scaling * torch.bmm(low, lora_B[experts].transpose(1, 2))              # [G, widest, N]
    out = torch.zeros(a_cat.shape[0], lora_B.shape[1], dtype=d.dtype, device=dev)
    out[:total] = d[grp, pos] if none is None else d[grp, pos].masked_fill(none, 0)
    return out


def fused_grouped_lora(a_cat, packed, absmax, sizes, expert_ids, lora_A=None, lora_B=None, weights_fn=None,
                       scaling=1.0, dgrad_kernel=True):
    """Frozen 4-bit projection (differentiable in ``a_cat``) plus the trainable low-rank delta
    (differentiable in ``lora_A`` / ``lora_B``), summed before any activation (ref ``:286-305``)."""
    out = gemm_4bit_grouped_train(a_cat, packed, absmax, sizes, expert_ids, weights_fn=weights_fn,
                                  dgrad_kernel=dgrad_kernel)
    if lora_A is None or lora_B is None:
        return out
    delta = lora_delta_grouped(a_cat, lora_A, lora_B, sizes, expert_ids, scaling)
    return out if delta is None else out + delta.to(out.dtype)


# --------------------------------------------------------------------------- #
# both operands in MXFP4
# --------------------------------------------------------------------------- #
class FusedGroupedMxfp4W4A4(torch.autograd.Function):
    """Forward ``gemm_mxfp4_grouped_w4a4`` on the quantised rows; backward ``dgrad_mxfp4_grouped``, the quantiser taken
    as the identity (straight-through)."""

    @staticmethod
    def forward(ctx, a_cat, blocks, scales, sizes, expert_ids):
        from mxfp4_grouped import gemm_mxfp4_grouped_w4a4, quantize_mxfp4
        ctx.stack = (blocks, scales)
        ctx.sizes, ctx.expert_ids = sizes, expert_ids
        ctx.a_dtype = a_cat.dtype
        return gemm_mxfp4_grouped_w4a4(*quantize_mxfp4(a_cat), blocks, scales, sizes, expert_ids)

    @staticmethod
    def backward(ctx, grad_out):
        if not ctx.needs_input_grad[0]:
            return (None,) * 5
        grad = _product_gradient(_dgrad_mxfp4, "gemm_mxfp4_grouped_w4a4_train", grad_out, *ctx.stack, ctx.sizes, ctx.expert_ids)
        return (grad.to(ctx.a_dtype),) + (None,) * 4


def gemm_mxfp4_grouped_w4a4_train(a_cat, blocks, scales, sizes, expert_ids):
    """``quantize_mxfp4`` then ``gemm_mxfp4_grouped_w4a4``, with the gradient of the unquantised product."""
    return FusedGroupedMxfp4W4A4.apply(a_cat, blocks, scales, sizes, expert_ids)


# --------------------------------------------------------------------------- #
# the activation between an expert's products, its input kept in 8 bits
# --------------------------------------------------------------------------- #
CKPT_BLOCK = 64        # gate (or up) values that share one fp32 step
_GLU_ACTS = {"silu": 0, "gpt_oss": 1}        # GNF4B_ACT_*


class _GluTrain(torch.autograd.Function):
    @staticmethod
    def forward(ctx, gate_up, act, bias, row_expert):
        import _gnf4b
        from nf4_grouped import _call_on, _status_ptr
        dev = gate_up.device
        rows, h = gate_up.shape[0], gate_up.shape[1] // 2
        out = torch.empty(rows, h, dtype=torch.bfloat16, device=dev)
        codes = steps = None
        if ctx.needs_input_grad[0]:
            nb = -(-h // CKPT_BLOCK)
            codes = torch.empty(rows, nb, 2, CKPT_BLOCK, dtype=torch.int8, device=dev)
            steps = torch.empty(rows, nb, 2, dtype=torch.float32, device=dev)
        ptr = lambda t: t.data_ptr() if t is not None else None  # noqa: E731
        rc = _call_on(dev, _gnf4b.load().gnf4b_glu_ckpt8_fwd, gate_up.data_ptr(), rows, h, act, ptr(bias), ptr(row_expert),
                      bias.shape[0] if bias is not None else 0, out.data_ptr(), ptr(codes), ptr(steps), _status_ptr(dev))
        if rc:
            _gnf4b.check(rc, "gnf4b_glu_ckpt8_fwd")
        if codes is not None:
            ctx.save_for_backward(codes, steps)
        ctx.act, ctx.h = act, h
        return out

    @staticmethod
    def backward(ctx, grad_out):
        grad = _glu_backward(ctx, grad_out)
        # create_graph=True: the gradient depends on gate_up, whatever comes in
        return (first_derivative_only(grad, "glu_train") if torch.is_grad_enabled() else grad), None, None, None


def _glu_backward(ctx, grad_out):
    import _gnf4b
    from nf4_grouped import _call_on
    codes, steps = ctx.saved_tensors
    grad_out = grad_out.contiguous()
    rows = codes.shape[0]
    grad = torch.empty(rows, 2 * ctx.h, dtype=torch.bfloat16, device=codes.device)
    rc = _call_on(codes.device, _gnf4b.load().gnf4b_glu_ckpt8_bwd, grad_out.data_ptr(), codes.data_ptr(), steps.data_ptr(), rows,
                  ctx.h, ctx.act, grad.data_ptr())
    if rc:
        _gnf4b.check(rc, "gnf4b_glu_ckpt8_bwd")
    return grad


def glu_train(gate_up, act: str = "silu", *, bias=None, row_expert=None):
    """The activation between an expert's two products, differentiable: ``gate_up [rows, 2h]`` bf16 -> ``[rows, h]`` bf16.
    ``act="silu"``: SiLU(gate) * up over column halves; ``act="gpt_oss"``: gate and up interleaved, clamped at 7,
    (up + 1) * gate * sigmoid(1.702 gate), with an optional frozen ``bias`` bf16 ``[E, 2h]`` added by ``row_expert [rows]``.
    fp32 inside, one rounding: not the bits of ``mxfp4_grouped.glu_gpt_oss`` and what is built on it (``ffn_mxfp4_grouped``,
    ``glu_quantize_mxfp4``), which round the bias sum and four intermediate results to bf16 as a chain of tensor operations
    does.

    What stays until the backward pass is gate and up in 8 bits (per 64 values of a row one fp32 step, their largest
    magnitude / 127): 2.1 bytes per pair where autograd through tensor operations keeps 10 and more, and neither
    ``gate_up`` nor the result need stay alive.  The gradient is the formula's, taken at the kept values.  Without a
    gradient to compute nothing is kept."""
    from nf4_grouped import _require_cuda
    if act not in _GLU_ACTS:
        raise ValueError("act is 'gpt_oss' or 'silu'")
    _require_cuda(gate_up, "glu_train", "")
    if gate_up.dtype != torch.bfloat16:
        raise TypeError(f"gate_up must be bfloat16, got {gate_up.dtype}")
    if gate_up.dim() != 2 or gate_up.shape[1] == 0 or gate_up.shape[1] % 2:
        raise ValueError(f"gate_up must be [rows, 2h], got {tuple(gate_up.shape)}")
    if bias is not None:
        rows, dev = gate_up.shape[0], gate_up.device
        if act != "gpt_oss" or row_expert is None:
            raise ValueError("bias goes with act='gpt_oss' and row_expert")
        if bias.requires_grad and torch.is_grad_enabled():
            raise ValueError("the bias of glu_train is frozen: add a trainable one to gate_up before the call")
        if bias.dtype != torch.bfloat16 or bias.dim() != 2 or bias.shape[1] != gate_up.shape[1] or bias.shape[0] == 0 or bias.device != dev:
            raise ValueError(f"bias must be a bfloat16 tensor [E, {gate_up.shape[1]}] on {dev}")
        if tuple(row_expert.shape) != (rows,) or row_expert.device != dev or row_expert.dtype not in (torch.int32, torch.int64):
            raise ValueError(f"row_expert must be an integer tensor of {rows} expert ids on {dev}")
        bias, row_expert = bias.detach().contiguous(), row_expert.to(torch.int32).contiguous()
    if not torch.is_grad_enabled():
        gate_up = gate_up.detach()        # autograd asks a function for its inputs' gradients under no_grad all the same
    return _GluTrain.apply(gate_up.contiguous(), _GLU_ACTS[act], bias, row_expert)


def ffn_4bit_grouped_train(a_cat, packed_gu, absmax_gu, packed_dn, absmax_dn, sizes, expert_ids, *, act: str = "silu",
                           lora_gu=None, lora_dn=None, scaling=1.0, dgrad_kernel=True):
    """One NF4 expert FFN per row for training: gate_up and down through ``fused_grouped_lora`` (frozen stacks,
    ``lora_gu`` / ``lora_dn`` optional ``(lora_A, lora_B)`` pairs) with ``glu_train`` between them.  ``[T, K]`` bf16 ->
    ``[T, N_dn]`` bf16; besides the low-rank branch, a layer keeps its gate_up activations in 8 bits and nothing else."""
    gu = fused_grouped_lora(a_cat, packed_gu, absmax_gu, sizes, expert_ids, *(lora_gu or (None, None)), scaling=scaling,
                            dgrad_kernel=dgrad_kernel)
    return fused_grouped_lora(glu_train(gu, act), packed_dn, absmax_dn, sizes, expert_ids, *(lora_dn or (None, None)),
                              scaling=scaling, dgrad_kernel=dgrad_kernel)


def ffn_mxfp4_grouped_train(a_cat, blocks_gu, scales_gu, blocks_dn, scales_dn, sizes, expert_ids, *, act: str = "gpt_oss",
                            bias_gu=None, row_expert=None, rows: str = "bf16"):
    """The MXFP4 counterpart on frozen stacks; ``bias_gu`` (bf16 ``[E, N_gu]``, ``act="gpt_oss"``) by ``row_expert [T]``.  The
    activation is ``glu_train``: the result is not the bits of ``ffn_mxfp4_grouped``.  ``rows="mxfp4"`` multiplies MXFP4 rows
    forward (``gemm_mxfp4_grouped_w4a4_train``), ``"bf16"`` the rows as they are."""
    if rows not in ("bf16", "mxfp4"):
        raise ValueError("rows is 'bf16' or 'mxfp4'")
    product = gemm_mxfp4_grouped_train if rows == "bf16" else gemm_mxfp4_grouped_w4a4_train
    gu = product(a_cat, blocks_gu, scales_gu, sizes, expert_ids)
    return product(glu_train(gu, act, bias=bias_gu, row_expert=row_expert), blocks_dn, scales_dn, sizes, expert_ids)
