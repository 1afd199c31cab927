"""Cases for timing four operators of a mixture-of-experts layer, with their plain forms.

  quantize   rows -> MXFP4 (e2m1 elements and one e8m0 exponent per 32) and back (mxfp4_grouped.quantize_mxfp4,
             dequantize_mxfp4)
  product    grouped product of MXFP4 rows with MXFP4 expert stacks (mxfp4_grouped.gemm_mxfp4_grouped_w4a4)
  router     top-k routing, per-expert counts, balance and z losses, and the gradient of all of them with respect to the
             logits (ep_moe.route_topk_train)
  glu        the activation between an expert's two products whose backward pass reads an 8-bit checkpoint of its
             input (nf4_qlora.glu_train)

``run`` computes them with elementary tensor operations, or, where ``own`` is true, by the package's entry points.
"""
import sys
from pathlib import Path

import torch

own = False

E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0)
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
ALPHA, LIMIT = 1.702, 7.0           # the clamped GLU of gpt-oss
CKPT_BLOCK = 64                     # values per scale of the 8-bit checkpoint
CKPT_TINY = 2.0 ** -100             # a block whose largest magnitude is below this is held as zeros


def _package():
    root = str(Path(__file__).resolve().parents[1] / "grouped-nf4-gemm_b200")
    if root not in sys.path:
        sys.path.insert(0, root)


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one decoded token of gpt-oss-20b before its experts: a single row, latency is all there is
        {"name": "quantize-1x2880", "op": "quantize", "rows": 1, "k": 2880, "dtype": "bf16"},
        # a router-sized fp32 batch with an odd row count
        {"name": "quantize-1237x7168-fp32", "op": "quantize", "rows": 1237, "k": 7168, "dtype": "fp32"},
        # the rows of a gpt-oss-20b prefill of 8192 tokens, four experts each
        {"name": "quantize-32768x2880", "op": "quantize", "rows": 32768, "k": 2880, "dtype": "bf16"},
        # one decoded token of gpt-oss-20b: gate_up of its four experts, one row each
        {"name": "product-decode-gptoss", "op": "product", "experts": 32, "top_k": 4, "tokens": 1, "n": 5760, "k": 2880, "skew": 0.0},
        # 37 sequences decoding together through the down projection of Qwen3-30B-A3B: nearly every expert, few rows
        {"name": "product-batch37-qwen3-down", "op": "product", "experts": 128, "top_k": 8, "tokens": 37, "n": 2048, "k": 768, "skew": 0.0},
        # a 4096-token prefill through gate_up of Qwen3-30B-A3B
        {"name": "product-prefill-qwen3", "op": "product", "experts": 128, "top_k": 8, "tokens": 4096, "n": 1536, "k": 2048, "skew": 0.0},
        # an 8192-token prefill through gate_up of gpt-oss-20b with a few popular experts: ragged and long groups
        {"name": "product-prefill-gptoss-skewed", "op": "product", "experts": 32, "top_k": 4, "tokens": 8192, "n": 5760, "k": 2880, "skew": 1.1},
        # the router of a small micro-batch
        {"name": "router-64x128", "op": "router", "tokens": 64, "experts": 128, "top_k": 8, "mode": 0, "norm": True, "dtype": "fp32", "masked": 0.0},
        # gpt-oss's router (softmax over the chosen) on bf16 logits, a padded batch
        {"name": "router-8191x32-bf16", "op": "router", "tokens": 8191, "experts": 32, "top_k": 4, "mode": 1, "norm": False, "dtype": "bf16", "masked": 0.3},
        # a long-context training batch over 256 experts
        {"name": "router-65536x256", "op": "router", "tokens": 65536, "experts": 256, "top_k": 8, "mode": 0, "norm": False, "dtype": "fp32", "masked": 0.1},
        # an odd number of rows of Qwen3-30B-A3B between its expert products
        {"name": "glu-2047x768", "op": "glu", "rows": 2047, "h": 768, "act": "silu"},
        # gpt-oss-20b, a training batch of 8192 tokens with four experts each
        {"name": "glu-32768x2880-gptoss", "op": "glu", "rows": 32768, "h": 2880, "act": "gpt_oss"},
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, spread evenly over its logarithm."""
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(("quantize", "product", "product", "router", "glu"))
    if op == "quantize":
        k = 32 * _log(rng, 1, 224)
        dtype = rng.choice(("bf16", "bf16", "fp16", "fp32"))
        return {"op": op, "rows": _log(rng, 1, min(65536, (94_000_000 if dtype != "fp32" else 47_000_000) // k)), "k": k, "dtype": dtype}
    if op == "product":
        n = rng.choice((8 * _log(rng, 8, 720), _log(rng, 64, 5760)))
        k = 32 * _log(rng, 2, 224)
        experts = _log(rng, 4, max(4, min(128, 530_000_000 // (n * k))))
        top_k = rng.randint(1, min(8, experts))
        # the plain form pads every expert's rows to the longest group
        most = min(8192, int(3.0e11 / (n * k * top_k)), int(4.0e12 / (n * k * experts)), int(2.2e9 / (experts * (n + k))))
        tokens = _log(rng, 1, max(1, most))
        return {"op": op, "experts": experts, "top_k": top_k, "tokens": tokens, "n": n, "k": k, "skew": rng.choice((0.0, 0.0, 0.6, 1.1))}
    if op == "router":
        experts = rng.choice((8, 16, 32, 60, 64, 96, 128, 160, 256, 384, 512))
        mode = rng.randint(0, 1)
        return {"op": op, "tokens": _log(rng, 1, min(131072, 16_000_000 // experts)), "experts": experts, "top_k": rng.randint(1, min(10, experts)),
                "mode": mode, "norm": mode == 0 and rng.random() < 0.5, "dtype": rng.choice(("fp32", "fp32", "bf16")), "masked": rng.choice((0.0, 0.1, 0.5))}
    h = rng.choice((8 * _log(rng, 8, 512), _log(rng, 64, 4096)))
    return {"op": op, "rows": _log(rng, 1, min(65536, 94_000_000 // h)), "h": h, "act": rng.choice(("silu", "gpt_oss"))}


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dev = torch.device("cuda")
    s = {"case": case}
    if case["op"] == "quantize":
        # hidden rows: normal values, a few columns much larger than the rest
        x = torch.randn(case["rows"], case["k"], generator=g, device=dev)
        x *= 1.0 + 15.0 * (torch.rand(case["k"], generator=g, device=dev) < 0.01)
        s["x"] = x.to(DTYPES[case["dtype"]])
    elif case["op"] == "product":
        E, n, k, top_k, tokens = (case[f] for f in ("experts", "n", "k", "top_k", "tokens"))
        s["w"] = torch.randint(0, 256, (E, n, k // 2), generator=g, device=dev, dtype=torch.uint8)
        s["ws"] = torch.randint(119, 126, (E, n, k // 32), generator=g, device=dev, dtype=torch.uint8)
        logits = torch.randn(tokens, E, generator=g, device=dev)
        if case["skew"]:
            rank = torch.randperm(E, generator=g, device=dev) + 1.0
            logits -= case["skew"] * torch.log(rank)
        ids = torch.argsort(-logits, dim=1, stable=True)[:, :top_k]
        count = torch.zeros(E, dtype=torch.int64, device=dev).scatter_add_(0, ids.reshape(-1), torch.ones_like(ids.reshape(-1)))
        used = torch.nonzero(count).reshape(-1)
        s["sizes"] = count[used]
        s["ids"] = used.to(torch.int32)
        s["offsets"] = torch.cat((torch.zeros_like(used[:1]), torch.cumsum(s["sizes"], 0))).to(torch.int32)
        s["widest"] = int(count.max())
        rows = tokens * top_k
        s["x"] = torch.randint(0, 256, (rows, k // 2), generator=g, device=dev, dtype=torch.uint8)
        s["xs"] = torch.randint(124, 129, (rows, k // 32), generator=g, device=dev, dtype=torch.uint8)
    elif case["op"] == "router":
        T, E, k = case["tokens"], case["experts"], case["top_k"]
        s["logits"] = (1.5 * torch.randn(T, E, generator=g, device=dev)).to(DTYPES[case["dtype"]])
        s["mask"] = torch.rand(T, generator=g, device=dev) >= case["masked"] if case["masked"] else None
        s["g_w"] = torch.randn(T, k, generator=g, device=dev)
        s["g_balance"] = 0.01 * (1 + torch.rand((), generator=g, device=dev)) * T
        s["g_z"] = 0.001 * (1 + torch.rand((), generator=g, device=dev)) * T
    else:
        s["gate_up"] = (2.0 * torch.randn(case["rows"], 2 * case["h"], generator=g, device=dev)).to(torch.bfloat16)
        s["g_out"] = torch.randn(case["rows"], case["h"], generator=g, device=dev).to(torch.bfloat16)
    return s


# ------------------------------------------------------------------------------------------------ plain forms
def _values(blocks, scales):
    """The numbers that packed MXFP4 rows stand for, fp32 (every one is exact)."""
    table = torch.tensor(E2M1, device=blocks.device)
    codes = torch.stack((blocks & 15, blocks >> 4), dim=-1).to(torch.int32)
    v = table[codes].reshape(*scales.shape, 32)
    return (v * torch.exp2(scales.float() - 127.0)[..., None]).reshape(*blocks.shape[:-1], -1)


def _plain_quantize(x):
    b = x.float().reshape(x.shape[0], -1, 32)
    top = b.abs().amax(-1).clamp_min(1e-20).double()
    # the least power of two that brings the block's largest magnitude to at most 6: frexp is exact at the borders
    m, p = torch.frexp(top / 4.0)
    e = torch.where(m <= 0.75, p - 1, p).clamp(-127, 127)
    v = torch.ldexp(b.double(), -e[..., None])
    a = v.abs()
    steps = torch.tensor((0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0), device=x.device, dtype=torch.float64)
    code = torch.bucketize(a, steps)                      # the nearest entry, the lower one on a tie
    mags = torch.tensor(E2M1[:8], device=x.device, dtype=torch.float64)[code]
    values = torch.ldexp(torch.where(v < 0, -mags, mags), e[..., None]).reshape(x.shape)
    return values.to(_held(x.dtype)), (e + 127).to(torch.uint8)


def _held(dtype):
    """The type that MXFP4 values of rows of this type are read back in: one that holds each of them exactly."""
    return torch.bfloat16 if dtype == torch.bfloat16 else torch.float32


def _plain_product(s):
    sizes, rows = s["sizes"], s["x"].shape[0]
    groups = sizes.numel()
    at = torch.arange(rows, device=sizes.device)
    grp = torch.repeat_interleave(torch.arange(groups, device=sizes.device), sizes, output_size=rows)
    pos = at - s["offsets"].long()[grp]
    w = _values(s["w"][s["ids"].long()], s["ws"][s["ids"].long()])
    x = torch.zeros(groups, s["widest"], w.shape[2], device=w.device)
    x[grp, pos] = _values(s["x"], s["xs"])
    return torch.bmm(x, w.transpose(1, 2))[grp, pos].to(torch.bfloat16)


def _plain_router(s):
    c, lg = s["case"], s["logits"].float()
    T, E, k = c["tokens"], c["experts"], c["top_k"]
    keep = torch.ones(T, dtype=torch.bool, device=lg.device) if s["mask"] is None else s["mask"]
    idx = torch.argsort(-lg, dim=1, stable=True)[:, :k]
    top = lg.amax(1, keepdim=True)
    ex = torch.exp(lg - top)
    z = ex.sum(1, keepdim=True)
    p = ex / z
    lse = (top + torch.log(z)).squeeze(1)
    sel = torch.gather(p, 1, idx)
    renorm = c["mode"] == 1 or c["norm"]
    w = sel / sel.sum(1, keepdim=True) if renorm else sel
    hit = torch.zeros_like(lg).scatter_(1, idx, 1.0) * keep[:, None]
    counts = hit.sum(0).to(torch.int32)
    n = keep.sum().clamp_min(1)
    share = counts.float() / (n * k)
    mean_p = (p * keep[:, None]).sum(0) / n
    balance = E * (share * mean_p).sum()
    z_loss = (lse.square() * keep).sum() / n
    # gradient: of the weights, of the balance loss (its shares are constants), of the z loss
    g_w = s["g_w"]
    if renorm:
        d = torch.zeros_like(lg).scatter_(1, idx, w * (g_w - (g_w * w).sum(1, keepdim=True)))
    else:
        d = p * (torch.zeros_like(lg).scatter_(1, idx, g_w) - (g_w * w).sum(1, keepdim=True))
    a = s["g_balance"] * E * share / n
    b = p * (a - (p * a).sum(1, keepdim=True)) + p * (2.0 * s["g_z"] * lse / n)[:, None]
    return {"idx": idx, "weights": w, "counts": counts, "balance": balance, "z": z_loss, "grad": (d + b * keep[:, None]).to(s["logits"].dtype)}


def _ckpt(v):
    """v [rows, h] as its 8-bit checkpoint holds it: whole steps of a 127th of the block's largest magnitude."""
    rows, h = v.shape
    pad = -h % CKPT_BLOCK
    b = torch.cat((v, v.new_zeros(rows, pad)), 1).reshape(rows, -1, CKPT_BLOCK) if pad else v.reshape(rows, -1, CKPT_BLOCK)
    top = b.abs().amax(-1, keepdim=True)
    top = torch.where(top < CKPT_TINY, torch.zeros_like(top), top)
    q = torch.where(top > 0, torch.round(b * (127.0 / top)), torch.zeros_like(b))
    return (q * (top / 127.0)).reshape(rows, -1)[:, :h]


def _glu_parts(gate_up, act):
    h = gate_up.shape[1] // 2
    f = gate_up.float()
    return (f[:, :h], f[:, h:]) if act == "silu" else (f[:, 0::2], f[:, 1::2])


def _glu_joined(g, u, act):
    return torch.cat((g, u), 1) if act == "silu" else torch.stack((g, u), -1).reshape(g.shape[0], -1)


def _plain_glu(s):
    act = s["case"]["act"]
    g, u = _glu_parts(s["gate_up"], act)
    go = s["g_out"].float()
    cg, cu = _ckpt(g), _ckpt(u)
    if act == "silu":
        out = g / (1.0 + torch.exp(-g)) * u
        sig = 1.0 / (1.0 + torch.exp(-cg))
        dg = go * cu * sig * (1.0 + cg * (1.0 - sig))
        du = go * cg * sig
    else:
        g7, u7 = g.clamp(max=LIMIT), u.clamp(-LIMIT, LIMIT)
        out = (u7 + 1.0) * g7 / (1.0 + torch.exp(-ALPHA * g7))
        g7, u7 = cg.clamp(max=LIMIT), cu.clamp(-LIMIT, LIMIT)
        sig = 1.0 / (1.0 + torch.exp(-ALPHA * g7))
        dg = go * (u7 + 1.0) * sig * (1.0 + ALPHA * g7 * (1.0 - sig)) * (cg <= LIMIT)
        du = go * g7 * sig * (cu.abs() <= LIMIT)
    return {"out": out.to(torch.bfloat16), "grad": _glu_joined(dg, du, act).to(torch.bfloat16)}


# ------------------------------------------------------------------------------------------------ one pass
def run(s):
    c = s["case"]
    if not own:
        if c["op"] == "quantize":
            values, scales = _plain_quantize(s["x"])
            return {"values": values, "scales": scales}
        return {"product": _plain_product, "router": _plain_router, "glu": _plain_glu}[c["op"]](s)
    _package()
    if c["op"] == "quantize":
        import mxfp4_grouped
        blocks, scales = mxfp4_grouped.quantize_mxfp4(s["x"])
        return {"values": mxfp4_grouped.dequantize_mxfp4(blocks, scales, _held(s["x"].dtype)), "scales": scales}
    if c["op"] == "product":
        import mxfp4_grouped
        return mxfp4_grouped.gemm_mxfp4_grouped_w4a4(s["x"], s["xs"], s["w"], s["ws"], None, s["ids"], group_offsets=s["offsets"],
                                                     max_rows=s["widest"])
    if c["op"] == "router":
        import ep_moe
        logits = s["logits"].detach().requires_grad_()
        r = ep_moe.route_topk_train(logits, c["top_k"], c["mode"], c["norm"], token_mask=s["mask"])
        grad, = torch.autograd.grad((r.weights, r.balance_loss, r.z_loss), (logits,), (s["g_w"], s["g_balance"], s["g_z"]))
        return {"idx": r.idx, "weights": r.weights.detach(), "counts": r.counts, "balance": r.balance_loss.detach(), "z": r.z_loss.detach(), "grad": grad}
    import nf4_qlora
    gate_up = s["gate_up"].detach().requires_grad_()
    out = nf4_qlora.glu_train(gate_up, c["act"])
    grad, = torch.autograd.grad(out, gate_up, s["g_out"])
    return {"out": out.detach(), "grad": grad}


def work(case):
    if case["op"] == "quantize":
        n = case["rows"] * case["k"]
        # there: the rows in, the packed form out; back: the packed form in, its values out
        read, back = (2 if case["dtype"] != "fp32" else 4), (2 if case["dtype"] == "bf16" else 4)
        return {"bytes": n * (read + back) + 2 * n * 17 / 32, "flops": 3 * n}
    if case["op"] == "product":
        rows, n, k = case["tokens"] * case["top_k"], case["n"], case["k"]
        # experts that get a token: all that the choices can reach, or the number expected of an even choice
        reached = min(case["experts"], case["experts"] * (1 - (1 - case["top_k"] / case["experts"]) ** case["tokens"]) if case["tokens"] > 1 else case["top_k"])
        return {"bytes": reached * n * k * 17 / 32 + rows * k * 17 / 32 + 2 * rows * n, "flops": 2 * rows * n * k}
    if case["op"] == "router":
        T, E, k = case["tokens"], case["experts"], case["top_k"]
        item = 4 if case["dtype"] == "fp32" else 2
        # logits read forward and backward, the gradient written; ids, weights and their gradient; the mask
        return {"bytes": 3 * T * E * item + T * k * (8 + 4 + 4) + T + 4 * E, "flops": 12 * T * E}
    n = case["rows"] * case["h"]
    # forward: the bf16 pair in, the result and the 8-bit pair out; backward: the 8-bit pair and the gradient in, the pair's out
    return {"bytes": n * (4 + 2 + 2) + n * (2 + 2 + 4) + 4 * 4 * n / CKPT_BLOCK, "flops": 40 * n}


# ------------------------------------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    f64 = torch.float64
    if case["op"] == "quantize":
        x = s["x"].to(f64).reshape(case["rows"], -1, 32)
        mags = x.abs()
        e = torch.full(mags.shape[:2], -69.0, dtype=f64, device=x.device)      # the exponent of the least scale, 6 * 2^-69 > 1e-20
        top = mags.amax(-1)
        guess = torch.ceil(torch.log2((top / 6.0).clamp_min(1e-30))) - 1
        guess = torch.where(top > 6.0 * torch.exp2(guess), guess + 1, guess)
        e = torch.maximum(e, torch.where(top > 6.0 * torch.exp2(guess), guess + 1, guess))
        a = mags / torch.exp2(e)[..., None]
        # half steps below 2, whole steps below 4, steps of two above; the lower of two equally near
        low, mid, high = torch.ceil(2 * a - 0.5) / 2, torch.ceil(a - 0.5), 2 * torch.ceil(a / 2 - 0.5)
        v = torch.where(a <= 2, low, torch.where(a <= 4, mid, high))
        return {"values": (torch.sign(x) * v * torch.exp2(e)[..., None]).reshape(s["x"].shape), "scales": None}
    if case["op"] == "product":
        def num(b, sc):
            lo, hi = (b & 15).to(torch.int16), (b >> 4).to(torch.int16)
            c = torch.stack((lo, hi), -1).reshape(*b.shape[:-1], -1)
            m = (c & 7).to(f64)
            v = torch.where(m < 4, m / 2, torch.where(m < 6, m - 2, 2 * m - 8))
            v = torch.where(c > 7, -v, v).reshape(*sc.shape, 32)
            return torch.ldexp(v, (sc.to(torch.int32) - 127)[..., None]).reshape(c.shape)
        sizes = s["sizes"].tolist()
        parts = [num(x, xs) @ num(s["w"][e], s["ws"][e]).t()
                 for x, xs, e in zip(s["x"].split(sizes), s["xs"].split(sizes), s["ids"].tolist())]
        return torch.cat(parts)
    if case["op"] == "router":
        lg = s["logits"].to(f64).requires_grad_()
        T, E, k = case["tokens"], case["experts"], case["top_k"]
        keep = torch.ones(T, dtype=f64, device=lg.device) if s["mask"] is None else s["mask"].to(f64)
        _, idx = torch.sort(lg.detach(), dim=1, descending=True, stable=True)
        idx = idx[:, :k]
        logp = torch.log_softmax(lg, 1)
        chosen = torch.gather(lg if (case["mode"] == 1 or case["norm"]) else logp, 1, idx)
        w = torch.softmax(chosen, 1) if (case["mode"] == 1 or case["norm"]) else torch.exp(chosen)
        n = max(1.0, float(keep.sum()))
        counts = torch.bincount(idx[keep > 0].reshape(-1), minlength=E).to(f64)
        balance = E * (counts / (n * k) * (torch.exp(logp) * keep[:, None]).sum(0) / n).sum()
        z = (torch.logsumexp(lg, 1) ** 2 * keep).sum() / n
        total = (w * s["g_w"].to(f64)).sum() + balance * s["g_balance"].to(f64) + z * s["g_z"].to(f64)
        grad, = torch.autograd.grad(total, lg)
        return {"idx": None, "weights": w.detach(), "counts": None, "balance": balance.detach(), "z": z.detach(), "grad": grad}
    gu = s["gate_up"].to(f64)
    rows, h = case["rows"], case["h"]
    pair = gu.reshape(rows, 2, h) if case["act"] == "silu" else gu.reshape(rows, h, 2).transpose(1, 2)

    def formula(p):
        if case["act"] == "silu":
            return torch.nn.functional.silu(p[:, 0]) * p[:, 1]
        gate, up = torch.clamp(p[:, 0], max=LIMIT), torch.clamp(p[:, 1], min=-LIMIT, max=LIMIT)
        return (up + 1) * gate * torch.sigmoid(ALPHA * gate)

    held = torch.zeros(rows, 2, -(-h // CKPT_BLOCK) * CKPT_BLOCK, dtype=f64, device=gu.device)
    held[:, :, :h] = pair
    blocks = held.view(rows, 2, -1, CKPT_BLOCK)
    step = blocks.abs().amax(-1, keepdim=True) / 127.0
    held = (torch.round(blocks / step.clamp_min(1e-300)) * step).view(rows, 2, -1)[:, :, :h].detach().requires_grad_()
    grad, = torch.autograd.grad(formula(held), held, s["g_out"].to(f64))
    grad = grad.reshape(rows, 2 * h) if case["act"] == "silu" else grad.transpose(1, 2).reshape(rows, 2 * h)
    return {"out": formula(pair), "grad": grad}
