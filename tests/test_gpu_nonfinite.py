"""A NaN or an infinity on its way through the experts' activation and FFN: it stays non-finite in its own row and leaves the
others alone."""
import pytest
import torch

import mxfp4_grouped as M
import nf4_grouped
import nf4_qlora as Q
import synth

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
NAN, INF = float("nan"), float("inf")


def gen(seed):
    return torch.Generator().manual_seed(seed)


def chain(gu):
    """The activation as a chain of bf16 tensor operations."""
    gate, up = gu[..., 0::2].clamp(max=7.0), gu[..., 1::2].clamp(-7.0, 7.0)
    return (up + 1) * (gate * torch.sigmoid(gate * 1.702))


def same(a, b):
    return torch.equal(torch.isnan(a), torch.isnan(b)) and torch.equal(a.nan_to_num(nan=0.0), b.nan_to_num(nan=0.0))


def pairs():
    """Every pair of special and ordinary values as (gate, up), interleaved, [rows, 64]."""
    v = torch.tensor([NAN, -NAN, INF, -INF, 0.0, -0.0, 7.0, -7.0, 7.5, -7.5, 1.0, -0.25, 300.0, -300.0, 3.0, -3.0])
    return torch.stack(torch.meshgrid(v, v, indexing="ij"), -1).reshape(-1, 64).to(torch.bfloat16).to(DEV)


def test_gpt_oss_glu_keeps_nan():
    gu = pairs()
    got, want = M.glu_gpt_oss(gu), chain(gu)
    assert torch.isnan(got).any() and same(got, want)
    bias = torch.zeros(1, 64, dtype=torch.bfloat16, device=DEV)
    bias[0, 5] = NAN
    who = torch.zeros(gu.shape[0], dtype=torch.int64, device=DEV)
    assert same(M.glu_gpt_oss(gu, bias, who), chain(gu + bias)) and torch.isnan(M.glu_gpt_oss(gu, bias, who)[:, 2]).all()


def test_packed_and_training_glu_agree_on_what_is_not_finite():
    gu = pairs()
    bad = ~torch.isfinite(chain(gu)).reshape(gu.shape[0], 1, 32).all(-1)
    blocks, scales = M.glu_quantize_mxfp4(gu, "gpt_oss")
    assert torch.equal(scales == 255, bad) and bad.any()
    assert torch.equal(torch.isnan(Q.glu_train(gu, "gpt_oss")), torch.isnan(chain(gu)))


@pytest.mark.parametrize("bad", [NAN, INF, -INF])
@pytest.mark.parametrize("act", ["gpt_oss", "silu"])
@pytest.mark.parametrize("sizes", [[1, 1, 1, 1], [3, 20], [400]])
def test_ffn_on_mxfp4_rows_keeps_a_bad_row_bad(sizes, act, bad):
    E, K, h, N = 4, 1344, 96, 72
    g = gen(3)
    gu, dn = synth.mxfp4_stack(E, 2 * h, K, g, device=DEV), synth.mxfp4_stack(E, N, h, g, device=DEV)
    x = torch.randn(sum(sizes), K, generator=g).to(torch.bfloat16).to(DEV)
    ids = [(i + 2) % E for i in range(len(sizes))]
    clean = M.ffn_mxfp4_grouped_w4a4(x, *gu, *dn, sizes, ids, act=act)
    assert torch.isfinite(clean).all()
    x[1, 70] = bad
    out = M.ffn_mxfp4_grouped_w4a4(x, *gu, *dn, sizes, ids, act=act)
    assert not torch.isfinite(out[1]).any()
    rest = torch.arange(len(x), device=DEV) != 1
    assert torch.equal(out[rest], clean[rest])


@pytest.mark.parametrize("fused", [True, False])
@pytest.mark.parametrize("fmt", ["nf4", "mxfp4"])
@pytest.mark.parametrize("sizes", [[1, 1, 1, 1], [3, 20]])
def test_ffn_on_bf16_rows_keeps_nan(sizes, fmt, fused):
    E, K, h, N = 4, 128, 64, 72
    g = gen(4)
    stack = synth.nf4_stack if fmt == "nf4" else synth.mxfp4_stack
    gu, dn = stack(E, 2 * h, K, g, device=DEV), stack(E, N, h, g, device=DEV)
    x = torch.randn(sum(sizes), K, generator=g).to(torch.bfloat16).to(DEV)
    ids = [(i + 2) % E for i in range(len(sizes))]
    ffn = nf4_grouped.ffn_4bit_grouped if fmt == "nf4" else M.ffn_mxfp4_grouped      # SiLU and the clamped form
    clean = ffn(x, *gu, *dn, sizes, ids, fused=fused)
    x[1, 70] = NAN
    out = ffn(x, *gu, *dn, sizes, ids, fused=fused)
    assert torch.isnan(out[1]).all()
    rest = torch.arange(len(x), device=DEV) != 1
    assert torch.equal(out[rest], clean[rest])
