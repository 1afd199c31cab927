"""Argument checks of the MXFP4 quantiser and of the product of two MXFP4 operands: no GPU needed."""
import ctypes

import pytest
import torch

import _gnf4b
import mxfp4_grouped as M

u8 = torch.uint8


def test_cpu_tensors_are_refused_with_the_cpu_counterpart():
    with pytest.raises(RuntimeError, match="quantize_pack_mxfp4"):
        M.quantize_mxfp4(torch.zeros(2, 64))
    with pytest.raises(RuntimeError, match="dequant_mxfp4"):
        M.dequantize_mxfp4(torch.zeros(2, 32, dtype=u8), torch.zeros(2, 2, dtype=u8))
    with pytest.raises(RuntimeError, match="dequant_mxfp4"):
        M.gemm_mxfp4_grouped_w4a4(torch.zeros(2, 32, dtype=u8), torch.zeros(2, 2, dtype=u8), torch.zeros(1, 8, 32, dtype=u8),
                                  torch.zeros(1, 8, 2, dtype=u8), [2], [0])
    with pytest.raises(RuntimeError, match="CUDA"):
        M.glu_quantize_mxfp4(torch.zeros(2, 64, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="act is"):
        M.glu_quantize_mxfp4(torch.zeros(2, 64, dtype=torch.bfloat16), act="relu")


def test_c_entry_points_check_before_they_launch():
    """Every refusal here returns before anything touches a device (this runs without one)."""
    lib = _gnf4b.load()
    buf = ctypes.create_string_buffer(4096)
    p = (ctypes.addressof(buf) + 255) // 256 * 256
    q = lib.gnf4b_quantize_mxfp4
    assert q(p, 3, 1, 32, 32, p, p, None) == -1 and q(p, 0, -1, 32, 32, p, p, None) == -1
    assert q(p, 0, 1, 48, 48, p, p, None) == -2 and q(p, 0, 1, 0, 0, p, p, None) == -2
    assert q(None, 0, 1, 32, 32, p, p, None) == -1 and q(p, 0, 1, 32, 32, p + 1, p, None) == -1
    assert q(p, 2, 1, 32, 32, p, None, None) == -1 and q(p + 2, 2, 1, 32, 32, p, p, None) == -1
    assert q(p, 0, 1, 32, -32, p, p, None) == -1 and q(p, 0, 1 << 62, 32, 32, p, p, None) == -6
    assert q(None, 0, 0, 32, 32, None, None, None) == 0
    d = lib.gnf4b_dequantize_mxfp4
    assert d(p, p, -1, 0, p, None) == -1 and d(p, p, 1, 5, p, None) == -1 and d(p, p, 1, 0, p + 2, None) == -1
    assert d(p, None, 1, 0, p, None) == -1 and d(p, p, 1 << 62, 0, p, None) == -6 and d(None, None, 0, 0, None, None) == 0
    g = lib.gnf4b_glu_quantize_mxfp4
    assert g(p, 1, 32, 2, None, None, 0, p, p, None, None) == -1 and g(p, 1, 40, 0, None, None, 0, p, p, None, None) == -2
    assert g(p, 1, 32, 0, p, p, 1, p, p, None, None) == -1 and g(p, 1, 32, 1, p, None, 1, p, p, None, None) == -1
    assert g(p, 1, 32, 1, p, p, 0, p, p, None, None) == -1 and g(None, 0, 32, 0, None, None, 0, None, None, None, None) == 0
    m = lib.gnf4b_gemm_grouped_w4a4

    def call(xb=p, xs=p, T=4, W=p, wse=1024, wsn=32, S=p, sse=64, ssn=2, off=p, ids=p, G=1, E=1, N=32, K=64, out=p):
        return m(xb, xs, T, W, wse, wsn, S, sse, ssn, off, ids, G, E, N, K, -1, out, None, None)

    assert call(T=-1) == -1 and call(G=-1) == -1 and call(K=48) == -2 and call(N=0) == -2 and call(E=0) == -2
    assert call(T=(1 << 31) - 200) == -6 and call(N=(1 << 31) - 200) == -6 and call(K=1 << 32) == -6
    assert call(xb=None) == -1 and call(xs=None) == -1 and call(W=None) == -1 and call(S=None) == -1
    assert call(off=None) == -1 and call(ids=None) == -1 and call(out=None) == -1 and call(out=p + 2) == -1
    assert call(sse=-1) == -1 and call(ssn=-2) == -1
    assert call(xb=p + 8) == -5 and call(W=p + 4) == -5 and call(wsn=40) == -5 and call(wsn=-32) == -5 and call(E=2, wse=0) == -5
    assert call(T=0) == 0 and call(G=0) == 0


@pytest.mark.parametrize("T,G,N,max_rows", [(1, 1, 1, 1), (4, 4, 5760, 1), (296, 128, 2048, 8), (32768, 128, 1536, -1), (300, 3, 100, 129)])
def test_tile_plan_fits(T, G, N, max_rows):
    """The tile plan restated: shared memory, tensor memory and the loads' bounds for every row cap."""
    for longest in sorted({1, 16, 17, 33, 64, 65, 128, 129, 144, 192, 224, 240, 255, 256, min(T, max_rows if max_rows > 0 else T)}):
        cap = (min(longest, 256) + 15) // 16 * 16
        box = 16 if cap <= 16 else 32 if cap <= 64 else 64
        x_rows = (cap + box - 1) // box * box
        blocks = (cap + 127) // 128
        stage = 16384 + x_rows * 128
        span = 8 * 512 * (1 + blocks)
        fixed = 1024 + 2 * span + 256 * 16 + 257 * 4 + 16 * 4 + 4 + 512
        stages = min(12, (232448 - fixed) // stage)
        assert stages >= 4 and fixed + stages * stage <= 232448
        slots = stages * 8 * (1 + blocks)
        bufs = 2 if 2 * cap + slots <= 512 else 1
        assert bufs * cap + slots <= 512
        for tokens in range(1, cap + 1):
            assert (tokens + box - 1) // box * box <= x_rows and (tokens + 15) // 16 * 16 <= x_rows
            # the widest read of the epilogue stays in tensor memory
            assert (bufs - 1) * cap + (tokens + 31) // 32 * 32 <= 512
