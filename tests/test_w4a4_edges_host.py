"""The product of two MXFP4 operands on the host: stride rules of its C entry point, the tiles it plans.  No GPU needed."""
import ctypes

import pytest

import _gnf4b

SMS, SMEM = 148, 232448          # a B200
FIELDS = ("pair", "rows_w", "tok_cap", "xbox", "x_bytes", "x_blocks", "stages", "acc_bufs", "smem")


def plan(T, G, N, K, max_rows=-1, sms=SMS, smem=SMEM):
    out = (ctypes.c_int32 * len(FIELDS))()
    assert _gnf4b.load().gnf4b_w4a4_plan(T, G, N, K, max_rows, sms, smem, out) == 0
    return dict(zip(FIELDS, out))


def test_the_stride_of_a_dimension_of_one_is_not_checked():
    """The calls have too many items to be launched anywhere: what comes back is that, or, without a device, a CUDA error."""
    lib = _gnf4b.load()
    buf = ctypes.create_string_buffer(4096)
    p = (ctypes.addressof(buf) + 255) // 256 * 256
    T, G = (1 << 31) - 300, (1 << 31) - 1

    def call(N, E, wsn, wse):
        return lib.gnf4b_gemm_grouped_w4a4(p, p, T, p, wse, wsn, p, 2, 2, p, p, G, E, N, 64, -1, p, None, None)

    for N, E, wsn, wse in ((1, 4, 40, 64), (1, 4, 0, 64), (1, 4, -8, 64), (4, 1, 32, 72), (4, 1, 32, 0), (1, 1, 3, 5)):
        assert call(N, E, wsn, wse) in (-4, _gnf4b.ETOOBIG), (N, E, wsn, wse)
    for N, E, wsn, wse in ((2, 4, 40, 64), (2, 4, 0, 64), (1, 4, 32, 72), (1, 4, 32, -64), (4, 2, 32, 0)):
        assert call(N, E, wsn, wse) == _gnf4b.EUNSUPPORTED, (N, E, wsn, wse)


LENGTHS = sorted({1, 2, 15, 16, 17, 33, 64, 65, 96, 128, 129, 144, 192, 224, 240, 255, 256, 257, 300, 383, 384, 385, 511, 512, 1000, 20000})


@pytest.mark.parametrize("K", [32, 64, 768, 1280, 1312, 2048, 2080, 2880, 5120, 5152, 5376, 7168, 14336])
@pytest.mark.parametrize("G,N", [(1, 1), (4, 5760), (32, 61), (128, 2048), (2000, 1536)])
def test_planned_tiles_fit(G, N, K):
    """What the kernel's addresses rest on: shared memory, tensor memory, whole boxes, for every number of rows an item may have."""
    seen = set()
    for longest in LENGTHS:
        for T, hint in ((longest * G, longest), (longest, -1)):
            p = plan(T, G, N, K, hint)
            cap, pair = p["tok_cap"], p["pair"]
            seen.add(pair)
            assert pair in (0, 1) and p["acc_bufs"] in (1, 2) and 2 <= p["stages"] <= 12
            assert 64 <= p["rows_w"] <= 128 and p["rows_w"] % 8 == 0 and (not pair or p["rows_w"] == 128)
            assert 16 <= cap <= 256 and cap % (32 if pair else 16) == 0 and cap >= min(longest, 256)
            assert p["x_blocks"] == -(-cap // 128) and p["x_bytes"] % 1024 == 0
            # tiles of all stages, two spans of eight times 128 elements' scales, the group table, the barriers, 1 KiB of alignment
            table = 256 * 16 + 257 * 4 + 16 * 4 + 4
            barriers = 8 * (12 * 3 + 4 + 4) + 8
            need = p["stages"] * (16384 + p["x_bytes"]) + 2 * 8 * 512 * (1 + p["x_blocks"]) + (table + 15) // 16 * 16 + barriers
            assert need + 1023 <= p["smem"] <= SMEM
            # accumulators and the stages' scale slots
            columns = p["acc_bufs"] * cap + p["stages"] * 8 * (1 + p["x_blocks"])
            assert columns <= 512
            for tokens in range(1, cap + 1):
                mma = -(-tokens // (32 if pair else 16)) * (32 if pair else 16)          # rows that the MMA multiplies
                rows = mma // 2 if pair else tokens                                       # rows that this CTA loads
                assert mma <= cap and -(-rows // p["xbox"]) * p["xbox"] * 128 <= p["x_bytes"]
                assert (mma // 2 if pair else mma) * 128 <= p["x_bytes"]
                assert (p["acc_bufs"] - 1) * cap + -(-tokens // 32) * 32 <= 512           # the epilogue's last read
    if K in (1312, 2080, 2880, 5152):
        assert seen == {0, 1}


def test_a_plan_takes_no_nonsense():
    lib = _gnf4b.load()
    out = (ctypes.c_int32 * len(FIELDS))()
    assert lib.gnf4b_w4a4_plan(4, 4, 64, 64, -1, SMS, 48 << 10, out) == _gnf4b.EUNSUPPORTED
    assert lib.gnf4b_w4a4_plan(4, 4, 64, 64, -1, SMS, 1 << 10, out) == _gnf4b.EUNSUPPORTED
    ok = dict(T=4, G=4, N=64, K=64, max_rows=-1, sms=SMS, smem=SMEM)
    for bad, rc in ((dict(T=0), -1), (dict(G=0), -1), (dict(sms=0), -1), (dict(smem=0), -1), (dict(N=0), -2), (dict(K=48), -2),
                    (dict(T=(1 << 31) - 200), -6), (dict(K=1 << 32), -6)):
        v = {**ok, **bad}
        assert lib.gnf4b_w4a4_plan(v["T"], v["G"], v["N"], v["K"], v["max_rows"], v["sms"], v["smem"], out) == rc, bad
    assert lib.gnf4b_w4a4_plan(4, 4, 64, 64, -1, SMS, SMEM, None) == -1
