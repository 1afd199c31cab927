"""The product of two MXFP4 operands on the host: stride rules of its C entry point.  No GPU needed."""
import ctypes

import _gnf4b


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
