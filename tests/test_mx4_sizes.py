"""CPU test of the sizes that no launch of the 4-bit calls can hold: refused as unsupported, before
anything is launched.  (A launch of 2^32 lanes and more in x would run a part of them without an error.)"""
import fufft_amd as ff

P = [1 << 44, 2 << 44, 3 << 44, 4 << 44, 5 << 44, 6 << 44, 7 << 44]       # checked and never read
L = ff.lib


def test_sizes_beyond_a_launch():
    for k in (1 << 35, 1 << 38):                        # rows: 2^24 workgroups of 256 lanes
        assert L.fufft_mx4_quantize(P[0], 1, k, 1, k, 0, None, P[1], P[2], None, None, None) == ff.ERR_UNSUPPORTED
        assert L.fufft_mx4_dequantize(P[1], P[2], P[0], 1, k, 1, k, None) == ff.ERR_UNSUPPORTED
        assert L.fufft_mx4_cache_write(P[0], 1, k, P[1], 1, k, P[2], P[3], 1, None) == ff.ERR_UNSUPPORTED
        assert L.fufft_mx4_cache_read(P[0], P[1], 1, 1, k, P[2], 1, P[3], 1, 1, P[4], 1, 0, None) == ff.ERR_UNSUPPORTED
    k = 1 << 31                                         # along columns: a workgroup for 128
    assert L.fufft_mx4_quantize(P[0], 1, k, 1, k, 0, None, None, None, P[3], P[4], None) == ff.ERR_UNSUPPORTED
    assert L.fufft_mx4_cache_read(P[0], P[1], 1, 1, k, P[2], 1, P[3], 1, 1, P[4], 1, 1, None) == ff.ERR_UNSUPPORTED
    assert L.fufft_mx4_cache_conv(P[0], P[1], 1, 1, k, P[2], 1, P[3], 1, P[4], 1, 1, P[5], 0, None, 0, None) \
        == ff.ERR_UNSUPPORTED
    for m, n, k in ((1, 1 << 31, 128), (1, 1 << 28, 8192), (1 << 21, 1 << 21, 128), (1, 1, 1 << 38)):
        assert L.fufft_mx4_matmul(P[0], P[1], P[2], P[3], None, P[4], 1, n, m, n, k, None) == ff.ERR_UNSUPPORTED, (m, n, k)
    for m, n, k in ((1, 1 << 31, 128), (1, 1 << 28, 8192), (20, 1 << 31, 128), (1, 1, 1 << 38)):
        assert L.fufft_mx4_linear(P[0], 1, k, P[1], P[2], None, P[3], 1, n, m, n, k, None) == ff.ERR_UNSUPPORTED, (m, n, k)
