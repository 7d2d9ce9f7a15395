"""CPU test: mx4_linear's rows and results as columns of one array are refused where they share a byte."""
import fufft_amd as ff

INV = ff.ERR_INVALID
X, W, S = 0x10000000, 0x20000000, 0x30000000          # addresses that are checked and never read


def linear(o, x=X, ldx=100, xt=0, ld=100, type=0, m=4, n=8, k=64):
    return ff.lib.fufft_mx4_linear(x, xt, ldx, W, S, None, o, type, ld, m, n, k, None)


def test_columns_that_share_a_byte_are_refused():
    for bad in (dict(o=X), dict(o=X + 4 * 63), dict(o=X + 4 * 93), dict(o=X + 4 * 363), dict(o=X - 4 * 7), dict(o=X - 400 - 28),
                dict(o=X + 4 * 64, ld=101), dict(o=X + 4 * 64, ldx=101), dict(o=X + 4 * 63, m=1),
                dict(o=X + 2 * 127, type=1, ld=200), dict(o=X + 4 * 64, type=1, ld=100), dict(o=X + 4 * 64, n=37)):
        assert linear(**bad) == INV, bad
