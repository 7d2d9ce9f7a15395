"""CPU tests: the norm calls' rows may be columns of one array.  2^30 rows are more than a launch holds and are
refused last of all, as unsupported, so that nothing is launched here; the gradients have no such end and are only tested where they
are refused."""
import fufft_amd as ff

INV, UNSUP = ff.ERR_INVALID, ff.ERR_UNSUPPORTED
P = [(i + 1) << 44 for i in range(10)]          # addresses that are checked and never read
ROWS, K, LD = 1 << 30, 200, 1000


def norm(x=P[0], ldx=LD, res=None, ldr=LD, total=None, ldt=LD, st=1, w=P[1], o=P[2], ldo=LD, c=None, s=None, rows=ROWS):
    return ff.lib.fufft_rms_norm(x, 1, ldx, res, ldr, total, ldt, st, w, 1e-6, o, ldo, c, s, rows, K, None)


def test_norm():
    at = lambda col, size=2: P[0] + col * size  # noqa: E731
    taken = [dict(), dict(o=at(200)), dict(o=at(800)), dict(o=at(500)), dict(x=at(800), o=at(0)), dict(x=at(400), o=at(200), res=at(600), total=at(0)),
             dict(o=at(200), res=at(400), total=at(600)), dict(o=at(200), res=at(400), total=at(400)), dict(o=at(200), total=at(0)),
             # an fp32 stream beside bf16 rows: the same bytes from row to row
             dict(o=at(200), res=at(400), total=at(400), st=0, ldr=LD // 2, ldt=LD // 2),
             dict(o=at(200), res=at(400), total=at(800), st=0, ldr=LD, ldt=LD, ldx=2 * LD, ldo=2 * LD)]
    for call in taken:
        assert norm(**call) == UNSUP, call
    refused = [dict(o=at(199)), dict(o=at(1)), dict(o=at(801)), dict(x=at(200), o=at(1)), dict(o=at(200), ldo=LD + 1), dict(o=at(200), ldo=LD - 2),
               dict(o=at(200), total=at(200)), dict(o=at(200), total=at(399)), dict(o=at(200), res=at(399)), dict(o=at(0), total=at(0)),
               dict(o=at(200), res=at(400), total=at(599)), dict(o=at(200), res=at(400), total=at(798), st=0, ldr=LD // 2, ldt=LD // 2),
               # what lies without gaps, among an output's rows: the weight, codes
               dict(o=at(200), w=at(500)), dict(o=at(200), c=at(504), s=P[5])]
    for call in refused:
        assert norm(**call) == INV, call


def test_norm_grad_refusals():
    def grad(dy=P[0], h=P[1], dt=None, dx=P[2], ldy=LD, ldh=LD, ldt=LD, ldx=LD):
        return ff.lib.fufft_rms_norm_grad(dy, 1, ldy, h, ldh, dt, ldt, 1, P[3], 1e-6, dx, 1, ldx, P[4], P[5], 8, 1 << 20, K, None)
    at = lambda col: P[0] + col * 2  # noqa: E731
    for bad in (dict(dx=at(199)), dict(h=at(400), dx=at(201)), dict(h=at(400), dx=at(400)), dict(h=at(200), dx=at(801)), dict(dx=at(200), ldx=LD + 2),
                dict(dt=at(400), dx=at(300)), dict(dt=at(400), dx=at(400), ldt=LD + 1)):
        assert grad(**bad) == INV, bad
