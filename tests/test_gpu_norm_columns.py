"""GPU tests of the norm calls on columns of one array: as on arrays of their own, bit for bit, with everything
between the columns left as it was."""
import pytest

import layer_reference as R

pytestmark = pytest.mark.gpu


def columns(rows, k, n, dtype, dev, gap=3):
    """An array of n matrices side by side, `gap` elements between them, and the matrices."""
    import torch
    wide = torch.full((rows, n * (k + gap) + gap), 7.0, dtype=dtype, device=dev)
    return wide, [wide[:, gap + i * (k + gap):gap + i * (k + gap) + k] for i in range(n)]


# every kernel's width: 4, 16, 64, 128, 256, 512 and 1024 lanes a row, rows in several trips; results past the L2
@pytest.mark.parametrize("rows,k", [(70, 20), (33, 100), (37, 333), (9, 777), (21, 1601), (5, 4100), (3, 9000), (3, 16001), (2, 40001), (9000, 1001)])
@pytest.mark.parametrize("kind", R.TYPES)
def test_columns(dev, rows, k, kind):
    import torch
    import fufft_amd as ff
    print(f"case norm columns {rows}x{k} {kind}", flush=True)
    t = R.torch_type(kind)
    x, res, dy, dt = (torch.randn(rows, k, device=dev).to(t) for _ in range(4))
    w = torch.randn(k, device=dev)

    def gaps(wide):
        g = wide.shape[1] - (wide.shape[1] - 3) // (k + 3) * k
        keep = torch.ones(wide.shape[1], dtype=torch.bool, device=dev)
        for i in range((wide.shape[1] - 3) // (k + 3)):
            keep[3 + i * (k + 3):3 + i * (k + 3) + k] = False
        assert int(keep.sum()) == g and bool((wide[:, keep] == 7).all())
    # x, residual, total and out side by side
    out, total = torch.empty_like(x), torch.empty_like(x)
    ff.rms_norm(x, w, out, residual=res, total=total)
    wide, (cx, cr, ct, co) = columns(rows, k, 4, t, dev)
    cx.copy_(x), cr.copy_(res)
    ff.rms_norm(cx, w, co, residual=cr, total=ct)
    assert torch.equal(co, out) and torch.equal(ct, total) and torch.equal(cx, x) and torch.equal(cr, res)
    ff.rms_norm(cx, w, co, residual=cr, total=cr)               # the residual in place, beside the others
    assert torch.equal(co, out) and torch.equal(cr, total) and torch.equal(cx, x)
    gaps(wide)
    # gradients
    dw, dw2, work = torch.empty(k, device=dev), torch.empty(k, device=dev), torch.empty(40, k, device=dev)
    dx = torch.empty_like(x)
    ff.rms_norm_grad(dy, total, w, dx, dw, work, dtotal=dt)
    wide, (cy, ch, ct, cd) = columns(rows, k, 4, t, dev)
    cy.copy_(dy), ch.copy_(total), ct.copy_(dt)
    ff.rms_norm_grad(cy, ch, w, cd, dw2, work, dtotal=ct)
    assert torch.equal(cd, dx) and torch.equal(dw2, dw) and torch.equal(cy, dy) and torch.equal(ch, total) and torch.equal(ct, dt)
    ff.rms_norm_grad(cy, ch, w, ct, dw2, work, dtotal=ct)       # in dtotal's place
    assert torch.equal(ct, dx) and torch.equal(dw2, dw) and torch.equal(cy, dy) and torch.equal(ch, total)
    gaps(wide)
