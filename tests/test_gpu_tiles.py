"""The row norm, its gradient and the distillation loss where a workgroup walks several groups of rows one after the other:
reductions whose LDS slots are used again, weight gradients carried over groups, rows fetched ahead across the mask's
transitions.  Against the formulas in float64 on every row, with the tolerances derived in the operators' own tests."""
import pytest

from test_gpu_distill import _case, _check
from test_gpu_distill import _reference as _distillation
from test_gpu_norm import U, _check_rows, _inputs, _reference

pytestmark = pytest.mark.gpu


# two or more groups from 8192 groups on: 64 / G rows of a wave up to 1024 columns times four waves, one row past that
@pytest.mark.parametrize('n,f', [(530001, 16), (131111, 60), (33001, 250), (40003, 1000), (8200, 1030), (16500, 1433), (8199, 4100),
                                 (8193, 8200), (8195, 17003)])
def test_norm(n, f):
    import torch
    from gcn_amd import sparse
    x, r, w, _, _ = _inputs(n, f)
    x *= torch.logspace(-3, 3, n, device='cuda')[:, None]            # neighbouring rows differ: a stale sum would show
    x[1::2] *= 100.0
    y, h, inv = sparse.rms_norm(x, w, residual=r, eps=1e-5)
    assert torch.equal(h, x + r)
    q, h2, inv2 = sparse.rms_norm(x, w, residual=r, eps=1e-5, quant=True)
    assert torch.equal(h2, h) and torch.equal(inv2, inv)
    for lo in range(0, n, 1 << 15):
        rows = slice(lo, min(n, lo + (1 << 15)))
        ry, _, rinv = _reference(h[rows], None, w, 1e-5)
        assert bool(((inv[rows].double() - rinv).abs() <= 64 * U * rinv).all())
        assert bool(((y[rows].double() - ry).abs() <= 70 * U * ry.abs()).all())
        _check_rows(q.rows(rows.start, rows.stop), ry, None)


# two or more groups from 2049 groups on
@pytest.mark.parametrize('n,f', [(140001, 16), (300001, 60), (9000, 200), (20001, 1000), (5000, 1433), (4099, 2500), (2500, 8193),
                                 (2300, 16384), (4100, 17003)])
def test_norm_gradient(n, f):
    import torch
    from gcn_amd import sparse
    h, dy, w, dh, _ = _inputs(n, f, 1)
    h *= torch.logspace(-2, 2, n, device='cuda')[:, None]
    _, _, inv = sparse.rms_norm(h, w)
    for up in (None, dh):
        dx, dw = sparse.rms_norm_grad(dy, h, w, inv, grad_h=up)
        total = torch.zeros(f, dtype=torch.float64, device='cuda')
        size = torch.zeros(f, dtype=torch.float64, device='cuda')
        for lo in range(0, n, 1 << 14):
            rows = slice(lo, min(n, lo + (1 << 14)))
            g, hd, i = dy[rows].double() * w.double(), h[rows].double(), inv[rows].double()[:, None]
            along, reach = (g * hd).sum(1, keepdim=True) / f, (g * hd).abs().sum(1, keepdim=True) / f
            plus = 0 if up is None else up[rows].double()
            rdx = i * (g - hd * i * i * along) + plus
            bound = i * (g.abs() + hd.abs() * i * i * reach) + (0 if up is None else plus.abs())
            assert bool(((dx[rows].double() - rdx).abs() <= 128 * U * bound).all())
            terms = dy[rows].double() * hd * i
            total += terms.sum(0)
            size += terms.abs().sum(0)
        # the h inv of a term is rounded once and the term once; a lane adds n / 2048 or fewer groups one after the other,
        # then come 64 rows of a tree: within 4096 u of the magnitudes
        assert bool(((dw.double() - total).abs() <= 4096 * U * size).all())
        assert torch.equal(sparse.rms_norm_grad(dy, h, w, inv, grad_h=up)[1], dw)


# two or more groups from 8192 groups of 256 / G rows on; lists of one, two and four entries a lane and longer ones
@pytest.mark.parametrize('n,c,k', [(2100001, 3, 2), (1050001, 7, 3), (1050001, 7, 9), (530001, 20, 4), (530001, 20, 8), (530001, 20, 16),
                                   (530001, 20, 20), (270001, 47, 5), (270001, 47, 12), (270001, 47, 20), (270001, 47, 40),
                                   (140001, 100, 70), (70001, 200, 9), (70001, 200, 140)])
def test_distillation(n, c, k):
    import torch
    from gcn_amd import sparse
    for kept, dtype in ((0.5, 'float16'), (0.97, 'float32')):
        logits, values, idx, mask = _case(n, c, k, kept=kept, dtype=dtype)
        idx = idx.clone()
        idx[5::7, -1] = idx[5::7, 0]                               # a class twice
        idx[3::11] = -1                                            # nothing listed
        idx[2::5, k // 2] = c                                      # padding
        logits[1::2] += 30.0                                       # neighbouring rows differ: a stale maximum would show
        mean = float(mask.float().mean())
        stats, grad = sparse.distill_topk(logits, values, idx, mask, mean, temperature=2.0)
        _check(stats, grad, _distillation(logits, values, idx, mask, mean, 2.0))
        assert bool((grad[mask == 0] == 0).all()) and bool((stats[mask == 0] == 0).all())
        assert bool((grad[3::11] == 0).all()) and bool((stats[3::11] == 0).all())
