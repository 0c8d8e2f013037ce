"""The row norm (with the residual's addition, in float32 and as 8-bit rows) and its gradients against the formulas
in float64.

Tolerances, with u = 2^-24 the relative rounding of float32.  A sum of f products in a tree of depth log2(f) plus the
serial part a lane holds (at most 32 terms) is off by at most (32 + log2 f + 1) u of the sum of magnitudes; rsqrt by
2 u; each product by u.  So y is within 64 u of itself, and a gradient within 128 u of the magnitudes it is made of.
An 8-bit value is the true quotient rounded to nearest: off by half a step, 2^-4 of itself, or 2^-10 near zero (half
the smallest e4m3 value), both plus 64 u for the quotient."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
SHAPES = [(1, 1), (1, 7), (3, 2), (5, 3), (2708, 16), (130, 17), (77, 31), (65, 33), (9, 63), (1000, 64), (33, 100),
          (19, 127), (5, 129), (515, 256), (7, 257), (64, 500), (3, 511), (6, 1000), (11, 1433), (4, 2047), (3, 2049),
          (5, 3703), (2, 4097), (2, 8191), (2, 8193), (1, 16383), (2, 20001), (1, 32768),
          (5000, 16387)]


def _inputs(n, f, seed=0):
    import torch
    gen = torch.Generator().manual_seed(1000 * n + f + seed)
    return [torch.randn(s, generator=gen).cuda() for s in ((n, f), (n, f), (f,), (n, f), (n, f))]


def _reference(x, r, w, eps):
    h = x.double() + (0 if r is None else r.double())
    inv = (h.square().mean(1) + eps).rsqrt()
    y = h * inv[:, None] * (1 if w is None else w.double())
    return y, h, inv


def _bytes(q):
    import torch
    return q.data[:, :q.f].contiguous().view(torch.float8_e4m3fn).double()


def _check_rows(q, y, x):
    """q stands for y: the scale, every byte within half a step, and the padding zero."""
    import torch
    scale = (y.abs().amax(1) / 448.0).clamp(min=2.0 ** -120)
    assert bool(((q.scales.double() - scale).abs() <= 70 * U * scale).all())
    want = y / q.scales.double()[:, None]
    # half a step of a value with three mantissa bits is at most 2^-4 of it
    assert bool(((_bytes(q) - want).abs() <= want.abs() * (2.0 ** -4 + 80 * U) + 2.0 ** -10).all())
    top = (q.f + 15) // 16 * 16
    assert bool((q.data[:, q.f:top] == 0).all())


@pytest.mark.parametrize('n,f', SHAPES)
def test_norm_against_the_formula(n, f):
    import torch
    from gcn_amd import sparse
    x, r, w, _, _ = _inputs(n, f)
    for res in (None, r):
        for weight in (None, w):
            y, h, inv = sparse.rms_norm(x, weight, residual=res, eps=1e-5)
            ry, rh, rinv = _reference(x, res, weight, 1e-5)
            if res is None:
                assert h is x
            else:
                assert torch.equal(h, x + res)
                rh = h.double()                       # the sum itself is one float32 addition; the rest goes by it
                ry, rh, rinv = _reference(h, None, weight, 1e-5)
            assert bool(((inv.double() - rinv).abs() <= 64 * U * rinv).all())
            assert bool(((y.double() - ry).abs() <= 70 * U * ry.abs()).all())
            q, h2, inv2 = sparse.rms_norm(x, weight, residual=res, eps=1e-5, quant=True)
            assert torch.equal(h2, h) and torch.equal(inv2, inv)
            _check_rows(q, ry, x)


@pytest.mark.parametrize('n,f', SHAPES)
def test_gradients_against_the_formula(n, f):
    import torch
    from gcn_amd import sparse
    h, dy, w, dh, _ = _inputs(n, f, 1)
    _, _, inv = sparse.rms_norm(h, w)
    for weight in (None, w):
        for up in (None, dh):
            dx, dw = sparse.rms_norm_grad(dy, h, weight, inv, grad_h=up)
            g = dy.double() * (1 if weight is None else weight.double())
            i = inv.double()[:, None]
            along = (g * h.double()).sum(1, keepdim=True) / f
            rdx = i * (g - h.double() * i * i * along) + (0 if up is None else up.double())
            size = i * (g.abs() + h.double().abs() * i * i * (g * h.double()).abs().sum(1, keepdim=True) / f) \
                + (0 if up is None else up.double().abs())
            assert bool(((dx.double() - rdx).abs() <= 128 * U * size).all())
            terms = dy.double() * h.double() * i
            # n terms, added serially inside a workgroup and over workgroups: (n + 8) u of the magnitudes at most
            assert bool(((dw.double() - terms.sum(0)).abs() <= min(n + 8, 4096) * U * terms.abs().sum(0)).all())
            again = sparse.rms_norm_grad(dy, h, weight, inv, grad_h=up)
            assert torch.equal(again[0], dx) and torch.equal(again[1], dw)
    only, none = sparse.rms_norm_grad(dy, h, w, inv, want_weight=False)
    assert none is None and torch.equal(only, sparse.rms_norm_grad(dy, h, w, inv)[0])


def test_gradient_against_differences():
    """Central differences of sum(y * v) in float64 on the formula, step 1e-5: their own error is about 1e-9."""
    import torch
    from gcn_amd import sparse
    x, v, w, _, _ = _inputs(3, 10, 2)
    _, _, inv = sparse.rms_norm(x, w, eps=1e-3)
    dx, dw = sparse.rms_norm_grad(v, x, w, inv)

    def value(xx, ww):
        return float((_reference(xx, None, ww, 1e-3)[0] * v.double()).sum())
    for i, j in ((0, 0), (1, 9), (2, 4)):
        e = torch.zeros((3, 10), dtype=torch.float64, device='cuda')
        e[i, j] = 1e-5
        slope = (value(x.double() + e, w) - value(x.double() - e, w)) / 2e-5
        assert abs(slope - float(dx[i, j])) <= 1e-5
        e = torch.zeros(10, dtype=torch.float64, device='cuda')
        e[j] = 1e-5
        slope = (value(x, w.double() + e) - value(x, w.double() - e)) / 2e-5
        assert abs(slope - float(dw[j])) <= 1e-5


@pytest.mark.parametrize('f', [16, 37, 256, 2500, 17003])
def test_views_outputs_and_aliases(f):
    """Rows inside a wider matrix at an odd offset, outputs given by the caller, h written over x or the residual,
    the memory between and behind the rows untouched."""
    import torch
    from gcn_amd import sparse
    n = 21
    wide = torch.randn((n, 2 * f + 9), device='cuda')
    x, r = wide[:, 1:1 + f], wide[:, f + 4:2 * f + 4]
    w = torch.randn(f, device='cuda')
    y, h, inv = sparse.rms_norm(x, w, residual=r)
    room = torch.full((n + 2, f + 5), 7.0, device='cuda')
    y2, h2, _ = sparse.rms_norm(x.contiguous(), w, residual=r.contiguous(), out=room[1:n + 1, 2:2 + f])
    assert torch.equal(y2, y) and torch.equal(h2, h)
    untouched = torch.ones_like(room, dtype=torch.bool)
    untouched[1:n + 1, 2:2 + f] = False
    assert bool((room[untouched] == 7.0).all())
    for into in (0, 1):
        both = [x.clone().contiguous(), r.clone().contiguous()]
        y3, h3, inv3 = sparse.rms_norm(both[0], w, residual=both[1], sum_out=both[into])
        assert h3 is both[into] and torch.equal(h3, h) and torch.equal(y3, y) and torch.equal(inv3, inv)
    # y over x
    one = x.clone().contiguous()
    y4, _, _ = sparse.rms_norm(one, w, out=one)
    assert torch.equal(y4, sparse.rms_norm(x, w)[0])
    # 8-bit rows into the middle of a larger block
    pitch = sparse.QuantRows.pitch(f) + 32
    block = torch.full((n + 2, pitch), 9, dtype=torch.uint8, device='cuda')
    scales = torch.full((n + 2,), 5.0, device='cuda')
    q = sparse.QuantRows(n + 2, f, block, scales)
    sparse.rms_norm(x, w, residual=r, quant=True, out=q.rows(1, n + 1))
    ref = sparse.rms_norm(x, w, residual=r, quant=True)[0]
    top = (f + 15) // 16 * 16
    assert torch.equal(block[1:n + 1, :top], ref.data[:, :top]) and torch.equal(scales[1:n + 1], ref.scales)
    assert bool((block[0] == 9).all()) and bool((block[n + 1] == 9).all()) and bool((block[:, top:] == 9).all())
    assert float(scales[0]) == 5.0 and float(scales[n + 1]) == 5.0


@pytest.mark.parametrize('f', [5, 64, 300, 5000])
def test_rows_of_zeros_extremes_and_non_finite_values(f):
    import torch
    from gcn_amd import sparse
    x = torch.randn((7, f), device='cuda')
    x[0] = 0.0
    x[1] = 1e-30
    x[2] *= 1e15
    x[3, f // 2] = float('nan')
    x[4, 0] = float('inf')
    x[5] *= 1e-12
    y, _, inv = sparse.rms_norm(x, eps=0.0 if f == 5 else 1e-6)
    q, _, _ = sparse.rms_norm(x, eps=1e-6, quant=True)
    ry = _reference(x, None, None, 1e-6)[0]
    fine = [0, 1, 2, 5, 6]
    if f != 5:
        assert bool(((y.double() - ry)[fine].abs() <= 70 * U * ry[fine].abs()).all())
        assert bool((y[0] == 0).all())
    assert bool(torch.isnan(y[3]).all()) and bool(torch.isnan(y[4, 0]))
    # a zero row: the smallest scale, every byte zero; rows that are not finite: NaN as a whole
    assert float(q.scales[0]) == 2.0 ** -120 and bool((q.data[0, :f] == 0).all())
    assert bool(torch.isnan(q.scales[3:5]).all()) and bool(torch.isfinite(q.scales[fine]).all())
    sub = sparse.rms_norm(x[fine], eps=1e-6, quant=True)[0]
    _check_rows(sub, ry[fine], x)


def test_empty_matrix_and_one_past_the_last_row():
    import torch
    from gcn_amd import sparse
    x = torch.empty((0, 12), device='cuda')
    y, h, inv = sparse.rms_norm(x, torch.ones(12, device='cuda'))
    assert y.shape == (0, 12) and inv.shape == (0,)
    assert sparse.rms_norm(x, quant=True)[0].n_rows == 0
    dx, dw = sparse.rms_norm_grad(y, h, None, inv)
    assert dx.shape == (0, 12) and bool((dw == 0).all())


def test_another_stream_and_a_graph():
    """The call goes to the current stream; recorded with its gradient and replayed on new inputs it gives the eager
    results, with eager work in between."""
    import torch
    from gcn_amd import sparse
    n, f = 3000, 100
    x, r, w, dy, _ = _inputs(n, f, 5)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y, h, inv = sparse.rms_norm(x, w, residual=r)
        dx, dw = sparse.rms_norm_grad(dy, h, w, inv)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        gy, gh, ginv = sparse.rms_norm(x, w, residual=r, quant=True)
        gdx, gdw = sparse.rms_norm_grad(dy, gh, w, ginv)
    for k in range(3):
        x.copy_(torch.randn_like(x))
        graph.replay()
        q, h, inv = sparse.rms_norm(x, w, residual=r, quant=True)
        dx, dw = sparse.rms_norm_grad(dy, h, w, inv)
        torch.cuda.synchronize()
        assert torch.equal(gy.data[:, :f], q.data[:, :f]) and torch.equal(gy.scales, q.scales)
        assert torch.equal(gdx, dx) and torch.equal(gdw, dw)


def test_element_offsets_past_32_bits():
    """2.2 million rows of 1000 columns: offsets past 2^31 elements; the last rows against the formula, forward (float32 and
    8 bits) and backward."""
    import torch
    from gcn_amd import sparse
    n, f, m = 2200000, 1000, 20
    if torch.cuda.mem_get_info()[0] < 60 << 30:
        pytest.skip('needs 60 GB of free device memory')
    x = torch.empty((n, f), device='cuda').normal_(generator=torch.Generator('cuda').manual_seed(1))
    w = torch.rand(f, device='cuda')
    y, h, inv = sparse.rms_norm(x, w)
    ry = _reference(x[-m:], None, w, 1e-6)[0]
    assert bool(((y[-m:].double() - ry).abs() <= 70 * U * ry.abs()).all())
    dx, _ = sparse.rms_norm_grad(y, h, w, inv)
    small, _ = sparse.rms_norm_grad(y[-m:], x[-m:], w, inv[-m:])
    assert torch.equal(dx[-m:], small)
    del y, dx
    q, _, _ = sparse.rms_norm(x, w, quant=True)
    _check_rows(q.rows(n - m, n), ry, x)


def test_refusals():
    import torch
    from gcn_amd import sparse
    x = torch.randn((4, 6), device='cuda')
    w = torch.ones(6, device='cuda')
    bad = [lambda: sparse.rms_norm(x, torch.ones(5, device='cuda')), lambda: sparse.rms_norm(x, w, residual=x[:3]),
           lambda: sparse.rms_norm(x.cpu(), w), lambda: sparse.rms_norm(x, w.cpu()), lambda: sparse.rms_norm(x[0], w),
           lambda: sparse.rms_norm(x, w, eps=-1.0), lambda: sparse.rms_norm(x, w, eps=float('nan')),
           lambda: sparse.rms_norm(x, w, sum_out=x), lambda: sparse.rms_norm(x, w, residual=x, out=x, sum_out=x), lambda: sparse.rms_norm(x, w, quant=True, out=x),
           lambda: sparse.rms_norm(x, w, out=x[:3]), lambda: sparse.rms_norm(torch.ones((2, 32769), device='cuda')),
           lambda: sparse.rms_norm(torch.ones((2, 0), device='cuda')),
           lambda: sparse.rms_norm_grad(x, x[:3], w, torch.ones(3, device='cuda')),
           lambda: sparse.rms_norm_grad(x, x, w, torch.ones(3, device='cuda')),
           lambda: sparse.rms_norm_grad(x, x, w, torch.ones(4, device='cuda'), grad_h=x[:, :3]),
           lambda: sparse.QuantRows(4, 6, torch.zeros((4, 15), dtype=torch.uint8, device='cuda'), torch.ones(4, device='cuda')),
           lambda: sparse.QuantRows(4, 6, torch.zeros((4, 24), dtype=torch.uint8, device='cuda'), torch.ones(4, device='cuda')),
           lambda: sparse.QuantRows(4, 6, torch.zeros((4, 16), dtype=torch.int8, device='cuda'), torch.ones(4, device='cuda')),
           lambda: sparse.QuantRows(4, 6, torch.zeros((4, 16), dtype=torch.uint8, device='cuda'), torch.ones(3, device='cuda')),
           lambda: sparse.QuantRows(4, 6, torch.zeros((5, 16), dtype=torch.uint8, device='cuda').flatten()[8:72].view(4, 16),
                                    torch.ones(4, device='cuda'))]
    for call in bad:
        with pytest.raises(ValueError):
            call()
    assert np.isfinite(sparse.rms_norm(x, w)[0].cpu().numpy()).all()


@pytest.mark.parametrize('f', [7, 64, 300, 1500, 17003])
def test_a_weight_that_is_not_finite_makes_whole_rows_nan(f):
    """The maximum of a row with a NaN in it is no number: the row's scale is NaN, as where the row itself is not finite."""
    import torch
    from gcn_amd import sparse
    x = torch.randn((9, f), device='cuda')
    x[4, f - 1] = 0.0                                              # 0 * inf is NaN as well
    for bad in (float('nan'), float('inf'), -float('inf')):
        for at in (0, f // 2, f - 1):
            w = torch.ones(f, device='cuda')
            w[at] = bad
            q = sparse.rms_norm(x, w, quant=True)[0]
            assert bool(torch.isnan(q.scales).all()) and bool(torch.isnan(q.dense()).all())


@pytest.mark.parametrize('n,f', [(4000, 16), (3000, 100), (2000, 256), (1500, 500), (700, 1433), (90, 5001), (40, 9000), (30, 20001)])
def test_bytes_are_the_quotients_by_the_scale(n, f):
    """Scale and bytes as they are defined, with no rounding more: the float32 output (the same y) divided by 448 and by the
    scale, IEEE division on the host, rounded to nearest even.  Equal bit for bit."""
    import torch
    from gcn_amd import sparse
    x, r, w, _, _ = _inputs(n, f, 7)
    q = sparse.rms_norm(x, w, residual=r, quant=True)[0]
    y = sparse.rms_norm(x, w, residual=r)[0].cpu()
    scale = (y.abs().amax(1) / 448.0).clamp(min=2.0 ** -120)
    assert torch.equal(q.scales.cpu(), scale)
    assert torch.equal(q.data[:, :f].cpu(), (y / scale[:, None]).to(torch.float8_e4m3fn).view(torch.uint8))
