"""A dense layer's product with bias, activation and residual in its store, and its backward pass, against float64.

Tolerances, u = 2^-24: a sum of k products in any order is off by at most k u of the sum S of their magnitudes (k + 64 with
the joins of a cut product), the bias adds one rounding: E = (k + 66) u S.  The activations change by at most 1.13 times
their argument's error; their own arithmetic is off by (12 + z^2) u of the value (the exponent of e^(-z^2/2) has z^2 / 2
to round).  The slopes are off by at most (24 + 2 |z|) u (1 - s of the sigmoid carries u, times z)."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
ACTS = [None, 'relu', 'gelu', 'silu']


def _act(z, act):
    import torch
    if act == 'relu':
        return z.clamp(min=0), (z > 0).double()
    if act == 'gelu':
        cdf = 0.5 * torch.special.erfc(-z / np.sqrt(2.0))
        return z * cdf, cdf + z * torch.exp(-z * z / 2) / np.sqrt(2 * np.pi)
    if act == 'silu':
        s = torch.sigmoid(z)
        return z * s, s * (1 + z * (1 - s))
    return z, torch.ones_like(z)


def _inputs(m, n, k, seed=0, trans_b=False):
    import torch
    gen = torch.Generator().manual_seed(m * 7 + n * 3 + k + seed)
    shapes = ((m, k), (n, k) if trans_b else (k, n), (n,), (m, n), (m, n))
    a, b, bias, r, g = (torch.randn(s, generator=gen).cuda() for s in shapes)
    return a, b / max(k, 1) ** 0.5, bias, r, g


def _check(a, b, trans_b, bias, act, r, out, pre=None):
    bd = b.double().t().contiguous() if trans_b else b.double()
    k = a.shape[1]
    size = a.double().abs() @ bd.abs() + (0 if bias is None else bias.double().abs())
    z = a.double() @ bd + (0 if bias is None else bias.double())
    err = (k + 66) * U * size
    if pre is not None:
        assert bool(((pre.double() - z).abs() <= err).all())
    v, _ = _act(z, act)
    want = v + (0 if r is None else r.double())
    tol = 1.13 * err + (12 + z * z) * U * v.abs() + 2 * U * want.abs()
    assert bool(((out.double() - want).abs() <= tol).all())


SHAPES = [(1, 1, 1), (1, 7, 5), (3, 16, 1433), (2708, 16, 1433), (1, 300, 700), (130, 33, 17), (127, 65, 64), (128, 128, 32),
          (129, 129, 33), (256, 256, 256), (300, 256, 96), (1000, 128, 500), (515, 47, 256), (64, 3, 16), (77, 64, 300),
          (2, 500, 2000), (40, 130, 0), (1025, 384, 160), (31, 1000, 12)]


@pytest.mark.parametrize('m,n,k', SHAPES)
def test_forward_with_every_part(m, n, k):
    import torch
    from gcn_amd import sparse
    for trans_b in (False, True):
        a, b, bias, r, _ = _inputs(m, n, k, trans_b=trans_b)
        for act in ACTS:
            for bb, rr in ((bias, r), (None, None), (bias, None), (None, r)):
                out, pre = sparse.gemm_epilogue(a, b, trans_b=trans_b, bias=bb, act=act, residual=rr, want_pre=True)
                _check(a, b, trans_b, bb, act, rr, out, pre)
                assert torch.equal(out, sparse.gemm_epilogue(a, b, trans_b=trans_b, bias=bb, act=act, residual=rr))


def test_plain_product_bits_do_not_change_with_an_empty_epilogue():
    import torch
    from gcn_amd import sparse
    for m, n, k in ((1000, 256, 96), (777, 48, 40), (300, 130, 33)):
        a, b, _, _, _ = _inputs(m, n, k)
        assert torch.equal(sparse.gemm_epilogue(a, b), sparse.gemm(a, b)) or k >= 128


@pytest.mark.parametrize('m,n,k', [(130, 33, 17), (2708, 16, 300), (300, 256, 96), (517, 200, 64), (65, 500, 640)])
def test_views_aliases_and_untouched_memory(m, n, k):
    import torch
    from gcn_amd import sparse
    a, b, bias, r, _ = _inputs(m, n, k)
    ref = sparse.gemm_epilogue(a, b, bias=bias, act='gelu', residual=r)
    wide_a = torch.randn((m, k + 5), device='cuda')
    wide_a[:, 3:3 + k] = a
    wide_r = torch.randn((m, n + 3), device='cuda')
    wide_r[:, 1:1 + n] = r
    room = torch.full((m + 2, n + 9), 3.0, device='cuda')
    view = room[1:m + 1, 4:4 + n]
    sparse.gemm_epilogue(wide_a[:, 3:3 + k], b, bias=bias, act='gelu', residual=wide_r[:, 1:1 + n], out=view)
    assert bool(((view - ref).abs() <= 4 * (k + 80) * U * (1 + ref.abs().max())).all())
    rest = torch.ones_like(room, dtype=torch.bool)
    rest[1:m + 1, 4:4 + n] = False
    assert bool((room[rest] == 3.0).all())
    own = r.clone()
    assert sparse.gemm_epilogue(a, b, bias=bias, act='gelu', residual=own, out=own) is own and torch.equal(own, ref)


@pytest.mark.parametrize('m,n', [(1, 1), (1, 300), (7, 3), (2708, 16), (130, 17), (1000, 64), (33, 100), (515, 256),
                                 (77, 257), (64, 500), (9, 1000), (100001, 8), (20000, 130), (4, 2049)])
def test_gradient_of_activation_and_bias(m, n):
    import torch
    from gcn_amd import sparse
    _, _, _, pre, g = _inputs(m, n, 1, seed=4)
    pre = pre * 3
    for act in ACTS:
        dz, dbias = sparse.act_grad(g, pre, act)
        _, slope = _act(pre.double(), act)
        want = g.double() * slope
        err = g.double().abs() * (24 + 2 * pre.double().abs()) * U
        if act is None:
            assert dz is g
        assert bool(((dz.double() - want).abs() <= err + 2 * U * want.abs()).all())
        # rows in serial runs of at most tile length, workgroups in 16 serial runs: (m + 8) u of the magnitudes at most
        tol = err.sum(0) + min(m + 8, 8192) * U * want.abs().sum(0)
        assert bool(((dbias.double() - want.sum(0)).abs() <= tol).all())
        again = sparse.act_grad(g, pre, act)
        assert torch.equal(again[1], dbias) and torch.equal(again[0], dz)
        only, none = sparse.act_grad(g, pre, act, want_bias=False)
        assert none is None and torch.equal(only, dz)


def test_slopes_and_values_over_the_whole_range():
    """Every activation at 10^5 points in [-30, 30], at zero, and at the ends of float32 (a product with the 1 x 1 identity)."""
    import torch
    from gcn_amd import sparse
    z = torch.linspace(-30, 30, 100001, device='cuda')[:, None]
    one = torch.ones((1, 1), device='cuda')
    for act in ACTS[1:]:
        v, s = _act(z.double(), act)
        out = sparse.gemm_epilogue(z, one, act=act)
        assert bool(((out.double() - v).abs() <= (12 + z.double() ** 2) * U * v.abs() + 1e-37).all())
        dz, _ = sparse.act_grad(torch.ones_like(z), z, act)
        assert bool(((dz.double() - s).abs() <= (24 + 2 * z.double().abs()) * U).all())
        ends = torch.tensor([[0.0], [3e38], [-3e38], [float('inf')], [float('nan')]], device='cuda')
        out = sparse.gemm_epilogue(ends, one, act=act).flatten().tolist()
        assert out[0] == 0 and out[1] == float(ends[1]) and out[2] == 0 and out[3] == float('inf') and np.isnan(out[4])
        dz = sparse.act_grad(torch.ones((3, 1), device='cuda'), ends[:3], act)[0].flatten().tolist()
        assert dz[1] == 1.0 and dz[2] == 0.0 and dz[0] == (0.0 if act == 'relu' else 0.5)


def test_gradients_of_a_layer_against_differences():
    """All five gradients of sum(v * layer) by central differences in float64, step 1e-6: their error is about 1e-9; the
    float32 gradients are sums of at most 9 terms of magnitude below 10."""
    import torch
    from gcn_amd import sparse
    m, n, k = 5, 7, 9
    a, b, bias, r, v = _inputs(m, n, k, seed=9)
    for act in ACTS[2:]:
        out, pre = sparse.gemm_epilogue(a, b, bias=bias, act=act, residual=r, want_pre=True)
        dz, dbias = sparse.act_grad(v, pre, act)
        grads = [sparse.gemm(dz, b, trans_b=True), sparse.gemm_tn(a, dz), dbias, v]
        ins = [t.double() for t in (a, b, bias, r)]

        def value(parts):
            return float(((_act(parts[0] @ parts[1] + parts[2], act)[0] + parts[3]) * v.double()).sum())
        for which, grad in enumerate(grads):
            for at in (0, grad.numel() // 2, grad.numel() - 1):
                e = torch.zeros_like(ins[which]).flatten()
                e[at] = 1e-6
                up = [t + e.view_as(t) if i == which else t for i, t in enumerate(ins)]
                down = [t - e.view_as(t) if i == which else t for i, t in enumerate(ins)]
                assert abs((value(up) - value(down)) / 2e-6 - float(grad.flatten()[at])) <= 1e-5


def test_replayed_graph_of_a_step():
    import torch
    from gcn_amd import sparse
    a, b, bias, r, g = _inputs(700, 48, 640)

    def step():
        out, pre = sparse.gemm_epilogue(a, b, bias=bias, act='silu', residual=r, want_pre=True)
        dz, dbias = sparse.act_grad(g, pre, 'silu')
        return out, dbias, sparse.gemm(dz, b, trans_b=True), sparse.gemm_tn(a, dz)
    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for _ in range(3):
        a.copy_(torch.randn_like(a))
        graph.replay()
        eager = step()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(outs, eager))


def test_empty_and_refusals():
    import torch
    from gcn_amd import sparse
    a, b, bias, r, g = _inputs(6, 5, 4)
    assert sparse.gemm_epilogue(a[:0], b, bias=bias).shape == (0, 5)
    dz, db = sparse.act_grad(g[:0], r[:0], 'relu')
    assert dz.shape == (0, 5) and bool((db == 0).all())
    for call in (lambda: sparse.gemm_epilogue(a, b, act='tanh'), lambda: sparse.gemm_epilogue(a, b[:3]),
                 lambda: sparse.gemm_epilogue(a, b, bias=bias[:4]), lambda: sparse.gemm_epilogue(a, b, residual=r[:5]),
                 lambda: sparse.gemm_epilogue(a, b, out=r[:5]), lambda: sparse.gemm_epilogue(a, b, bias=bias.cpu()),
                 lambda: sparse.gemm_epilogue(a.cpu(), b), lambda: sparse.act_grad(g, r[:5], 'relu'),
                 lambda: sparse.act_grad(g, r, 'softplus'), lambda: sparse.act_grad(g, None, 'relu'),
                 lambda: sparse.act_grad(g.cpu(), r, 'relu')):
        with pytest.raises(ValueError):
            call()


@pytest.mark.parametrize('trans_b', [False, True])
@pytest.mark.parametrize('m,n,k', [(300, 17, 96), (300, 47, 70), (257, 134, 64), (300, 200, 96), (1500, 16, 1433), (150000, 130, 64),
                                   (150001, 200, 65), (129, 3, 33), (129, 1, 64), (5000, 333, 300)])
def test_operands_inside_matrices_of_nan(m, n, k, trans_b):
    """What lies around the operands does not reach the result, and the result has the bits of the packed operands'."""
    import torch
    from gcn_amd import sparse
    a = torch.randn((m, k), device='cuda')
    b = torch.randn((n, k) if trans_b else (k, n), device='cuda')
    room_a = torch.full((m + 2, k + 5), float('nan'), device='cuda')
    room_b = torch.full((b.shape[0] + 2, b.shape[1] + 7), float('nan'), device='cuda')
    room_a[1:m + 1, 2:2 + k] = a
    room_b[1:b.shape[0] + 1, 3:3 + b.shape[1]] = b
    va, vb = room_a[1:m + 1, 2:2 + k], room_b[1:b.shape[0] + 1, 3:3 + b.shape[1]]
    for f in (lambda x, y: sparse.gemm_epilogue(x, y, trans_b=trans_b, act='silu'), lambda x, y: sparse.gemm(x, y, trans_b=trans_b),
              lambda x, y: sparse.gemm(x, y, trans_b=trans_b, relu=True)):
        assert torch.equal(f(va, vb), f(a, b))


def test_a_result_over_an_operand_is_refused():
    import torch
    from gcn_amd import sparse
    a, b = torch.randn((64, 64), device='cuda'), torch.randn((64, 64), device='cuda')
    for out in (a, b):
        with pytest.raises(ValueError):
            sparse.gemm_epilogue(a, b, out=out)


@pytest.mark.parametrize('n,k', [(260, 40), (256, 64), (250, 40), (240, 8)])
def test_element_offsets_past_32_bits(n, k):
    """Nine million rows: 2^31 elements and more in the result, the residual and the pre-activation; sampled rows."""
    import torch
    from gcn_amd import sparse
    m = 9000001
    if torch.cuda.mem_get_info()[0] < 60 << 30:
        pytest.skip('needs 60 GB of free device memory')
    gen = torch.Generator('cuda').manual_seed(n + k)
    a = torch.empty((m, k), device='cuda').normal_(generator=gen)
    b = torch.empty((k, n), device='cuda').normal_(generator=gen) / k ** 0.5
    bias = torch.empty(n, device='cuda').normal_(generator=gen)
    r = torch.empty((m, n), device='cuda').normal_(generator=gen)
    out, pre = sparse.gemm_epilogue(a, b, bias=bias, act='gelu', residual=r, want_pre=True)
    dz, db = sparse.act_grad(r, pre, 'gelu')
    for lo in (0, (1 << 31) // n - 20, (1 << 30) // n - 20, m - 40):
        rows = slice(lo, lo + 40)
        _check(a[rows], b, False, bias, 'gelu', r[rows], out[rows], pre[rows])
        _, s = _act(pre[rows].double(), 'gelu')
        want = r[rows].double() * s
        assert bool(((dz[rows].double() - want).abs() <= (26 + 2 * pre[rows].double().abs()) * U * r[rows].double().abs()).all())
    total = torch.zeros(n, dtype=torch.float64, device='cuda')
    size = torch.zeros(n, dtype=torch.float64, device='cuda')
    for lo in range(0, m, 1 << 20):
        total += dz[lo:lo + (1 << 20)].double().sum(0)
        size += dz[lo:lo + (1 << 20)].double().abs().sum(0)
    # at most m / 2048 rows of a group and a tree over the groups and workgroups: (4395 + 64) u of the magnitudes
    assert bool(((db.double() - total).abs() <= 4500 * U * size).all())
