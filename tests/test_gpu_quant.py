"""The product that gathers 8-bit rows against float64 sums of the same values.

Tolerance: a row of m entries is a sum of m products a_e s q in some fixed order; with u = 2^-24 the weight a_e s is
rounded once, every fused multiply-add and every addition of two partial sums once, so the sum is off by at most
(m + 8) u of the sum of magnitudes."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def _matrix(n_rows, n_cols, lengths, seed):
    """CSR with the given row lengths; columns may repeat inside a row (every entry counts)."""
    import torch
    from gcn_amd import sparse
    rng = np.random.default_rng(seed)
    ip = np.zeros(n_rows + 1, dtype=np.int64)
    ip[1:] = np.cumsum(lengths)
    ix = rng.integers(0, n_cols, int(ip[-1])).astype(np.int32)
    v = rng.standard_normal(int(ip[-1])).astype(np.float32)
    return sparse.DeviceCSR(n_rows, n_cols, torch.as_tensor(ip).cuda(), torch.as_tensor(ix).cuda(), torch.as_tensor(v).cuda())


def _rows(n, f, seed, pitch=None):
    import torch
    from gcn_amd import sparse
    gen = torch.Generator().manual_seed(seed)
    pitch = sparse.QuantRows.pitch(f) if pitch is None else pitch
    data = torch.zeros((n, pitch), dtype=torch.uint8)
    bits = torch.randint(0, 256, (n, f), generator=gen).to(torch.uint8)
    bits[(bits & 127) == 127] = 0                                  # every value but the two NaN codes
    data[:, :f] = bits
    return sparse.QuantRows(n, f, data.cuda(), torch.rand(n, generator=gen).cuda() + 0.01)


def _dense(q):
    import torch
    return q.data[:, :q.f].contiguous().view(torch.float8_e4m3fn).double() * q.scales.double()[:, None]


def _check(a, q, out, relu=False):
    import torch
    b = _dense(q)
    row = torch.repeat_interleave(torch.arange(a.n_rows, device='cuda'), a.indptr[1:] - a.indptr[:-1])
    terms = a.values.double()[:, None] * b[a.indices.long()]
    want = torch.zeros((a.n_rows, q.f), dtype=torch.float64, device='cuda').index_add_(0, row, terms)
    size = torch.zeros((a.n_rows, q.f), dtype=torch.float64, device='cuda').index_add_(0, row, terms.abs())
    if relu:
        want = want.clamp(min=0)
    m = (a.indptr[1:] - a.indptr[:-1]).double()[:, None]
    assert bool(((out.double() - want).abs() <= (m + 8) * U * size).all())


FS = [1, 3, 15, 16, 17, 31, 32, 33, 50, 64, 65, 100, 127, 128, 129, 200, 255, 256, 257, 500, 512, 513, 1000, 1024, 1025, 2100]


@pytest.mark.parametrize('f', FS)
def test_product_at_every_width(f):
    """Rows of 0, 1, 2 ... 70 entries, around multiples of 64, long ones past the split, and 37 x 91 in shape."""
    from gcn_amd import sparse
    import torch
    lengths = [0, 1, 2, 3, 4, 5, 7, 8, 9, 15, 16, 17, 31, 32, 33, 63, 64, 65, 70, 127, 128, 129, 0, 0, 200, 255, 256, 257, 1023,
               1024, 1025, 3000, 2049, 1, 0, 6, 0]
    a = _matrix(len(lengths), 91, lengths, f)
    q = _rows(91, f, f)
    for relu in (False, True):
        out = sparse.spmm_quant(a, q, relu=relu)
        _check(a, q, out, relu)
        assert torch.equal(out, sparse.spmm_quant(a, q, relu=relu))
    # a wider pitch, and an output inside a wider matrix whose other elements stay
    wide = _rows(91, f, f, pitch=(f + 15) // 16 * 16 + 48)
    for extra, start in ((7, 2), (8, 4)):
        room = torch.full((a.n_rows + 2, f + extra), 5.0, device='cuda')
        view = room[1:a.n_rows + 1, start:start + f]
        sparse.spmm_quant(a, wide, relu=True, out=view)
        assert torch.equal(view, out)
        rest = torch.ones_like(room, dtype=torch.bool)
        rest[1:a.n_rows + 1, start:start + f] = False
        assert bool((room[rest] == 5.0).all())


@pytest.mark.parametrize('f,scale', [(16, 12), (40, 13), (100, 13), (256, 12), (600, 11)])
def test_product_on_a_power_law_graph(f, scale):
    """R-MAT: strips of many rows, hubs in chunks."""
    from gcn_amd import sparse
    import torch
    n = 1 << scale
    ip, ix = sparse.rmat_csr(scale, 16, self_loops=True)
    a = sparse.DeviceCSR(n, n, ip, ix, torch.rand(ix.numel(), generator=torch.Generator('cuda').manual_seed(1), device='cuda'))
    _check(a, _rows(n, f, 3), sparse.spmm_quant(a, _rows(n, f, 3)))


def test_rows_that_are_not_finite_reach_only_their_neighbours():
    import torch
    from gcn_amd import sparse
    a = _matrix(40, 30, [5] * 40, 8)
    q = _rows(30, 70, 9)
    clean = sparse.spmm_quant(a, q)
    q.scales[7] = float('nan')
    q.data[11, 3] = 0x7f                                            # one NaN element
    out = sparse.spmm_quant(a, q)
    cols = a.indices.view(40, 5)
    hit7, hit11 = (cols == 7).any(1), (cols == 11).any(1)
    assert bool(torch.isnan(out[hit7]).all()) and bool(torch.isnan(out[hit11, 3]).all())
    assert torch.equal(out[~hit7 & ~hit11], clean[~hit7 & ~hit11])
    keep = [c for c in range(70) if c != 3]
    assert torch.equal(out[~hit7][:, keep], clean[~hit7][:, keep])


def test_empty_matrices_and_one_entry():
    import torch
    from gcn_amd import sparse
    q = _rows(6, 20, 1)
    out = sparse.spmm_quant(_matrix(5, 6, [0] * 5, 1), q)
    assert out.shape == (5, 20) and bool((out == 0).all())
    assert sparse.spmm_quant(_matrix(0, 6, [], 1), q).shape == (0, 20)
    a = _matrix(1, 6, [1], 1)
    _check(a, q, sparse.spmm_quant(a, q))


@pytest.mark.parametrize('f', [33, 130])
def test_joined_long_rows_leave_the_columns_behind_them(f):
    """Rows longer than the split, a width that is no multiple of 4, into a slice of a wider matrix with 16-byte aligned
    rows: the packed and the 8-bit product alike write their columns only."""
    import torch
    from gcn_amd import sparse
    a = _matrix(6, 500, [4000, 3, 2500, 0, 1100, 9], 3)
    b = torch.randn((500, f), device='cuda') * (torch.rand((500, f), device='cuda') < 0.5)
    packed, q = sparse.pack_rows(b), sparse.rms_norm(b, quant=True)[0]
    for product in (lambda out: sparse.spmm_packed(a, packed, out=out), lambda out: sparse.spmm_quant(a, q, out=out)):
        room = torch.full((6, f + 7 - (f + 7) % 4 + 4), 5.0, device='cuda')
        product(room[:, :f])
        assert bool((room[:, f:] == 5.0).all()) and torch.equal(room[:, :f], product(None))


def test_element_offsets_past_32_bits():
    """9 million rows of 512 bytes: a byte offset past 2^32 in the operand; the last rows are gathered."""
    import torch
    from gcn_amd import sparse
    n, f, m = 9000000, 500, 300
    data = torch.zeros((n, 512), dtype=torch.uint8, device='cuda')
    tail = _rows(m, f, 5)
    data[n - m:, :] = tail.data
    q = sparse.QuantRows(n, f, data, torch.ones(n, device='cuda'))
    q.scales[n - m:] = tail.scales
    small = _matrix(50, m, [9] * 50, 4)
    a = sparse.DeviceCSR(50, n, small.indptr, small.indices + (n - m), small.values)
    assert torch.equal(sparse.spmm_quant(a, q), sparse.spmm_quant(small, tail))


def test_streams_and_two_graphs_that_are_replayed_together():
    """Each call has a workspace of its own: two recorded products of one plan replay on two streams at a time."""
    import torch
    from gcn_amd import sparse
    a = _matrix(60, 200, [3000] * 20 + [10] * 40, 2)
    qs = [_rows(200, 100, s) for s in (1, 2)]
    want = [sparse.spmm_quant(a, q) for q in qs]
    graphs, outs = [], []
    for q in qs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(sparse.spmm_quant(a, q))
        graphs.append(g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        eager = sparse.spmm_quant(a, qs[0])
        assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1]) and torch.equal(eager, want[0])


def test_norm_then_product_is_the_product_of_the_rows_it_stands_for():
    import torch
    from gcn_amd import sparse
    n, f = 500, 72
    a = _matrix(n, n, [7] * n, 5)
    q, _, _ = sparse.rms_norm(torch.randn((n, f), device='cuda'), torch.rand(f, device='cuda'), quant=True)
    _check(a, q, sparse.spmm_quant(a, q))


@pytest.mark.parametrize('f', [1, 3, 16, 50, 129, 1025])
def test_dense_form(f):
    """scale times value, one rounding: the same bits as torch's product of the same float32 numbers."""
    import torch
    from gcn_amd import sparse
    q = _rows(37, f, f)
    want = q.data[:, :f].contiguous().view(torch.float8_e4m3fn).float() * q.scales[:, None]
    assert torch.equal(q.dense(), want)
    room = torch.full((39, f + 5), 2.0, device='cuda')
    q.dense(out=room[1:38, 3:3 + f])
    assert torch.equal(room[1:38, 3:3 + f], want) and float(room.sum()) == pytest.approx(
        float(want.double().sum()) + 2.0 * (room.numel() - want.numel()), rel=1e-4, abs=1.0)
    assert sparse.QuantRows.empty(0, f, 'cuda').dense().shape == (0, f)
    assert torch.equal(q.rows(5, 9).dense(), want[5:9])


def test_refusals():
    import torch
    from gcn_amd import sparse
    a = _matrix(4, 6, [2] * 4, 1)
    q = _rows(6, 20, 1)
    for call in (lambda: sparse.spmm_quant(a, q.data), lambda: sparse.spmm_quant(a, q.rows(0, 5)),
                 lambda: sparse.spmm_quant(a, q, out=torch.empty((4, 19), device='cuda')),
                 lambda: sparse.spmm_quant(a, q, out=torch.empty((4, 20), dtype=torch.float64, device='cuda')),
                 lambda: sparse.spmm_quant(a, q, out=torch.empty((4, 20)))):
        with pytest.raises(ValueError):
            call()


@pytest.mark.parametrize('f', [7, 40, 70, 256, 600])
def test_relu_keeps_what_is_not_a_number(f):
    """A row of B that stands for NaN as a whole makes its neighbours NaN under the ReLU too, rows summed in chunks and
    their join among them; the others keep their bits."""
    import torch
    from gcn_amd import sparse
    lengths = [5] * 40 + [3000, 1100, 2048]
    a = _matrix(len(lengths), 300, lengths, 8)
    a.indices[a.indices == 7] = 8                                   # row 7 is met by three rows only
    a.indices[2], a.indices[200 + 2900], a.indices[200 + 3000] = 7, 7, 7
    assert a.plan.n_chunks > 0
    q = _rows(300, f, 9)
    clean = sparse.spmm_quant(a, q, relu=True)
    q.scales[7] = float('nan')
    out = sparse.spmm_quant(a, q, relu=True)
    hit = torch.zeros(a.n_rows, dtype=torch.bool, device='cuda')
    hit[[0, 40, 41]] = True
    assert bool(torch.isnan(out[hit]).all()) and torch.equal(out[~hit], clean[~hit])


def test_quant_dot_with_relu_shows_a_row_that_is_not_finite():
    import torch
    from gcn_amd import layers
    n = 60
    a = _matrix(n, n, [4] * n, 11)
    x = torch.randn((n, 24), device='cuda')
    x[13, 5] = float('inf')
    out = layers.quant_dot(a, x, fuse_relu=True)
    hit = (a.indices.view(n, 4) == 13).any(1)
    assert bool(hit.any()) and bool(torch.isnan(out[hit]).all()) and bool(torch.isfinite(out[~hit]).all())
