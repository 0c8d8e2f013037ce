"""CPU: the argument checks of the row norm, the 8-bit product, the dense epilogue and the
distillation loss through the C ABI -- they return before any HIP call -- and what the
Python operators refuse on a host without a GPU."""
import ctypes

import pytest

BAD, WORKSPACE = 1, 4
P = 4096                       # a non-null address that no call dereferences


def _lib():
    from gcn_amd import _lib as lib
    return lib.load()


def test_quant_pitch():
    lib, out = _lib(), ctypes.c_int64()
    for f, want in ((1, 16), (16, 16), (17, 32), (33, 64), (65, 128), (128, 128), (129, 192), (256, 256), (500, 512),
                    (32768, 32768)):
        assert lib.gcn_quant_pitch(f, ctypes.byref(out)) == 0 and out.value == want
    for f in (0, -1, 32769):
        assert lib.gcn_quant_pitch(f, ctypes.byref(out)) == BAD
    assert lib.gcn_quant_pitch(4, None) == BAD


def _norm(n=4, f=6, x=P, ldx=6, r=None, ldr=0, eps=1e-6, h=None, ldh=6, inv=P, y=P, ldy=6, q=None, ldq=0, scales=None):
    return _lib().gcn_rms_norm_f32(n, f, x, ldx, r, ldr, None, eps, h, ldh, inv, y, ldy, q, ldq, scales, None)


def test_norm_refuses():
    assert _norm(n=0) == 0
    for bad in (dict(n=-1), dict(f=0), dict(f=32769, ldx=32769, ldy=32769), dict(n=(1 << 32) + 1), dict(ldx=5),
                dict(ldy=5), dict(r=P, ldr=5, h=P), dict(r=P, ldr=6, h=P, ldh=5), dict(r=P, ldr=6, h=None),
                dict(x=None), dict(inv=None), dict(y=None), dict(r=P, ldr=6, h=P), dict(q=P, ldq=16, scales=P), dict(eps=-1.0),
                dict(eps=float('nan')), dict(y=None, q=P, ldq=16, scales=None), dict(y=None, q=P, ldq=8, scales=P),
                dict(y=None, q=P, ldq=24, scales=P), dict(y=None, q=P + 8, ldq=16, scales=P)):
        assert _norm(**bad) == BAD, bad


def _norm_grad(n=4, f=6, dy=P, lddy=6, h=P, ldh=6, inv=P, dh=None, lddh=0, dx=P, lddx=6, dw=None, ws=None, nbytes=0):
    return _lib().gcn_rms_norm_grad_f32(n, f, dy, lddy, h, ldh, None, inv, dh, lddh, dx, lddx, dw, ws, nbytes, None)


def test_norm_gradient_refuses():
    assert _norm_grad(n=0) == 0 and _norm_grad(dx=None) == 0
    for bad in (dict(n=-1), dict(f=0), dict(lddy=5), dict(ldh=5), dict(dh=P, lddh=5), dict(lddx=5), dict(dy=None),
                dict(h=None), dict(inv=None)):
        assert _norm_grad(**bad) == BAD, bad
    need = ctypes.c_size_t()
    assert _lib().gcn_rms_norm_grad_workspace_bytes(4, 6, ctypes.byref(need)) == 0 and need.value >= 24
    for bad in (dict(ws=None, nbytes=need.value), dict(ws=P, nbytes=need.value - 1), dict(ws=P + 4, nbytes=need.value)):
        assert _norm_grad(dw=P, **bad) == WORKSPACE, bad
    assert _lib().gcn_rms_norm_grad_workspace_bytes(4, 0, ctypes.byref(need)) == BAD
    assert _lib().gcn_rms_norm_grad_workspace_bytes(4, 6, None) == BAD


def _distill(n=4, c=6, x=P, ldx=6, v=P, vt=0, ldv=3, i=P, ldi=3, k=3, mask=P, mean=0.5, temp=1.0, up=None, stats=P, d=P,
             ldd=6):
    return _lib().gcn_distill_topk_f32(n, c, x, ldx, v, vt, ldv, i, ldi, k, mask, mean, temp, up, stats, d, ldd, None)


def test_distillation_refuses():
    assert _distill(n=0) == 0 and _distill(stats=None, d=None) == 0
    for bad in (dict(n=-1), dict(c=0), dict(c=2 ** 31, ldx=2 ** 31, ldd=2 ** 31), dict(ldx=5), dict(ldd=5), dict(k=0),
                dict(k=257, ldv=257, ldi=257), dict(ldv=2), dict(ldi=2), dict(vt=3), dict(mean=0.0), dict(mean=float('nan')),
                dict(temp=0.0), dict(temp=-1.0), dict(temp=float('inf')), dict(temp=float('nan')), dict(x=None), dict(v=None),
                dict(i=None), dict(stats=P + 4)):
        assert _distill(**bad) == BAD, bad


def _dense(m=4, n=5, k=6, a=P, lda=6, b=P, ldb=5, tb=0, bias=P, act=1, r=P, ldr=5, pre=P, ldp=5, c=P, ldc=5, ws=None, nb=0):
    return _lib().gcn_gemm_epilogue_f32(m, n, k, a, lda, b, ldb, tb, bias, act, r, ldr, pre, ldp, c, ldc, ws, nb, None)


def test_dense_epilogue_refuses():
    assert _dense(m=0) == 0 and _dense(n=0, ldb=0) == 0
    for bad in (dict(m=-1), dict(n=-1), dict(k=-1), dict(lda=5), dict(ldb=4), dict(ldc=4), dict(ldr=4), dict(ldp=4),
                dict(tb=1, ldb=5), dict(act=-1), dict(act=4), dict(a=None), dict(b=None), dict(c=None), dict(ldc=1 << 22),
                dict(ldr=1 << 22), dict(ldp=1 << 22)):
        assert _dense(**bad) == BAD, bad
    need = ctypes.c_size_t()
    assert _lib().gcn_gemm_epilogue_workspace_bytes(128, 16, 2048, ctypes.byref(need)) == 0 and need.value > 0
    long = dict(m=128, n=16, k=2048, lda=2048, ldb=16, ldc=16, ldr=16, ldp=16)
    for bad in (dict(ws=None, nb=need.value), dict(ws=P, nb=need.value - 1), dict(ws=P + 4, nb=need.value)):
        assert _dense(**long, **bad) == WORKSPACE, bad
    assert _lib().gcn_gemm_epilogue_workspace_bytes(1 << 20, 256, 256, ctypes.byref(need)) == 0 and need.value == 0
    assert _lib().gcn_gemm_epilogue_workspace_bytes(-1, 1, 1, ctypes.byref(need)) == BAD


def _act_grad(m=4, n=5, act=2, g=P, ldo=5, pre=P, ldp=5, dz=P, ldz=5, db=None, ws=None, nb=0):
    return _lib().gcn_act_grad_f32(m, n, act, g, ldo, pre, ldp, dz, ldz, db, ws, nb, None)


def test_activation_gradient_refuses():
    assert _act_grad(m=0) == 0 and _act_grad(n=0) == 0 and _act_grad(dz=None) == 0
    for bad in (dict(m=-1), dict(n=-1), dict(act=9), dict(ldo=4), dict(ldp=4), dict(ldz=4), dict(g=None), dict(pre=None)):
        assert _act_grad(**bad) == BAD, bad
    need = ctypes.c_size_t()
    assert _lib().gcn_act_grad_workspace_bytes(4, 5, ctypes.byref(need)) == 0 and need.value >= 20
    for bad in (dict(ws=None, nb=need.value), dict(ws=P, nb=need.value - 1), dict(ws=P + 8, nb=need.value)):
        assert _act_grad(db=P, **bad) == WORKSPACE, bad


def test_quant_product_refuses():
    lib = _lib()
    assert lib.gcn_quant_dense_f32(0, 4, None, 16, None, None, 4, None) == 0
    for n, f, q, ldq, s, y, ldy in ((-1, 4, P, 16, P, P, 4), (2, 0, P, 16, P, P, 4), (2, 4, P, 8, P, P, 4), (2, 4, P, 24, P, P, 4),
                                    (2, 4, P, 16, P, P, 3), (2, 4, None, 16, P, P, 4), (2, 4, P, 16, None, P, 4),
                                    (2, 4, P, 16, P, None, 4), (2, 4, P + 8, 16, P, P, 4), (2, 17, P, 16, P, P, 17)):
        assert lib.gcn_quant_dense_f32(n, f, q, ldq, s, y, ldy, None) == BAD
    assert lib.gcn_spmm_csr_quant_f32(None, P, P, P, 4, P, 16, P, P, 4, 0, None, 0, None) == BAD


def test_host_tensors_are_refused():
    import torch
    from gcn_amd import sparse
    if torch.cuda.is_available():
        pytest.skip('host-only check')
    x = torch.ones(2, 4)
    for call in (lambda: sparse.rms_norm(x), lambda: sparse.rms_norm_grad(x, x, None, torch.ones(2)),
                 lambda: sparse.gemm_epilogue(x, x, trans_b=True), lambda: sparse.act_grad(x, x, 'relu'),
                 lambda: sparse.distill_topk(x, x, x.int(), None, 1.0), lambda: sparse.QuantRows(2, 4, torch.zeros((2, 16), dtype=torch.uint8), torch.ones(2))):
        with pytest.raises(ValueError):
            call()


def test_recording_over_a_live_eager_graph_is_refused(monkeypatch):
    """The check marks a leaf's accumulator in eager calls; the mark lives as long as a graph holds the accumulator."""
    import torch
    from gcn_amd import layers
    capturing = [False]
    monkeypatch.setattr(torch.cuda, 'is_current_stream_capturing', lambda: capturing[0])
    leaf = torch.ones(3, requires_grad=True)
    nodes = layers._accumulators(leaf, None, torch.ones(2))
    assert len(nodes) == 1
    held = (leaf * 2).sum()                       # what a wrapper's call does while it holds the nodes
    del nodes
    capturing[0] = True
    with pytest.raises(RuntimeError):
        layers._accumulators(leaf)
    with torch.no_grad():
        assert layers._accumulators(leaf) == []
    del held
    assert len(layers._accumulators(leaf)) == 1


def test_recording_over_an_eager_graph_of_a_transposed_leaf_is_refused(monkeypatch):
    import torch
    from gcn_amd import layers
    capturing = [False]
    monkeypatch.setattr(torch.cuda, 'is_current_stream_capturing', lambda: capturing[0])
    w, x = torch.ones((2, 3), requires_grad=True), torch.ones((3, 2), requires_grad=True)
    turned = w.t() * 2
    moved = x + w.sum()
    assert layers._accumulators(turned, moved) == []
    loss = (turned * moved).sum()               # what a wrapper's call does with them
    capturing[0] = True
    for again in (w, x, w.t(), turned, moved.exp(), (w.t() + 1).exp()):
        with pytest.raises(RuntimeError):
            layers._accumulators(again)
    other = torch.ones(3, requires_grad=True)
    assert len(layers._accumulators(other, other * 2)) == 1
    del turned, moved, loss, again
    assert len(layers._accumulators(w, w.t().exp(), x)) == 2


def test_calls_go_to_the_device_of_their_tensors(monkeypatch):
    import torch
    from gcn_amd import sparse

    class OnGpu(object):
        def __init__(self, index):
            self.index, self.device = index, 'cuda:%d' % index

        def get_device(self):
            return self.index
    entered = []
    monkeypatch.setattr(torch.cuda, 'current_device', lambda: 0)
    monkeypatch.setattr(torch.cuda, 'device', lambda index: entered.append(index))
    assert sparse._on_device(OnGpu(0), None, OnGpu(0)) is sparse._NO_GUARD and entered == []
    sparse._on_device(OnGpu(1), OnGpu(1))
    assert entered == [1]
    with pytest.raises(ValueError):
        sparse._on_device(OnGpu(0), OnGpu(1))
    with pytest.raises(ValueError):
        sparse._on_device(OnGpu(0), torch.ones(1))
    with pytest.raises(ValueError):
        sparse._on_device(torch.ones(1))


def test_the_distillation_loss_is_averaged_on_the_device_of_its_rows(monkeypatch):
    """With another GPU current, the rows' mean is enqueued where the rows are."""
    import contextlib
    import torch
    from gcn_amd import metrics, sparse
    current, calls = ['cuda:0'], []

    @contextlib.contextmanager
    def on_device(first, *others):
        before, current[0] = current[0], 'cuda:1'
        yield
        current[0] = before

    def distill(preds, *args, **kwargs):
        with sparse._on_device(preds):
            calls.append(('rows', current[0]))
        return torch.zeros((preds.shape[0], 2)), None

    def summary(stats, weights, decay):
        calls.append(('mean', current[0]))
        return torch.zeros(2)
    monkeypatch.setattr(torch.cuda, 'is_current_stream_capturing', lambda: False)
    monkeypatch.setattr(sparse, '_on_device', on_device)
    monkeypatch.setattr(sparse, 'distill_topk', distill)
    monkeypatch.setattr(sparse, 'loss_summary', summary)
    metrics.masked_distillation(torch.zeros(3, 4), torch.zeros(3, 2), torch.zeros((3, 2), dtype=torch.int32), mask_mean=1.0)
    assert calls == [('rows', 'cuda:1'), ('mean', 'cuda:1')] and current == ['cuda:0']


def test_outputs_across_operands_are_refused():
    """Shifted views of one buffer: where operand and result, or two results, share rows otherwise than row by row, the call
    is refused before any launch.  4 rows of 6 columns are 96 bytes; addresses far apart stand for memory of its own."""
    X, R, W, H, Y, Q, S, I = (P + (k << 16) for k in range(1, 9))
    need = ctypes.c_size_t()
    lib = _lib()

    def norm(**kw):
        return _norm(**dict(dict(x=X, r=R, ldr=6, h=H, inv=I, y=Y), **kw))
    for bad in (dict(y=X + 24), dict(y=X - 24), dict(y=X + 92), dict(y=R - 4), dict(y=H + 24), dict(y=H - 92), dict(y=X, ldy=7),
                dict(h=X + 24), dict(h=R, ldh=8), dict(inv=X + 80), dict(inv=Y), dict(inv=H + 4),
                dict(y=None, q=X, ldq=16, scales=S), dict(y=None, q=H + 80, ldq=16, scales=S), dict(y=None, q=Q, ldq=16, scales=Q + 48),
                dict(y=None, q=Q, ldq=16, scales=I + 12), dict(y=None, q=Q, ldq=16, scales=R)):
        assert norm(**bad) == BAD and b'null' not in lib.gcn_last_error_string(), bad
    assert lib.gcn_rms_norm_f32(4, 6, X, 6, None, 0, W, 1e-6, None, 6, I, W - 72, 6, None, 0, None, None) == BAD
    for bad in (dict(dx=X + 24), dict(dx=H - 92), dict(dx=R + 4, dh=R, lddh=6), dict(dx=X, lddx=9), dict(dx=I + 8)):
        assert _norm_grad(**dict(dict(dy=X, h=H, inv=I), **bad)) == BAD, bad
    assert lib.gcn_rms_norm_grad_workspace_bytes(4, 6, ctypes.byref(need)) == 0
    assert _norm_grad(dy=X, h=H, inv=I, dx=Y, dw=Y + 72, ws=Q, nbytes=need.value) == BAD

    def dense(**kw):
        return _dense(**dict(dict(a=X, b=W, bias=S, r=R, pre=H, c=Y), **kw))
    for bad in (dict(c=X), dict(c=X + 92), dict(c=X - 76), dict(c=W + 100), dict(c=W + 116), dict(c=H + 20), dict(c=H - 4), dict(c=R + 20),
                dict(c=R, ldc=6), dict(c=S), dict(pre=X + 4), dict(pre=W), dict(pre=R), dict(pre=S - 76),
                dict(tb=1, ldb=6, c=W + 116)):
        assert dense(**bad) == BAD, bad
    for bad in (dict(dz=X + 20), dict(dz=X, ldz=7), dict(dz=H - 20), dict(dz=H + 76)):
        assert _act_grad(**dict(dict(g=X, pre=H), **bad)) == BAD, bad
    assert lib.gcn_act_grad_workspace_bytes(4, 5, ctypes.byref(need)) == 0
    assert _act_grad(g=X, pre=H, dz=Y, db=Y + 60, ws=Q, nb=need.value) == BAD

    def distill(**kw):
        return _distill(**dict(dict(x=X, v=R, i=W, mask=S, stats=I, d=Y), **kw))
    for bad in (dict(d=X), dict(d=X + 24), dict(d=X - 92), dict(d=R + 44), dict(d=W - 8), dict(d=S + 12), dict(stats=X + 88),
                dict(stats=Y + 88), dict(stats=S), dict(up=Y + 4)):
        assert distill(**bad) == BAD, bad
    assert lib.gcn_quant_dense_f32(4, 6, Q, 16, S, Q + 60, 6, None) == BAD
    assert lib.gcn_quant_dense_f32(4, 6, Q, 16, S, S - 88, 6, None) == BAD


def test_streams_of_host_graphs():
    """The operator loads and walks a deep graph with shared nodes; host nodes belong to no stream, a leaf that nothing
    holds has no node."""
    import torch
    from gcn_amd import layers
    streams = layers._graph_streams()
    w = torch.ones(3, requires_grad=True)
    x = w
    for _ in range(5000):
        x = x + x
    assert list(streams([w, x, torch.ones(2)])) == [] and list(streams([])) == []
    del x
    assert list(streams([w])) == []


def test_distillation_refuses_a_temperature_without_an_inverse():
    """A logit of the maximum times an infinite 1 / T would be NaN."""
    for temp in (1e-45, 1e-39, 4e-39):
        assert _distill(x=P, v=P + (1 << 16), i=P + (2 << 16), mask=P + (3 << 16), stats=P + (4 << 16), d=P + (5 << 16), temp=temp) == BAD
