"""The in-place calls the C ABI allows, against the same calls into memory of their own: equal bit for bit, the columns
behind the rows untouched.  Every row is read before it is written, by the lanes that write it."""
import ctypes

import pytest

pytestmark = pytest.mark.gpu

WIDTHS = [1, 2, 3, 5, 7, 18, 64, 255, 257, 1001, 2049, 4098, 8193, 16387, 20002, 32767]


def _stream():
    import torch
    return ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)


def _into(t, pad):
    """The same values as rows of a wider matrix: (the view, the whole)."""
    import torch
    room = torch.full((t.shape[0], t.shape[1] + pad), 9.0, device='cuda')
    room[:, :t.shape[1]] = t
    return room[:, :t.shape[1]], room


def _at(t):
    return None if t is None else ctypes.c_void_p(t.data_ptr())


@pytest.mark.parametrize('f', WIDTHS)
@pytest.mark.parametrize('pad', [0, 3])
def test_norm_gradient_over_its_operands(f, pad):
    import torch
    from gcn_amd import _lib, sparse
    n = 37 if f > 1000 else 1031
    gen = torch.Generator('cuda').manual_seed(f)
    dy, h, dh = (torch.randn((n, f), device='cuda', generator=gen) for _ in range(3))
    w = torch.randn(f, device='cuda', generator=gen)
    inv = sparse.rms_norm(h, w)[2]
    for up in (None, dh):
        want, dw = sparse.rms_norm_grad(dy, h, w, inv, grad_h=up)
        for which in ('dy', 'h') + (('dh',) if up is not None else ()):
            own = {'dy': dy, 'h': h, 'dh': up}
            view, room = _into(own[which], pad)
            own[which] = view
            ld = {k: 0 if t is None else max(t.stride(0), f) for k, t in own.items()}
            need = ctypes.c_size_t()
            _lib.call('gcn_rms_norm_grad_workspace_bytes', n, f, ctypes.byref(need))
            ws, got_w = torch.empty(need.value, dtype=torch.uint8, device='cuda'), torch.empty(f, device='cuda')
            _lib.call('gcn_rms_norm_grad_f32', n, f, _at(own['dy']), ld['dy'], _at(own['h']), ld['h'], _at(w), _at(inv),
                      _at(own['dh']), ld['dh'], _at(view), ld[which], _at(got_w), _at(ws), need.value, _stream())
            assert torch.equal(view, want) and torch.equal(got_w, dw), which
            assert bool((room[:, f:] == 9.0).all())


@pytest.mark.parametrize('n', WIDTHS)
@pytest.mark.parametrize('pad', [0, 3])
def test_activation_gradient_over_its_operands(n, pad):
    import torch
    from gcn_amd import _lib, sparse
    m = 37 if n > 1000 else 5003
    gen = torch.Generator('cuda').manual_seed(n)
    g, pre = (torch.randn((m, n), device='cuda', generator=gen) for _ in range(2))
    for act in ('relu', 'gelu', 'silu'):
        want, db = sparse.act_grad(g, pre, act)
        for which in ('g', 'pre'):
            own = {'g': g, 'pre': pre}
            view, room = _into(own[which], pad)
            own[which] = view
            need = ctypes.c_size_t()
            _lib.call('gcn_act_grad_workspace_bytes', m, n, ctypes.byref(need))
            ws, got_b = torch.empty(need.value, dtype=torch.uint8, device='cuda'), torch.empty(n, device='cuda')
            _lib.call('gcn_act_grad_f32', m, n, sparse._ACTS[act], _at(own['g']), own['g'].stride(0), _at(own['pre']),
                      own['pre'].stride(0), _at(view), view.stride(0), _at(got_b), _at(ws), need.value, _stream())
            assert torch.equal(view, want) and torch.equal(got_b, db), (act, which)
            assert bool((room[:, n:] == 9.0).all())


@pytest.mark.parametrize('f', [3, 16, 130, 1100, 9001, 20002])
def test_norm_over_x_and_the_residual(f):
    """y over one of x and the residual and h over the other, y over x with the 8-bit rows' h over the residual."""
    import torch
    from gcn_amd import sparse
    n = 41
    x, r = torch.randn((n, f), device='cuda'), torch.randn((n, f), device='cuda')
    w = torch.randn(f, device='cuda')
    y, h, inv = sparse.rms_norm(x, w, residual=r)
    for y_over in (0, 1):
        both = [x.clone(), r.clone()]
        y2, h2, inv2 = sparse.rms_norm(both[0], w, residual=both[1], out=both[y_over], sum_out=both[1 - y_over])
        assert torch.equal(y2, y) and torch.equal(h2, h) and torch.equal(inv2, inv)


def test_views_of_one_buffer():
    """Shifted rows are refused by the Python operators; columns beside each other in one wider matrix are memory of their
    own and give the results of separate matrices."""
    import torch
    from gcn_amd import sparse
    n, f = 50, 24
    buf = torch.randn((n + 1, f), device='cuda')
    r, w, b = torch.randn((n, f), device='cuda'), torch.rand(f, device='cuda'), torch.randn((f, f), device='cuda')
    rows = sparse.QuantRows(n, f, torch.zeros((n, 32), dtype=torch.uint8, device='cuda'), torch.ones(n, device='cuda'))
    flat = rows.data.flatten().view(torch.float32)
    for call in (lambda: sparse.rms_norm(buf[:n], w, out=buf[1:]), lambda: sparse.rms_norm(buf[1:], w, out=buf[:n]),
                 lambda: sparse.rms_norm(buf[:n], w, residual=r, sum_out=buf[1:]),
                 lambda: sparse.rms_norm(r, w, residual=r, sum_out=buf[:n], out=buf[1:]),
                 lambda: sparse.gemm_epilogue(buf[:n], b, out=buf[1:]), lambda: sparse.gemm_epilogue(r, b, residual=buf[:n], out=buf[1:]),
                 lambda: sparse.gemm_epilogue(b[:, :8].contiguous(), b[:8], out=b),
                 lambda: rows.rows(0, 8).dense(out=flat[:8 * f].view(8, f))):
        with pytest.raises(ValueError):
            call()
    wide = torch.randn((n, 3 * f), device='cuda')
    x, h, y = wide[:, :f], wide[:, f:2 * f], wide[:, 2 * f:]
    want_y, want_h, _ = sparse.rms_norm(x.contiguous(), w, residual=r)
    sparse.rms_norm(x, w, residual=r, out=y, sum_out=h)
    assert torch.equal(y, want_y) and torch.equal(h, want_h)
    want = sparse.gemm_epilogue(x.contiguous(), b, act='silu', residual=h.contiguous())
    assert torch.equal(sparse.gemm_epilogue(x, b, act='silu', residual=h, out=y), want)
    a = sparse.DeviceCSR(n, n, torch.arange(n + 1, device='cuda'), torch.arange(n, dtype=torch.int32, device='cuda'), torch.ones(n, device='cuda'))
    block = torch.zeros((n, 256), dtype=torch.uint8, device='cuda')
    q = sparse.rms_norm(r, w, quant=True, out=sparse.QuantRows(n, f, block[:, :32], torch.empty(n, device='cuda')))[0]
    beside = block.view(torch.float32)[:, 16:16 + f]
    assert torch.equal(sparse.spmm_quant(a, q, out=beside), q.dense())
    with pytest.raises(ValueError):
        sparse.spmm_quant(a, q, out=block.view(torch.float32)[:, 4:4 + f])
