"""Row norm in 8 bits, the product that gathers it, the dense epilogue and the distillation loss together, as a deep
layer uses them: forward and gradients against float64, a step with Adam eager and as a replayed graph.

Tolerance: every operator has its own bounds in its own tests; chained they are compared relative to the largest
magnitude of the tensor.  A float32 chain of products of depth k <= 64 with magnitudes of order 1 is off by about
k u sqrt(layers) < 1e-5 of it (u = 2^-24); 1e-4 is asked."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def _graph(n, seed, self_loops=True):
    import torch
    from gcn_amd import sparse
    rng = np.random.default_rng(seed)
    rows, cols = rng.integers(0, n, 4 * n), rng.integers(0, n, 4 * n)
    rows, cols = np.concatenate([rows, cols]), np.concatenate([cols, rows])
    ip, ix, v = sparse.coo_to_csr(n, n, torch.as_tensor(rows).cuda(), torch.as_tensor(cols).cuda(), add_self_loops=self_loops)
    d = sparse.degree_scale(sparse.row_sums(ip, v))
    return sparse.DeviceCSR(n, n, ip, ix, sparse.normalize_values(ip, ix, v, d)[1])


def _setup(n=300, f=48, c=9, k=4, seed=0):
    import torch
    gen = torch.Generator().manual_seed(seed)

    def r(*shape, scale=1.0):
        return (scale * torch.randn(shape, generator=gen)).cuda()
    params = [1 + 0.1 * r(f), r(f, f, scale=f ** -0.5), 0.1 * r(f), 1 + 0.1 * r(f), r(f, f, scale=f ** -0.5), 0.1 * r(f),
              r(f, c, scale=f ** -0.5), 0.1 * r(c)]
    x = r(n, f)
    top = torch.topk(r(n, c, scale=2.0), k, dim=1)
    mask = (torch.rand(n, generator=gen) < 0.5).to(torch.int32).cuda()
    return x, [p.requires_grad_(True) for p in params], top.values.half(), top.indices.int(), mask


def _forward(a, x, params):
    """Two normalised layers with residuals and a classifier, on the framework's operators."""
    from gcn_amd import layers
    g1, w1, b1, g2, w2, b2, w3, b3 = params
    p = layers.quant_dot(a, x, g1)
    t = layers.dense(p, w1, b1, act='gelu')
    p, h = layers.quant_dot(a, t, g2, residual=x)
    z = layers.dense(p, w2, b2, act='silu', residual=h)
    return layers.dense(z, w3, b3)


class _Through:
    """The same in float64 with the 8-bit rows the kernels made: value q, gradient of y."""

    @staticmethod
    def rows(y, q):
        import torch
        value = q.data[:, :q.f].contiguous().view(torch.float8_e4m3fn).double() * q.scales.double()[:, None]
        return y + (value - y).detach()


def _reference(a, x, params, q1, q2):
    import torch
    dense_a = torch.zeros((a.n_rows, a.n_cols), dtype=torch.float64, device='cuda')
    row = torch.repeat_interleave(torch.arange(a.n_rows, device='cuda'), a.indptr[1:] - a.indptr[:-1])
    dense_a[row, a.indices.long()] = a.values.double()
    g1, w1, b1, g2, w2, b2, w3, b3 = params

    def norm(h, g):
        return h * torch.rsqrt((h * h).mean(1, keepdim=True) + 1e-6) * g
    t = dense_a @ _Through.rows(norm(x, g1), q1) @ w1 + b1
    t = 0.5 * t * (1 + torch.erf(t / 2 ** 0.5))
    h = t + x
    z = dense_a @ _Through.rows(norm(h, g2), q2) @ w2 + b2
    return (z * torch.sigmoid(z) + h) @ w3 + b3


def test_two_layers_and_the_loss_against_float64():
    import torch
    from gcn_amd import layers, metrics, sparse
    a = _graph(300, 1)
    x, params, values, idx, mask = _setup()
    x.requires_grad_(True)
    logits = _forward(a, x, params)
    loss, agreement = metrics.masked_distillation(logits, values, idx, mask, temperature=2.0)
    grads = torch.autograd.grad(loss, params + [x])
    with torch.no_grad():                                     # the rows the forward pass made
        q1 = sparse.rms_norm(x, params[0], quant=True)[0]
        t = layers.dense(sparse.spmm_quant(a, q1), params[1], params[2], act='gelu')
        q2 = sparse.rms_norm(t, params[3], residual=x, quant=True)[0]
    dparams = [p.detach().double().requires_grad_(True) for p in params]
    dx = x.detach().double().requires_grad_(True)
    ref = _reference(a, dx, dparams, q1, q2)
    assert float((logits - ref).detach().abs().max() / ref.detach().abs().max()) <= 1e-4
    logp = torch.log_softmax(values.double() / 2.0, 1)
    logq = torch.log_softmax(ref / 2.0, 1).gather(1, idx.long())
    w = mask.double() / mask.double().mean()
    ref_loss = (4.0 * (logp.exp() * (logp - logq)).sum(1) * w).mean()
    assert abs(float(loss) - float(ref_loss)) <= 1e-4 * float(ref_loss)
    hits = (logits.argmax(1) == idx[:, 0]).double() * w
    assert abs(float(agreement) - float(hits.mean())) <= 1e-6
    for got, want in zip(grads, torch.autograd.grad(ref_loss, dparams + [dx])):
        assert got.shape == want.shape
        assert float((got - want).abs().max() / want.abs().max()) <= 1e-4


def test_gradients_of_the_wrappers_with_shared_and_broadcast_inputs():
    """One tensor as x and residual, an input used by two calls, a gradient that arrives broadcast or for one output
    only, inputs that need none."""
    import torch
    from gcn_amd import layers
    x = torch.randn((20, 12), device='cuda', requires_grad=True)
    g = torch.rand(12, device='cuda', requires_grad=True)
    y, h = layers.rms_norm(x, g, residual=x)
    dx, dg = torch.autograd.grad(y.sum() + 3 * h.sum(), (x, g))
    xd, gd = x.detach().double().requires_grad_(True), g.detach().double().requires_grad_(True)
    hd = 2 * xd
    yd = hd * torch.rsqrt((hd * hd).mean(1, keepdim=True) + 1e-6) * gd
    wx, wg = torch.autograd.grad(yd.sum() + 3 * hd.sum(), (xd, gd))
    assert float((dx - wx).abs().max()) <= 1e-5 and float((dg - wg).abs().max()) <= 1e-5
    # one output only
    y, h = layers.rms_norm(x, g, residual=x)
    assert torch.equal(torch.autograd.grad(h.sum(), x)[0], torch.full_like(x, 2.0))
    y, h = layers.rms_norm(x, g, residual=x)
    assert float((torch.autograd.grad(y.sum(), g)[0] - wg).abs().max()) <= 1e-5
    # .backward() fills separate gradients
    r = x.detach().clone().requires_grad_(True)
    x.grad = None
    y, h = layers.rms_norm(x, g, residual=r)
    (y.sum() + h.sum()).backward()
    assert torch.equal(x.grad, r.grad) and x.grad.data_ptr() != r.grad.data_ptr()
    # a dense layer whose gradient is one number everywhere, without some of its inputs
    w = torch.randn((12, 5), device='cuda', requires_grad=True)
    for bias, act in ((None, None), (torch.zeros(5, device='cuda', requires_grad=True), 'relu')):
        out = layers.dense(x.detach(), w, bias, act=act)
        dw = torch.autograd.grad(out.sum(), w)[0]
        slope = torch.ones_like(out) if act is None else (out > 0).float()
        want = x.detach().double().t().contiguous() @ slope.double()
        assert float((dw - want).abs().max()) <= 1e-5
    out = layers.dense(x, w.detach(), act='silu', residual=out.detach())
    assert torch.autograd.grad(out.mean(), x)[0].shape == x.shape
    with pytest.raises(RuntimeError):
        first = torch.autograd.grad(layers.dense(x, w, act='gelu').sum(), w, create_graph=True)[0]
        torch.autograd.grad(first.sum(), x)


def test_step_with_adam_eager_and_as_a_graph():
    """Forward, loss, backward and Adam recorded once and replayed: the weights follow the eager steps bit for bit, with
    eager evaluations in between."""
    import torch
    from gcn_amd import metrics, models, sparse
    a = _graph(300, 2)
    a.plan, a.transpose().plan

    def trajectory(recorded):
        x, params, values, idx, mask = _setup(seed=5)
        mean = float(mask.float().mean())
        opt = models.TfAdam(params, 0.01)
        lr = torch.zeros((), device='cuda')

        def body():
            logits = _forward(a, x, params)
            loss, _ = metrics.masked_distillation(logits, values, idx, mask, temperature=2.0, mask_mean=mean)
            grads = torch.autograd.grad(loss, params)
            opt.step_fused(grads, lr, 5e-4)
            return loss.detach()
        graph, loss = None, None
        if recorded:
            saved = [t.detach().clone() for t in params + opt.m + opt.v]
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                body()
            torch.cuda.current_stream().wait_stream(side)
            with torch.no_grad():
                for t, s in zip(params + opt.m + opt.v, saved):
                    t.copy_(s)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                loss = body()
        losses = []
        for t in range(1, 7):
            lr.fill_(opt.step_size(t))
            if recorded:
                graph.replay()
            else:
                loss = body()
            losses.append(float(loss))
            with torch.no_grad():
                _forward(a, x, params)                        # eager work between the replays
        return losses, [p.detach().clone() for p in params]
    eager, recorded = trajectory(False), trajectory(True)
    assert eager[0] == recorded[0]
    assert all(torch.equal(p, q) for p, q in zip(eager[1], recorded[1]))


def test_recording_a_step_while_an_eager_graph_of_its_weights_lives_is_refused():
    import torch
    from gcn_amd import layers
    w = torch.randn((8, 8), device='cuda', requires_grad=True)
    x = torch.randn((4, 8), device='cuda')
    out = layers.dense(x, w, act='relu')
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match='eager autograd graph'):
        with torch.cuda.graph(graph):
            layers.dense(x, w, act='relu')
    del out, graph
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        grad = torch.autograd.grad(layers.dense(x, w, act='relu').sum(), w)[0]
    graph.replay()
    want = torch.autograd.grad(layers.dense(x, w, act='relu').sum(), w)[0]
    torch.cuda.synchronize()
    assert torch.equal(grad, want)


def test_two_recorded_steps_of_one_support_replay_side_by_side():
    """Hub rows and columns, so that forward and backward products have partial rows: the graphs share no workspace."""
    import torch
    from gcn_amd import layers, sparse
    n = 2500
    rng = np.random.default_rng(1)
    hub = np.concatenate([np.zeros(2400, int), np.ones(1500, int)])
    other = rng.integers(0, n, 3900)
    rows, cols = np.concatenate([hub, other, rng.integers(0, n, 9000)]), np.concatenate([other, hub, rng.integers(0, n, 9000)])
    ip, ix, v = sparse.coo_to_csr(n, n, torch.as_tensor(rows).cuda(), torch.as_tensor(cols).cuda(), add_self_loops=True)
    a = sparse.DeviceCSR(n, n, ip, ix, v.float())
    assert a.plan.n_chunks > 0 and a.transpose().plan.n_chunks > 0
    xs = [torch.randn((n, 96), device='cuda', requires_grad=True) for _ in range(2)]
    up = torch.randn((n, 96), device='cuda')

    def step(x):
        out = layers.quant_dot(a, x, fuse_relu=True)
        return out.detach(), torch.autograd.grad(out, x, up)[0]
    want = [step(x) for x in xs]
    graphs, outs = [], []
    for x in xs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(x))
        graphs.append(g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for o, w in zip(outs, want) for p, q in zip(o, w))


def test_a_plan_of_two_streams():
    import torch
    from gcn_amd import layers
    a = _graph(500, 3)
    a.plan
    xs = [torch.randn((500, 64), device='cuda') for _ in range(2)]
    want = [layers.quant_dot(a, x) for x in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    got = []
    for x, s in zip(xs, streams):
        with torch.cuda.stream(s):
            got.append(layers.quant_dot(a, x))
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(want, got))


def test_recording_over_eager_graphs_that_other_operations_built_is_refused():
    """A leaf that plain torch operations hold, one held through a view, an eager operand: refused while the eager graph lives
    (nothing is run backward there); afterwards the same calls record and replay."""
    import torch
    from gcn_amd import layers, metrics
    gen = torch.Generator('cuda').manual_seed(3)
    w = torch.randn((8, 8), device='cuda', generator=gen, requires_grad=True)
    x = torch.randn((4, 8), device='cuda', generator=gen)
    idx = torch.zeros((4, 1), dtype=torch.int32, device='cuda')
    # warm-up, as a recording wants it
    torch.autograd.grad(layers.dense(x, w, act='relu').sum() + layers.rms_norm(w).sum(), w)
    for eager in (lambda: (w * w).sum(), lambda: w.t().exp(), lambda: layers.dot(x, w)):
        alive = eager()
        for call in (lambda: layers.dense(x, w, act='relu'), lambda: layers.dense(x, w.t()), lambda: layers.rms_norm(w),
                     lambda: metrics.masked_distillation(w[:4], x[:, :1], idx, mask_mean=1.0)):
            with pytest.raises(RuntimeError, match='eager autograd graph'):
                with torch.cuda.graph(torch.cuda.CUDAGraph()):
                    call()
        del alive
        torch.cuda.synchronize()
    alive = w * 2
    with pytest.raises(RuntimeError, match='eager autograd graph'):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            layers.dense(x, alive)
    del alive
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        grad = torch.autograd.grad(layers.dense(x, w, act='relu').sum(), w)[0]
    for _ in range(3):
        graph.replay()
        want = torch.autograd.grad(layers.dense(x, w, act='relu').sum(), w)[0]
        torch.cuda.synchronize()
        assert torch.equal(grad, want)


def test_a_recorded_step_may_use_its_leaves_in_plain_operations_first():
    """A decay term and a transposed weight recorded before the layer that uses the weight: graphs of the recording itself."""
    import torch
    from gcn_amd import layers
    gen = torch.Generator('cuda').manual_seed(4)
    w = torch.randn((8, 8), device='cuda', generator=gen, requires_grad=True)
    x = torch.randn((4, 8), device='cuda', generator=gen)

    def step():
        decay = (w * w).sum()
        out = layers.dense(layers.dense(x, w, act='silu'), w.t())
        return torch.autograd.grad(out.sum() + decay, w)[0]
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        grad = step()
    for _ in range(3):
        with torch.no_grad():
            w.normal_(generator=gen)
        graph.replay()
        want = step()
        torch.cuda.synchronize()
        assert torch.equal(grad, want)
