"""Distillation from a teacher's top logits, and its gradient, against the formulas in float64.

Tolerances, with u = 2^-24: an exponent (s - max) / T of size z is off by 2 u |z| (one product with a rounded 1 / T), so
its exponential by (2 |z| + 2) u of itself; |z| counts only up to 104, where the exponential leaves float32.  A sum of c
terms in lanes of at most 64 serial terms and a tree is off by 80 u.  The inputs here have |z| <= 40, so q and p are
within 250 u of themselves, log q within (2 * 40 + 80 + 2) u + u |log q| < 300 u absolutely, a row's loss within
T^2 w (300 + 300) u (1 + sum p |log p - log q|), a gradient within 600 u of (q + P) T w / n.  Terms below the float32
normal range (2^-126) may be lost: 1e-37 is allowed on top."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def _case(n, c, k, seed=0, kept=0.7, dtype='float32', scale=3.0):
    import torch
    gen = torch.Generator().manual_seed(n * 131 + c * 7 + k + seed)
    logits = scale * torch.randn((n, c), generator=gen)
    teacher = logits + torch.randn((n, c), generator=gen)
    top = torch.topk(teacher, min(k, c), dim=1)
    values, idx = top.values, top.indices.to(torch.int32)
    if k > c:                                                   # padded lists
        values = torch.cat([values, torch.zeros(n, k - c)], 1)
        idx = torch.cat([idx, torch.full((n, k - c), -1, dtype=torch.int32)], 1)
    mask = (torch.rand(n, generator=gen) < kept).to(torch.int32)
    mask[0] = 1
    return logits.cuda(), values.to(getattr(torch, dtype)).cuda(), idx.cuda(), mask.cuda()


def _reference(logits, values, idx, mask, mean, temp):
    import torch
    n, c = logits.shape
    z = logits.double() / temp
    logq = torch.log_softmax(z, 1)
    here = (idx >= 0) & (idx < c)
    t = torch.where(here, values.double() / temp, -np.inf)
    any_ = (t > -np.inf).any(1)
    t = torch.where(any_[:, None], t, 0.0)
    logp = torch.log_softmax(t, 1)
    p = torch.where(any_[:, None] & here, logp.exp(), 0.0)
    at = torch.where(here, idx, 0).long()
    terms = torch.where(p > 0, p * (logp - logq.gather(1, at)), 0.0)
    w = (mask.double() if mask is not None else torch.ones(n, dtype=torch.float64, device='cuda')) / mean
    tied = torch.where(here & (t == t.amax(1, keepdim=True)), torch.arange(idx.shape[1], device=idx.device), 1 << 30)
    big = idx.gather(1, tied.amin(1).clamp(max=idx.shape[1] - 1)[:, None])[:, 0]
    agree = (logits.argmax(1) == big) & any_
    teacher = torch.zeros((n, c), dtype=torch.float64, device='cuda').scatter_add_(1, at, p)
    q = torch.where(any_[:, None], logq.exp(), 0.0)
    coef = (w * temp / n)[:, None]
    return (terms.sum(1) * w * temp ** 2, agree.double() * w, (q - teacher) * coef, (q + teacher) * coef,
            (1 + terms.abs().sum(1)) * w * temp ** 2)


def _check(stats, grad, ref):
    loss, agree, g, gsize, lsize = ref
    if stats is not None:
        assert bool(((stats[:, 0].double() - loss).abs() <= 600 * U * lsize + 1e-37).all())
        assert bool(((stats[:, 1].double() - agree).abs() <= 4 * U * agree).all())
    if grad is not None:
        assert bool(((grad.double() - g).abs() <= 600 * U * gsize + 1e-37).all())


SHAPES = [(1, 1, 1), (5, 2, 2), (1, 3, 5), (2708, 7, 3), (333, 4, 4), (130, 6, 1), (129, 8, 8), (77, 9, 4), (1000, 16, 5),
          (515, 17, 20), (64, 33, 7), (4099, 47, 5), (31, 64, 64), (9, 65, 3), (21, 128, 128), (7, 130, 256), (33, 256, 9),
          (5, 257, 65), (6, 512, 32), (3, 513, 100), (5, 1000, 256), (2, 1025, 7), (3, 4097, 33), (2, 8193, 64),
          (2, 20000, 200), (1, 32768, 32), (1, 50001, 5), (1, 65536, 256), (2, 65537, 17), (1, 200003, 50),
          (300, 33333, 9)]


@pytest.mark.parametrize('n,c,k', SHAPES)
def test_loss_agreement_and_gradient(n, c, k):
    import torch
    from gcn_amd import sparse
    for temp, dtype in ((1.0, 'float32'), (2.5, 'float16'), (4.0, 'bfloat16')):
        logits, values, idx, mask = _case(n, c, k, dtype=dtype)
        mean = float(mask.float().mean())
        stats, grad = sparse.distill_topk(logits, values, idx, mask, mean, temperature=temp)
        _check(stats, grad, _reference(logits, values, idx, mask, mean, temp))
        assert bool((grad[mask == 0] == 0).all()) and bool((stats[mask == 0] == 0).all())
        again, none = sparse.distill_topk(logits, values, idx, mask, mean, temperature=temp, want_grad=False)
        assert none is None and torch.equal(again, stats)
        none, only = sparse.distill_topk(logits, values, idx, mask, mean, temperature=temp, want_stats=False)
        assert none is None and torch.equal(only, grad)
        up = torch.tensor(0.25, device='cuda')
        assert torch.equal(sparse.distill_topk(logits, values, idx, mask, mean, temperature=temp, upstream=up)[1], grad * 0.25)
    stats, grad = sparse.distill_topk(logits, values, idx, None, 1.0)
    _check(stats, grad, _reference(logits, values, idx, None, 1.0, 1.0))


WIDTHS = [3, 7, 16, 47, 130, 300, 1000, 3000, 9000, 33000, 70000]


@pytest.mark.parametrize('c', WIDTHS)
def test_lists_with_repeats_padding_and_nothing_in_them(c):
    """A class listed several times counts every time, entries outside [0, c) not at all, rows without an entry (or with
    -inf only) have neither loss nor gradient; of equal logits the first listed one is the teacher's choice."""
    import torch
    from gcn_amd import sparse
    n, k = 9, 6
    logits, values, idx, _ = _case(n, c, k)
    idx = idx.clone()
    idx[0] = 1                                              # one class six times
    idx[1, 3:] = idx[1, 0]                                  # the top class four times
    idx[2, 1:] = torch.tensor([-1, c, 2 ** 31 - 1, -2 ** 31, -7], device='cuda', dtype=torch.int32)
    idx[3] = -1
    values[4] = float('-inf')
    values[5, 2:] = float('-inf')
    values[6] = 1.5                                         # all tied: the first listed class
    logits[6, int(idx[6, 0])] = 99.0
    values[8] = 1.5
    logits[8, int(idx[8, 1])] = 99.0
    values[7] += 1000.0                                     # large logits: only differences count
    mask = torch.ones(n, dtype=torch.int32, device='cuda')
    stats, grad = sparse.distill_topk(logits, values, idx, mask, 1.0, temperature=2.0)
    _check(stats, grad, _reference(logits, values, idx, mask, 1.0, 2.0))
    assert bool((stats[3:5] == 0).all()) and bool((grad[3:5] == 0).all()) and float(stats[6, 1]) == 1.0 and float(stats[8, 1]) == 0.0
    assert torch.equal(sparse.distill_topk(logits, values, idx, mask, 1.0, temperature=2.0)[1], grad)


@pytest.mark.parametrize('c', WIDTHS)
def test_masked_rows_are_not_read_and_infinities(c):
    import torch
    from gcn_amd import sparse
    n, k = 8, 2
    logits, values, idx, _ = _case(n, c, k)
    k = values.shape[1]
    mask = torch.tensor([1, 0, 1, 0, 1, 1, 1, 1], dtype=torch.int32, device='cuda')
    logits[1], values[3] = float('nan'), float('nan')        # rows outside the mask
    low = torch.finfo(torch.float32).min
    off = [j for j in range(c) if j not in idx[2].tolist()][:1]
    logits[2, off] = float('-inf')                           # a class ruled out
    off4 = [j for j in range(c) if j not in idx[4].tolist()][:1]
    logits[4, off4] = low                                    # and by the type's lowest value
    logits[5, c - 1] = float('nan')
    values[6, 0] = float('nan')
    logits[7, int(idx[7, 0])] = float('-inf')
    mean = 0.75
    stats, grad = sparse.distill_topk(logits, values, idx, mask, mean)
    ref = _reference(logits, values, idx, mask, mean, 1.0)
    for row in (0, 2, 4):
        _check(stats[row:row + 1], grad[row:row + 1], [r[row:row + 1] for r in ref])
    for row in (1, 3):
        assert bool((stats[row] == 0).all()) and bool((grad[row] == 0).all())
    for row in (5, 6):
        assert bool(torch.isnan(stats[row, 0])) and bool(torch.isnan(grad[row]).all())
    assert float(stats[7, 0]) == float('inf') and bool(torch.isfinite(grad[7]).all())
    _check(None, grad[7:], [None, None, ref[2][7:], ref[3][7:], None])


def test_gradient_against_differences():
    """Central differences of the mean loss in float64 on the formula, step 1e-5: their own error is about 1e-9."""
    import torch
    from gcn_amd import sparse
    logits, values, idx, mask = _case(6, 11, 4)
    mean = float(mask.float().mean())
    grad = sparse.distill_topk(logits, values, idx, mask, mean, temperature=1.7)[1]

    def value(x):
        return float(_reference(x, values, idx, mask, mean, 1.7)[0].mean())
    for i, j in ((0, 0), (0, 10), (3, 5), (5, int(idx[5, 0]))):
        e = torch.zeros((6, 11), dtype=torch.float64, device='cuda')
        e[i, j] = 1e-5
        assert abs((value(logits.double() + e) - value(logits.double() - e)) / 2e-5 - float(grad[i, j])) <= 1e-6


def test_views_streams_and_a_replayed_graph():
    import torch
    from gcn_amd import sparse
    n, c, k = 700, 19, 4
    logits, values, idx, mask = _case(n, c, k)
    wide = torch.zeros((n, c + 6), device='cuda')
    wide[:, 3:3 + c] = logits
    lists = torch.stack([idx, idx], 2)[:, :, 0]              # a strided view
    a = sparse.distill_topk(logits, values, idx, mask, 0.5)
    b = sparse.distill_topk(wide[:, 3:3 + c], values, lists, mask, 0.5)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        stats, grad = sparse.distill_topk(logits, values, idx, mask, 0.5, temperature=3.0)
        summary = sparse.loss_summary(stats, None, 0.0)
    for _ in range(3):
        logits.copy_(torch.randn_like(logits))
        graph.replay()
        s, g = sparse.distill_topk(logits, values, idx, mask, 0.5, temperature=3.0)
        torch.cuda.synchronize()
        assert torch.equal(s, stats) and torch.equal(g, grad) and torch.equal(sparse.loss_summary(s, None, 0.0), summary)


@pytest.mark.parametrize('n,c,at', [(4300001, 601, 3573000), (67109001, 9, (1 << 26) - 4), (4194400, 1030, (1 << 22) - 4)])
def test_more_rows_than_one_launch_takes_and_offsets_past_32_bits(n, c, at):
    """Element offsets past 2^31, and more rows than one launch takes of narrow and of wide ones; sampled rows against the
    formula, among them those around `at`: where the element offset passes 2^31, or where the second launch begins."""
    import torch
    from gcn_amd import sparse
    k = 3
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip('needs 40 GB of free device memory')
    logits = torch.empty((n, c), device='cuda').normal_(generator=torch.Generator('cuda').manual_seed(3))
    values = torch.randn((n, k), device='cuda')
    idx = torch.randint(0, c, (n, k), device='cuda', dtype=torch.int32)
    stats, grad = sparse.distill_topk(logits, values, idx, None, 1.0)
    for lo in (0, at - 20, 4194290, n - 40):
        rows = slice(lo, lo + 40)
        ref = list(_reference(logits[rows], values[rows], idx[rows], None, 1.0, 1.0))
        ref[2], ref[3] = ref[2] * 40 / n, ref[3] * 40 / n
        _check(stats[rows], grad[rows], ref)


def test_empty_and_refusals():
    import torch
    from gcn_amd import sparse
    logits, values, idx, mask = _case(4, 6, 2)
    s, g = sparse.distill_topk(logits[:0], values[:0], idx[:0], mask[:0], 1.0)
    assert s.shape == (0, 2) and g.shape == (0, 6)
    bad = [lambda: sparse.distill_topk(logits, values, idx.long(), mask, 1.0),
           lambda: sparse.distill_topk(logits, values.double(), idx, mask, 1.0),
           lambda: sparse.distill_topk(logits, values, idx, mask.float(), 1.0),
           lambda: sparse.distill_topk(logits, values[:3], idx[:3], mask, 1.0),
           lambda: sparse.distill_topk(logits, values, idx[:, :1], mask, 1.0),
           lambda: sparse.distill_topk(logits, values, idx, mask[:3], 1.0),
           lambda: sparse.distill_topk(logits, values, idx, mask, 0.0),
           lambda: sparse.distill_topk(logits, values, idx, mask, 1.0, temperature=0.0),
           lambda: sparse.distill_topk(logits, values[:, :0], idx[:, :0], mask, 1.0),
           lambda: sparse.distill_topk(logits, values.repeat(1, 200), idx.repeat(1, 200), mask, 1.0),
           lambda: sparse.distill_topk(logits, values.cpu(), idx, mask, 1.0),
           lambda: sparse.distill_topk(logits[0], values, idx, mask, 1.0),
           lambda: sparse.distill_topk(logits, values, idx, mask, 1.0, upstream=torch.ones(2, device='cuda'))]
    for call in bad:
        with pytest.raises(ValueError):
            call()


def test_masks_and_indices_as_the_framework_and_topk_give_them():
    """Bool masks and int64 indices through the loss, equal to the int32 ones bit for bit; an index past 32 bits is no
    entry, a mask of fractions and indices of another kind are refused."""
    import torch
    from gcn_amd import metrics
    logits, values, idx, mask = _case(300, 40, 5)
    logits.requires_grad_(True)
    idx[3, 1], idx[4, 2] = -1, 40
    want = metrics.masked_distillation(logits, values, idx, mask, temperature=2.0)
    grad = torch.autograd.grad(want[0], logits)[0]
    far = idx.long()
    far[3, 1], far[4, 2] = 2 ** 32 + 3, -2 ** 40 + 1
    for m in (mask.bool(), mask.long(), mask.to(torch.uint8)):
        got = metrics.masked_distillation(logits, values, far, m, temperature=2.0)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        assert torch.equal(torch.autograd.grad(got[0], logits)[0], grad)
    for bad in (lambda: metrics.masked_distillation(logits, values, idx, mask.float()),
                lambda: metrics.masked_distillation(logits, values, idx.float(), mask),
                lambda: metrics.masked_distillation(logits, values, idx, mask.bool()[:299], mask_mean=1.0),
                lambda: metrics.masked_distillation(logits, values, idx, torch.zeros_like(mask).bool())):
        with pytest.raises(ValueError):
            bad()
