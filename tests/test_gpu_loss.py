"""Cross entropy over the vocabulary matrix and its gradient (fw_lm_head_loss, fw_lm_head_loss_grad) against 64 bits.

Tolerances. Forward: a logit is a sum of `hidden` exact products in fp32 on the tensor cores; with each addition off
by at most 2^-23 of the running sum of magnitudes (the tensor core's adder may truncate), its error is at most
hidden * 2^-23 * A, A = max_v sum_k |h_k w_vk|; log-sum-exp is 1-Lipschitz in the largest logit error, and its own
arithmetic (exp2 of relative error 2^-21 for |z| < 2^3, sums of vocab terms in chunks) adds below 2^-17 in absolute
terms plus 2^-22 of the largest |z|. Gradient: each 16-bit rounding (p - [t], the scaled copy of h, the result) is off
by at most half a step u = finfo.eps / 2 of its value; so |dh - exact| <= u (|dh| + sum_v |dz w|) and
|dw - exact| <= u (|dw| + 2 sum_i |dz h|), plus the probabilities' relative error e_p = the logit bound above (in
absolute terms, exp turns it relative) times the same sums, and the fp32 accumulation.
"""

import pytest
import torch

pytestmark = pytest.mark.gpu
TYPES = {'fp16': torch.float16, 'bf16': torch.bfloat16}


def _inputs(n, vocab, hidden, dtype, seed=0, lean=5.0, ignore=-100):
    g = torch.Generator(device='cuda').manual_seed(1000 * n + vocab + seed)
    t = TYPES[dtype]
    w = (torch.randn(vocab, hidden, device='cuda', generator=g) * 1.4 / hidden ** 0.5).to(t)
    targets = torch.randint(vocab, (n,), device='cuda', generator=g)
    h = torch.randn(n, hidden, device='cuda', generator=g)
    h = (h + lean * torch.rand(n, 1, device='cuda', generator=g) * w[targets].float()).to(t)
    if n > 2:
        targets[torch.rand(n, device='cuda', generator=g) < 0.1] = ignore
    return h, w, targets


def _logit_error(h, w):
    size = (h.double().abs() @ w.double().abs().T).amax(1)
    z = (h.double() @ w.double().T).abs().amax(1)
    return h.size(1) * 2.0 ** -23 * size + 2.0 ** -17 + 2.0 ** -22 * z


def _want(h, w, targets, ignore=-100):
    z = h.double() @ w.double().T
    lse = torch.logsumexp(z, 1)
    kept = targets != ignore
    loss = torch.where(kept, lse - z.gather(1, targets.clamp(min=0)[:, None])[:, 0], torch.zeros_like(lse))
    return loss, lse, z, kept


SIZES = [(1, 1, 8), (1, 51866, 1280), (27, 51866, 1280), (3, 7, 64), (255, 256, 72), (256, 257, 128), (257, 255, 64),
         (700, 1000, 200), (130, 5003, 384), (2049, 3001, 768), (129, 51865, 512), (8300, 513, 64)]


@pytest.mark.parametrize('dtype', ['fp16', 'bf16'])
@pytest.mark.parametrize('n,vocab,hidden', SIZES)
def test_loss(ext, n, vocab, hidden, dtype):
    h, w, targets = _inputs(n, vocab, hidden, dtype)
    loss, lse = (torch.full((n,), float('nan'), device='cuda') for _ in range(2))
    ext.lm_head_loss(h, w, targets, loss, lse)
    assert ext.device_error() == 0
    want_loss, want_lse, _, _ = _want(h, w, targets)
    err = _logit_error(h, w)
    assert bool(((lse.double() - want_lse).abs() <= err).all()), float(((lse.double() - want_lse).abs() / err).max())
    assert bool(((loss.double() - want_loss).abs() <= 2 * err).all())
    again, lse2 = torch.empty_like(loss), torch.empty_like(lse)
    ext.lm_head_loss(h, w, targets, again, lse2)
    assert torch.equal(loss, again) and torch.equal(lse, lse2)


def _check_grad(h, w, targets, g, lse, dh, dw, ignore=-100, base=None):
    u = torch.finfo(h.dtype).eps / 2
    tiny = torch.finfo(h.dtype).smallest_normal * u
    _, _, z, kept = _want(h, w, targets, ignore)
    e_p = _logit_error(h, w)[:, None] * 3  # logits here, in lse, and the exponential
    dz = torch.exp(z - torch.logsumexp(z, 1)[:, None])
    err = dz * e_p  # of the probability
    dz[kept.nonzero()[:, 0], targets[kept]] -= 1.0
    gk = torch.where(kept, g, torch.zeros_like(g)).double()[:, None]
    # p - [t] as kept in 16 bits: half a step, and in fp16 half a subnormal step 2^-25 over the factor 2^12
    err = err + dz.abs() * u + 2.0 ** -37
    dz, err = dz * gk, err * gk.abs()
    k32 = 2.0 ** -23
    if dh is not None:
        want, size = dz @ w.double(), dz.abs() @ w.double().abs()
        bound = err @ w.double().abs() + size * w.size(0) ** 0.5 * k32 * 8 + want.abs() * u + tiny
        off = (dh.double() - want).abs()
        assert bool((off <= bound).all()), f'dh {float((off / bound).max())}'
    if dw is not None:
        want, size = dz.T @ h.double(), dz.abs().T @ h.double().abs()
        gmax = gk.abs().max()
        # the scaled copy of h: half a step, or half a subnormal step of its type
        copy = size * u + (dz.abs() / gk.abs().clamp(min=1e-30)).T @ torch.ones_like(h).double() * gmax * tiny
        if base is not None:
            want = want + base.double()
        bound = err.T @ h.double().abs() + copy + size * h.size(0) ** 0.5 * k32 * 8 + want.abs() * u + tiny
        off = (dw.double() - want).abs()
        assert bool((off <= bound).all()), f'dw {float((off / bound).max())}'


@pytest.mark.parametrize('dtype', ['fp16', 'bf16'])
@pytest.mark.parametrize('n,vocab,hidden', SIZES)
def test_loss_grad(ext, n, vocab, hidden, dtype):
    h, w, targets = _inputs(n, vocab, hidden, dtype, seed=1)
    gen = torch.Generator(device='cuda').manual_seed(n)
    for g in (torch.full((n,), 1.0 / n, device='cuda'), torch.randn(n, device='cuda', generator=gen)):
        loss, lse = torch.empty(n, device='cuda'), torch.empty(n, device='cuda')
        ext.lm_head_loss(h, w, targets, loss, lse)
        dh, dw = torch.full_like(h, float('nan')), torch.full_like(w, float('nan'))
        ext.lm_head_loss_grad(h, w, targets, lse, g, dh, dw)
        assert ext.device_error() == 0
        _check_grad(h, w, targets, g, lse, dh, dw)
        assert not dh[targets == -100].any()
        again, dw2 = torch.empty_like(dh), torch.empty_like(dw)
        ext.lm_head_loss_grad(h, w, targets, lse, g, again, dw2)
        assert torch.equal(dh, again) and torch.equal(dw, dw2), 'two runs differ'


@pytest.mark.parametrize('dtype', ['fp16', 'bf16'])
def test_loss_grad_in_several_pieces(ext, dtype):
    """Enough rows that the vocabulary is taken in several pieces, the last of them narrow."""
    n, vocab, hidden = 8000, 25000, 192
    h, w, targets = _inputs(n, vocab, hidden, dtype, seed=2)
    loss, lse = torch.empty(n, device='cuda'), torch.empty(n, device='cuda')
    ext.lm_head_loss(h, w, targets, loss, lse)
    g = torch.rand(n, device='cuda')
    dh, dw = torch.empty_like(h), torch.empty_like(w)
    ext.lm_head_loss_grad(h, w, targets, lse, g, dh, dw)
    _check_grad(h, w, targets, g, lse, dh, dw)


def test_loss_grad_parts(ext):
    """dh alone and dw alone are the same bits as both; accumulate adds to dw in place."""
    h, w, targets = _inputs(300, 2000, 256, 'bf16')
    loss, lse, g = (torch.rand(300, device='cuda') for _ in range(3))
    ext.lm_head_loss(h, w, targets, loss, lse)
    dh, dw, dh1, dw1 = torch.empty_like(h), torch.empty_like(w), torch.empty_like(h), torch.empty_like(w)
    ext.lm_head_loss_grad(h, w, targets, lse, g, dh, dw)
    ext.lm_head_loss_grad(h, w, targets, lse, g, dh1, None)
    ext.lm_head_loss_grad(h, w, targets, lse, g, None, dw1)
    assert torch.equal(dh, dh1) and torch.equal(dw, dw1)
    base = torch.randn_like(w)
    dw2 = base.clone()
    ext.lm_head_loss_grad(h, w, targets, lse, g, None, dw2, accumulate=True)
    _check_grad(h, w, targets, g, lse, None, dw2, base=base)


@pytest.mark.parametrize('dtype', ['fp16', 'bf16'])
def test_loss_ignored_rows_hold_anything(ext, dtype):
    """NaN and infinities in ignored rows (and their weights) reach no other row and no part of dw; rows of very small
    weight keep their own gradient."""
    h, w, targets = _inputs(300, 700, 128, dtype)
    targets[5], targets[7], targets[11] = -100, -100, 3
    clean = h.clone()
    g = torch.full((300,), 0.25, device='cuda')
    g[11] = 1e-9 if dtype == 'bf16' else 1e-4
    loss, lse, loss2, lse2 = (torch.empty(300, device='cuda') for _ in range(4))
    ext.lm_head_loss(clean, w, targets, loss, lse)
    dh, dw = torch.empty_like(h), torch.empty_like(w)
    ext.lm_head_loss_grad(clean, w, targets, lse, g, dh, dw)
    _check_grad(clean, w, targets, g, lse, dh, dw)
    h[5], h[7], g2 = float('nan'), float('inf'), g.clone()
    g2[5], g2[7] = float('nan'), float('inf')
    ext.lm_head_loss(h, w, targets, loss2, lse2)
    live = torch.ones(300, dtype=torch.bool, device='cuda')
    live[5] = live[7] = False
    assert torch.equal(loss, loss2) and torch.equal(lse[live], lse2[live])
    dh2, dw2 = torch.empty_like(h), torch.empty_like(w)
    ext.lm_head_loss_grad(h, w, targets, lse2, g2, dh2, dw2)
    assert torch.equal(dh, dh2) and torch.equal(dw, dw2)


def test_loss_all_ignored_and_bad_targets(ext):
    h, w, targets = _inputs(40, 300, 64, 'fp16')
    loss, lse, g = torch.empty(40, device='cuda'), torch.empty(40, device='cuda'), torch.ones(40, device='cuda')
    dh, dw = torch.empty_like(h), torch.empty_like(w)
    ext.lm_head_loss(h, w, torch.full_like(targets, 7), loss, lse, ignore_index=7)
    ext.lm_head_loss_grad(h, w, torch.full_like(targets, 7), lse, g, dh, dw, ignore_index=7)
    assert not loss.any() and not dh.any() and not dw.any() and ext.device_error() == 0
    bad = targets.clone()
    bad[3], bad[4] = 300, -7
    ext.lm_head_loss(h, w, bad, loss, lse)
    assert ext.device_error() == 2 and float(loss[3]) == 0.0 and float(loss[4]) == 0.0
    ext.lm_head_loss_grad(h, w, bad, lse, g, dh, dw)
    assert ext.device_error() == 2 and not dh[3].any() and not dh[4].any()
    skip = bad.clone()
    skip[3] = skip[4] = -100
    _check_grad(h, w, skip, g, lse, dh, dw)


def test_loss_no_rows(ext):
    h, w = torch.empty(0, 64, device='cuda').half(), torch.randn(10, 64, device='cuda').half()
    t, f = torch.empty(0, dtype=torch.long, device='cuda'), torch.empty(0, device='cuda')
    dw = torch.ones_like(w)
    ext.lm_head_loss(h, w, t, f, f.clone())
    ext.lm_head_loss_grad(h, w, t, f, f, h.clone(), dw, accumulate=True)
    assert bool((dw == 1).all())
    ext.lm_head_loss_grad(h, w, t, f, f, h.clone(), dw)
    assert not dw.any()


def test_loss_large_logits(ext):
    """Logits in the hundreds, one far above the rest: nothing overflows, and the loss of the sure rows is 0."""
    h, w, targets = _inputs(64, 900, 256, 'bf16', lean=0.0)
    targets = torch.arange(64, device='cuda')
    h = (w[:64].float() * 400).bfloat16()
    loss, lse = torch.empty(64, device='cuda'), torch.empty(64, device='cuda')
    ext.lm_head_loss(h, w, targets, loss, lse)
    want_loss, want_lse, _, _ = _want(h, w, targets)
    err = _logit_error(h, w)
    assert bool(((lse.double() - want_lse).abs() <= err).all() and ((loss.double() - want_loss).abs() <= 2 * err).all())


def test_loss_grad_is_the_derivative(ext):
    """Central differences of the 64-bit loss along a direction against the gradient's inner product with it; both are
    of the rounded inputs. Step 1e-4 of a direction of unit elements: the third-order term is below 1e-7 of the
    gradient's size; the gradient's own bound is its half steps, u * (sum of |grad . direction|) * 4."""
    h, w, targets = _inputs(60, 500, 64, 'fp16')
    g = torch.rand(60, device='cuda')
    loss, lse = torch.empty(60, device='cuda'), torch.empty(60, device='cuda')
    ext.lm_head_loss(h, w, targets, loss, lse)
    dh, dw = torch.empty_like(h), torch.empty_like(w)
    ext.lm_head_loss_grad(h, w, targets, lse, g, dh, dw)
    a, b = torch.randn(h.shape, device='cuda').double(), torch.randn(w.shape, device='cuda').double()

    def total(x, y):
        return float((_want(x, y, targets)[0] * g.double()).sum())

    for da, db, grad in ((a, b * 0, dh.double() * a), (a * 0, b, dw.double() * b)):
        e = 1e-4
        diff = (total(h.double() + e * da, w.double() + e * db) - total(h.double() - e * da, w.double() - e * db)) / (2 * e)
        assert abs(diff - float(grad.sum())) <= 4 * 2.0 ** -11 * float(grad.abs().sum()) + 1e-6 * float(grad.abs().sum())


def test_loss_captured_and_on_another_stream(ext):
    h, w, targets = _inputs(333, 3000, 128, 'fp16')
    loss, lse, g = torch.empty(333, device='cuda'), torch.empty(333, device='cuda'), torch.rand(333, device='cuda')
    dh, dw = torch.empty_like(h), torch.empty_like(w)
    ws = torch.empty(max(ext.lm_head_loss_workspace(333, 3000), ext.lm_head_loss_grad_workspace(333, 3000, 128)),
                     dtype=torch.uint8, device='cuda')

    def step():
        ext.lm_head_loss(h, w, targets, loss, lse, ws=ws)
        ext.lm_head_loss_grad(h, w, targets, lse, g, dh, dw, ws=ws)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    h.copy_(_inputs(333, 3000, 128, 'fp16', seed=5)[0])
    targets.copy_(_inputs(333, 3000, 128, 'fp16', seed=6)[2])
    for x in (dh, dw):
        x.fill_(float('nan'))
    graph.replay()
    _check_grad(h, w, targets, g, lse, dh, dw)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        dh2, dw2 = torch.empty_like(h), torch.empty_like(w)
        ext.lm_head_loss_grad(h, w, targets, lse, g, dh2, dw2)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(dh, dh2) and torch.equal(dw, dw2)


@pytest.mark.parametrize('n', [1, 16, 31, 32, 33, 63, 64, 65])
@pytest.mark.parametrize('vocab,hidden', [(1, 8), (33, 72), (129, 64), (4737, 136), (9600, 1280), (20001, 456)])
@pytest.mark.parametrize('dtype', ['fp16', 'bf16'])
def test_loss_of_few_rows(ext, n, vocab, hidden, dtype):
    """Both sides of 32 and 64 rows; shares of the vocabulary from one row to several cut tiles."""
    h, w, targets = _inputs(n, vocab, hidden, dtype)
    targets[-1] = vocab - 1
    need = ext.lm_head_loss_workspace(n, vocab)
    room = torch.full((need + 512,), 77, dtype=torch.uint8, device='cuda')
    loss, lse = (torch.full((n + 4,), 5.0, device='cuda') for _ in range(2))
    ext.lm_head_loss(h, w, targets, loss[:n], lse[:n], ws=room[:need])
    assert ext.device_error() == 0
    want_loss, want_lse, _, _ = _want(h, w, targets)
    err = _logit_error(h, w)
    assert bool(((lse[:n].double() - want_lse).abs() <= err).all())
    assert bool(((loss[:n].double() - want_loss).abs() <= 2 * err).all())
    assert bool((room[need:] == 77).all()) and bool((loss[n:] == 5).all()) and bool((lse[n:] == 5).all())


def test_loss_of_few_rows_with_rows_that_are_not_numbers(ext):
    """A row of NaN reaches its own loss only; rows of W that are NaN or infinite reach every row's."""
    h, w, targets = _inputs(20, 5000, 128, 'bf16')
    targets.clamp_(min=0)
    loss, lse = (torch.empty(20, device='cuda') for _ in range(2))
    ext.lm_head_loss(h, w, targets, loss, lse)
    h[3] = float('nan')
    bad, bad_lse = (torch.empty(20, device='cuda') for _ in range(2))
    ext.lm_head_loss(h, w, targets, bad, bad_lse)
    rest = torch.arange(20, device='cuda') != 3
    assert bool(bad[3].isnan()) and torch.equal(bad[rest], loss[rest]) and torch.equal(bad_lse[rest], lse[rest])
    w[4999] = float('nan')
    ext.lm_head_loss(h, w, targets, bad, bad_lse)
    assert bool(bad_lse.isnan().all())
