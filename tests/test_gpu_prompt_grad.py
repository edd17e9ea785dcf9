"""Gradient of the attention over packed sequences (fw_prompt_attention_grad) against 64 bits, sequence by sequence.

Tolerances, with u = finfo.eps / 2 of the 16-bit type and the forward's bounds (test_gpu_prompt.py): a probability is
off by e_p = 3 e + 2^-19 (1 + |lse|) of itself (its score, lse's error, the exponential), delta by the sum of |do|
times the bound of o, do . v by 64 * 2^-23 of its magnitudes. So ds is off by |ds| e_p + p (error of do . v and delta),
then by one rounding to 16 bits (u of it); p in its product with do by e_p + u. In fp16 the kept values are scaled so
that the largest |do| is 2^4 and p is 2^8: half a subnormal step, 2^-25, is 2^-33 of a probability and at most 2^-29 of
(largest |do|) for ds. fp32 sums of n terms: 2^-23 sqrt(n) * 4 of the magnitudes. The result is rounded once: u.
"""

import math

import pytest
import torch

from tests.test_gpu_prompt import _cu, _make, _per_head, _seen

pytestmark = pytest.mark.gpu


def _within(got, want, bound, what):
    """|got - want| <= bound; a value whose bound reaches past the type's largest number may round to infinity of its
    sign (rounding to nearest takes what lies half a step beyond the largest number there)."""
    over = (want.abs() + bound >= torch.finfo(got.dtype).max) & (got.double() == torch.sign(want) * math.inf)
    off = (got.double() - want).abs()
    assert bool(((off <= bound) | over).all()), f'{what}: {float((off / bound)[~over].max())}'


def _check_grad(q, k, v, dout, grads, lens_q, lens_k, scale, causal):
    u = torch.finfo(q.dtype).eps / 2
    tiny = torch.finfo(q.dtype).smallest_normal * u
    half = q.dtype == torch.float16
    group = q.size(1) // k.size(1)
    dq, dk, dv = grads
    want_k, want_v = torch.zeros(k.shape, dtype=torch.float64, device='cuda'), torch.zeros(v.shape, dtype=torch.float64,
                                                                                          device='cuda')
    err_k, err_v = torch.zeros_like(want_k), torch.zeros_like(want_v)
    big = float(dout.double().abs().max()) if dout.numel() else 0.0
    for rq, rk, h, x, y, z, s, e in _per_head(q, k, v, lens_q, lens_k, group, scale, causal):
        if s.numel() == 0:
            assert not dq[rq, h].any()
            continue
        d = dout[rq, h].double()
        lse = torch.logsumexp(s, 1, keepdim=True)
        lse = torch.where(lse == -math.inf, torch.zeros_like(lse), lse)
        p = torch.exp(s - lse)
        o = p @ z
        dp = d @ z.T
        delta = (d * o).sum(1, keepdim=True)
        ds = p * (dp - delta)
        worst = e.amax(1, keepdim=True)
        e_o = (p * (u + 2 * worst + 2.0 ** -20)) @ z.abs() + u * o.abs() + 2.0 ** -25 * (1 + half * z.abs().sum(0))
        e_delta = (d.abs() * (e_o + 2.0 ** -20 * o.abs())).sum(1, keepdim=True)
        e_p = 3 * worst + 2.0 ** -19 * (1 + lse.abs())
        seen = _seen(x.size(0), y.size(0), causal).double()
        e_ds = ds.abs() * (e_p + u) + p * (1 + u) * (64 * 2.0 ** -23 * (d.abs() @ z.abs().T) + e_delta)
        e_pp = p * (e_p + u)
        if half:
            e_ds = e_ds + seen * 2.0 ** -29 * big
            e_pp = e_pp + seen * 2.0 ** -33
        n32 = 4 * 2.0 ** -23
        want = scale * ds @ y
        bound = scale * (e_ds + ds.abs() * n32 * y.size(0) ** 0.5) @ y.abs() + u * want.abs() + tiny
        _within(dq[rq, h], want, bound, f'dq of head {h}')
        n = (x.size(0) * group) ** 0.5
        want_k[rk, h // group] += scale * ds.T @ x
        err_k[rk, h // group] += scale * (e_ds + ds.abs() * n32 * n).T @ x.abs()
        want_v[rk, h // group] += p.T @ d
        err_v[rk, h // group] += (e_pp + p * n32 * n).T @ d.abs()
    for got, want, err, name in ((dk, want_k, err_k, 'dk'), (dv, want_v, err_v, 'dv')):
        _within(got, want, err + u * (want.abs() + err) + tiny, name)


def _run(ext, q, k, v, dout, cq, ck, scale, causal, ws=None):
    out, lse = torch.empty(q.shape, dtype=q.dtype, device='cuda'), torch.empty(q.size(1), q.size(0), device='cuda')
    ext.prompt_attention(q, k, v, out, cq, ck, scale, causal=causal, lse=lse)
    grads = [torch.full(x.shape, float('nan'), dtype=x.dtype, device='cuda') for x in (q, k, v)]
    ext.prompt_attention_grad(q, k, v, out, dout, lse, cq, ck, scale, *grads, causal=causal, ws=ws)
    return out, lse, grads


CASES = [  # lq, lk, heads, kv_heads, causal, dtype
    ([1], [1], 1, 1, True, 'fp16'), ([4], [4], 2, 2, True, 'bf16'), ([64], [64], 1, 1, True, 'fp16'),
    ([128], [128], 1, 1, False, 'fp16'), ([448, 27], [448, 27], 20, 20, True, 'fp16'),
    ([127, 128, 129], [127, 128, 129], 2, 2, True, 'bf16'), ([255, 256, 257], [255, 256, 257], 2, 1, True, 'fp16'),
    ([700, 1, 0, 33], [700, 1, 0, 33], 8, 2, True, 'bf16'), ([27, 1, 100], [1500, 1500, 77], 4, 4, False, 'fp16'),
    ([100, 60, 3], [130, 300, 3], 6, 2, True, 'fp16'), ([50, 40], [20, 0], 5, 1, True, 'bf16'),
    ([300], [200], 10, 2, True, 'fp16'), ([90, 11, 0], [0, 140, 50], 7, 1, False, 'bf16'),
    ([385], [385], 14, 2, True, 'bf16'), ([70], [70], 128, 1, True, 'fp16'), ([65], [65], 96, 1, True, 'bf16'),
    ([1031], [1031], 6, 2, False, 'fp16'), ([1, 1, 1], [500, 1, 129], 8, 2, True, 'bf16'),
    ([2100], [2100], 4, 1, True, 'fp16')]


@pytest.mark.parametrize('lq,lk,heads,kv_heads,causal,dtype', CASES)
def test_prompt_attention_grad(ext, lq, lk, heads, kv_heads, causal, dtype):
    q, k, v = _make(lq, lk, heads, kv_heads, dtype)
    dout = torch.randn(q.shape, device='cuda').to(q.dtype)
    _, _, grads = _run(ext, q, k, v, dout, _cu(lq), _cu(lk), 1.5 / 8, causal)
    assert ext.device_error() == 0
    _check_grad(q, k, v, dout, grads, lq, lk, 1.5 / 8, causal)
    _, _, again = _run(ext, q, k, v, dout, _cu(lq), _cu(lk), 1.5 / 8, causal)
    assert all(torch.equal(a, b) for a, b in zip(grads, again)), 'two runs differ'


@pytest.mark.parametrize('size', [1e-6, 3e4])
def test_prompt_attention_grad_keeps_small_and_large_gradients(ext, size):
    """fp16 gradients near the type's ends: subnormal ones as well as large ones."""
    q, k, v = _make([300, 40], [300, 40], 4, 2, 'fp16')
    v = (v * 0.01).half() if size > 1 else v
    dout = (torch.rand(q.shape, device='cuda') * 2 - 1).mul(size).half()
    scale = 0.02 if size > 1 else 0.125
    _, _, grads = _run(ext, q, k, v, dout, _cu([300, 40]), _cu([300, 40]), scale, True)
    _check_grad(q, k, v, dout, grads, [300, 40], [300, 40], scale, True)


def test_prompt_attention_grad_layouts(ext):
    """Gradients written into a fused buffer's views and read from heads-first tensors: the same bits."""
    q, k, v = _make([140, 77], [140, 77], 6, 2, 'fp16')
    cu = _cu([140, 77])
    dout = torch.randn(217, 6, 64, device='cuda').half()
    out, lse, want = _run(ext, q, k, v, dout, cu, cu, 0.125, True)
    fused = torch.full((217, 11, 64), 5.0, dtype=q.dtype, device='cuda')

    def heads_first(x):
        return x.transpose(0, 1).contiguous().transpose(0, 1)

    ext.prompt_attention_grad(heads_first(q), heads_first(k), heads_first(v), heads_first(out), heads_first(dout), lse,
                              cu, cu, 0.125, fused[:, :6], fused[:, 6:8], fused[:, 8:10])
    assert torch.equal(fused[:, :6], want[0]) and torch.equal(fused[:, 6:8], want[1])
    assert torch.equal(fused[:, 8:10], want[2]) and bool((fused[:, 10] == 5).all())


@pytest.mark.parametrize('dtype', ['fp16', 'bf16'])
def test_prompt_attention_grad_neighbours_and_tails(ext, dtype):
    """NaN and infinities in rows of no sequence and in a neighbour sequence reach no other; rows of no sequence stay."""
    lens = [130, 61, 200]
    q, k, v = _make(lens, lens, 4, 2, dtype, fused=False)
    dout = torch.randn(q.shape, device='cuda').to(q.dtype)
    # the largest |do| is the same with and without the middle sequence, so the scaling is too
    dout[0, 0, 0] = 6.0
    cu = _cu(lens)
    _, _, want = _run(ext, q, k, v, dout, cu, cu, 0.2, True)

    def padded(x):
        fill = torch.full((45, *x.shape[1:]), float('nan'), dtype=x.dtype, device='cuda')
        return torch.cat([fill[:5], x, fill[:40]])

    q2, k2, v2, d2 = padded(q), padded(k), padded(v), padded(dout)
    a, b = 5 + 130, 5 + 191
    q2[a:b], k2[a:b], v2[a:b], d2[a:b] = float('nan'), float('inf'), float('nan'), float('-inf')
    out, lse = torch.zeros_like(q2), torch.zeros(4, q2.size(0), device='cuda')
    out[:5] = out[-40:] = float('nan')
    lse[:, :5] = lse[:, -40:] = float('nan')
    ext.prompt_attention(q2, k2, v2, out, cu + 5, cu + 5, 0.2, lse=lse)
    grads = [torch.full_like(x, 7.0) for x in (q2, k2, v2)]
    ext.prompt_attention_grad(q2, k2, v2, out, d2, lse, cu + 5, cu + 5, 0.2, *grads)
    for got, ref in zip(grads, want):
        assert bool((got[:5] == 7).all() and (got[-40:] == 7).all())
        assert torch.equal(got[5:a], ref[:130]) and torch.equal(got[b:-40], ref[191:])
    assert ext.device_error() == 0


def test_prompt_attention_grad_bad_offsets(ext):
    q, k, v = _make([64, 64], [64, 64], 2, 2, 'fp16', fused=False)
    dout = torch.randn(q.shape, device='cuda').half()
    out, lse, good = _run(ext, q, k, v, dout, _cu([64, 64]), _cu([64, 64]), 0.1, True)
    ext.device_error()
    for cq, ck in (([0, 64, 200], [0, 64, 128]), ([0, 64, 128], [0, 64, 300]), ([0, 64, 10], [0, 64, 128]),
                   ([0, 64, 128], [0, 64, -5])):
        grads = [torch.full_like(x, 3.0) for x in (q, k, v)]
        d = dout.clone()
        ext.prompt_attention_grad(q, k, v, out, d, lse, torch.tensor(cq, device='cuda'), torch.tensor(ck, device='cuda'),
                                  0.1, *grads)
        assert ext.device_error() == 2
        for got in grads:
            assert bool((got[64:] == 3).all()) and bool(got[:64].isfinite().all())


def test_prompt_attention_grad_is_the_derivative(ext):
    """Central differences of the 64-bit forward pass along directions of unit elements, step 1e-4 (third-order terms
    below 1e-6 of the size); the gradient itself within its half steps: 4 u of the sum of magnitudes."""
    lens = [50, 30]
    q, k, v = _make(lens, lens, 2, 1, 'fp16', fused=False)
    dout = torch.randn(q.shape, device='cuda').half()
    cu = _cu(lens)
    _, _, grads = _run(ext, q, k, v, dout, cu, cu, 0.125, True)
    base = [x.double() for x in (q, k, v)]

    def total(x):
        sums = 0.0
        for rq, _, h, _, _, z, s, _ in _per_head(*x, lens, lens, 2, 0.125, True):
            sums += float((torch.softmax(s, 1) @ z * dout[rq, h].double()).sum())
        return sums

    for i in range(3):
        step = torch.randn(base[i].shape, device='cuda').double()
        moved = [[b + sign * 1e-4 * step if i == j else b for j, b in enumerate(base)] for sign in (1, -1)]
        diff = (total(moved[0]) - total(moved[1])) / 2e-4
        prod = grads[i].double() * step
        assert abs(diff - float(prod.sum())) <= (4 * 2.0 ** -11 + 1e-6) * float(prod.abs().sum())


def test_prompt_attention_grad_captured_and_on_another_stream(ext):
    lens = [200, 130]
    q, k, v = _make(lens, lens, 8, 2, 'fp16', fused=False)
    dout = torch.randn(q.shape, device='cuda').half()
    cu = _cu(lens)
    ws = torch.empty(ext.prompt_attention_grad_workspace(330, 330, 2, 8, 2), dtype=torch.uint8, device='cuda')
    out, lse, grads = _run(ext, q, k, v, dout, cu, cu, 0.125, True, ws=ws)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ext.prompt_attention(q, k, v, out, cu, cu, 0.125, lse=lse)
        ext.prompt_attention_grad(q, k, v, out, dout, lse, cu, cu, 0.125, *grads, ws=ws)
    a, b, c = _make(lens, lens, 8, 2, 'fp16', seed=5, fused=False)
    q.copy_(a), k.copy_(b), v.copy_(c)
    cu.copy_(_cu([90, 240]))
    graph.replay()
    _check_grad(q, k, v, dout, grads, [90, 240], [90, 240], 0.125, True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = [torch.empty_like(x) for x in grads]
        ext.prompt_attention_grad(q, k, v, out, dout, lse, cu, cu, 0.125, *again)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(x, y) for x, y in zip(grads, again))


def test_prompt_attention_grad_nothing_to_do(ext):
    q = torch.empty(0, 4, 64, dtype=torch.float16, device='cuda')
    lse = torch.empty(4, 0, device='cuda')
    ext.prompt_attention_grad(q, q, q, q, q, lse, _cu([]), _cu([]), 0.1, q, q, q)
    ext.prompt_attention_grad(q, q, q, q, q, lse, _cu([0, 0]), _cu([0, 0]), 0.1, q, q, q)
    x = torch.randn(3, 4, 64, device='cuda').half()
    a, b, c = (torch.ones_like(x) for _ in range(3))
    ext.prompt_attention_grad(x, q, q, x, x, torch.zeros(4, 3, device='cuda'), _cu([3]), _cu([0]), 0.1, a, q, q)
    assert not a.any()
    ext.prompt_attention_grad(q, x, x, q, q, lse, _cu([0]), _cu([3]), 0.1, q, b, c)
    assert not b.any() and not c.any()
    assert ext.device_error() == 0
