"""Attention over packed sequences (fw_prompt_attention) and its gradient against 64 bits, sequence by sequence.

Tolerances. u = finfo.eps / 2 is half a step of the 16-bit type. A score is a sum of 64 exact products in fp32, off by
at most e = scale * 64 * 2^-23 * sum |q k| (the tensor core may truncate) plus 2^-22 of its size (the scaling); that
makes each probability off by 2 e + 2^-20 of itself (its own score, the sum's, the exponentials). In the product with v
a probability is rounded to 16 bits: u of it, and in fp16 at most half a subnormal step, 2^-25 (against a largest
probability of at least 1 on that scale). The result is rounded once more: u |o|.
"""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu
TYPES = {'fp16': torch.float16, 'bf16': torch.bfloat16}


def _cu(lens):
    return torch.tensor([0] + list(lens), device='cuda').cumsum(0)


def _seen(lq, lk, causal):
    i, j = torch.arange(lq, device='cuda')[:, None], torch.arange(lk, device='cuda')[None]
    return (j <= i + lk - lq) if causal else torch.ones(lq, lk, dtype=torch.bool, device='cuda')


def _per_head(q, k, v, lens_q, lens_k, group, scale, causal):
    """(rows of q, rows of k, head, 64-bit q, k, v, scores with -inf, error bound of the scores) of each sequence."""
    a = b = 0
    for lq, lk in zip(lens_q, lens_k):
        for h in range(q.size(1)):
            x, y, z = q[a:a + lq, h].double(), k[b:b + lk, h // group].double(), v[b:b + lk, h // group].double()
            s = (x @ y.T * scale).masked_fill(~_seen(lq, lk, causal), -math.inf)
            e = scale * (64 * 2.0 ** -23 * (x.abs() @ y.abs().T)) + 2.0 ** -22 * (x @ y.T * scale).abs()
            yield slice(a, a + lq), slice(b, b + lk), h, x, y, z, s, e
        a, b = a + lq, b + lk


def _make(lens_q, lens_k, heads, kv_heads, dtype, seed=0, fused=None):
    g = torch.Generator(device='cuda').manual_seed(seed + sum(lens_q) * 7 + heads)
    t = TYPES[dtype]

    def rand(*shape):
        return torch.randn(*shape, device='cuda', generator=g).to(t)

    if fused if fused is not None else lens_q == lens_k:
        x = rand(sum(lens_q), heads + 2 * kv_heads, 64)
        return x[:, :heads], x[:, heads:heads + kv_heads], x[:, heads + kv_heads:]
    return rand(sum(lens_q), heads, 64), rand(sum(lens_k), kv_heads, 64), rand(sum(lens_k), kv_heads, 64)


def _check(q, k, v, out, lse, lens_q, lens_k, scale, causal):
    u = torch.finfo(q.dtype).eps / 2
    group = q.size(1) // k.size(1)
    for rq, rk, h, x, y, z, s, e in _per_head(q, k, v, lens_q, lens_k, group, scale, causal):
        if s.numel() == 0:
            assert not out[rq, h].any() and bool((lse[h, rq] == -math.inf).all())
            continue
        want_lse = torch.logsumexp(s, 1)
        empty = want_lse == -math.inf
        p = torch.exp(s - torch.where(empty, torch.zeros_like(want_lse), want_lse)[:, None])
        want = p @ z
        worst = e.amax(1, keepdim=True)
        bound = (p * (u + 2 * worst + 2.0 ** -20)) @ z.abs() + u * want.abs() + 2.0 ** -25
        if q.dtype == torch.float16:
            bound = bound + 2.0 ** -25 * (_seen(x.size(0), y.size(0), causal).double() @ z.abs())
        off = (out[rq, h].double() - want).abs()
        assert bool((off <= bound).all()), f'head {h}: {float((off / bound).max())}'
        got = lse[h, rq].double()
        assert bool((got[empty] == -math.inf).all()) and not out[rq, h][empty].any()
        near = (got - want_lse).abs() <= worst[:, 0] + 2.0 ** -20 * (1 + want_lse.abs())
        assert bool(near[~empty].all()), f'lse of head {h}'


CASES = [  # lq, lk, heads, kv_heads, causal, dtype
    ([1], [1], 1, 1, True, 'fp16'), ([4], [4], 20, 20, True, 'fp16'), ([448], [448], 20, 20, True, 'fp16'),
    ([127, 128, 129], [127, 128, 129], 2, 2, True, 'bf16'), ([255, 256, 257], [255, 256, 257], 2, 1, True, 'fp16'),
    ([700, 1, 0, 33], [700, 1, 0, 33], 8, 2, True, 'bf16'), ([1] * 8, [448, 1500, 1, 37, 1499, 224, 700, 129], 20, 20,
                                                           True, 'fp16'),
    ([1, 1, 1], [5000, 1, 0], 8, 1, True, 'bf16'), ([27, 1, 448], [1500, 1500, 1500], 4, 4, False, 'fp16'),
    ([100, 60, 3], [130, 300, 3], 6, 2, True, 'fp16'), ([50, 40], [20, 0], 5, 1, True, 'bf16'),
    ([300], [200], 10, 2, True, 'fp16'), ([90, 11], [0, 140], 7, 1, False, 'bf16'),
    ([385], [385], 14, 2, True, 'bf16'), ([130], [130], 128, 1, True, 'fp16'), ([65], [65], 96, 1, True, 'bf16'),
    ([1031], [1031], 12, 4, False, 'fp16'), ([2], [4097], 2, 2, True, 'fp16')]


@pytest.mark.parametrize('lq,lk,heads,kv_heads,causal,dtype', CASES)
def test_prompt_attention(ext, lq, lk, heads, kv_heads, causal, dtype):
    q, k, v = _make(lq, lk, heads, kv_heads, dtype)
    scale = 1.5 / 8
    out = torch.full((sum(lq), heads, 64), float('nan'), dtype=q.dtype, device='cuda')
    lse = torch.full((heads, sum(lq)), float('nan'), device='cuda')
    ext.prompt_attention(q, k, v, out, _cu(lq), _cu(lk), scale, causal=causal, lse=lse)
    assert ext.device_error() == 0
    _check(q, k, v, out, lse, lq, lk, scale, causal)
    again = torch.empty_like(out)
    ext.prompt_attention(q, k, v, again, _cu(lq), _cu(lk), scale, causal=causal)
    assert torch.equal(out, again)


@pytest.mark.parametrize('dtype', ['fp16', 'bf16'])
def test_prompt_attention_large_scores(ext, dtype):
    """Scores in the hundreds whose maximum moves from block to block."""
    q, k, v = _make([600], [600], 4, 2, dtype)
    k = k * (torch.arange(600, device='cuda')[:, None, None] / 40).to(k.dtype)
    out, lse = torch.empty(600, 4, 64, dtype=q.dtype, device='cuda'), torch.empty(4, 600, device='cuda')
    ext.prompt_attention(q, k, v, out, _cu([600]), _cu([600]), 2.0, lse=lse)
    _check(q, k, v, out, lse, [600], [600], 2.0, True)


def test_prompt_attention_layouts(ext):
    """Heads before rows, rows with gaps, a strided output: the same bits as the plain layout."""
    q, k, v = _make([140, 77], [140, 77], 6, 2, 'fp16', fused=False)
    cu = _cu([140, 77])
    want = torch.empty_like(q)
    ext.prompt_attention(q, k, v, want, cu, cu, 0.125)
    hq = q.transpose(0, 1).contiguous().transpose(0, 1)
    wide = torch.full((217, 9, 64), 5.0, dtype=q.dtype, device='cuda')
    gaps = torch.zeros(217, 2, 80, dtype=q.dtype, device='cuda')
    gaps[:, :, :64] = k
    ext.prompt_attention(hq, gaps[:, :, :64], v.transpose(0, 1).contiguous().transpose(0, 1), wide[:, 1:7], cu, cu, 0.125)
    assert torch.equal(wide[:, 1:7], want)
    assert bool((wide[:, 0] == 5).all() and (wide[:, 7:] == 5).all())


@pytest.mark.parametrize('tokens', [True, False])
@pytest.mark.parametrize('behind', [2, 40])
def test_prompt_attention_neighbours_and_tails(ext, tokens, behind):
    """Rows before the first and behind the last sequence hold NaN and stay as they are; a neighbour's NaN and
    infinities reach no other sequence: the others' bits are those of a call of the same sizes without any. (How many
    rows there are chooses between the kernels, so sizes are kept alike.)"""
    lk = [130, 61, 200]
    lq = [1, 1, 1] if tokens else lk
    q, k, v = _make(lq, lk, 4, 2, 'bf16', fused=False)
    cq, ck = _cu(lq) + 5, _cu(lk) + 5

    def padded(x, fill):
        return torch.cat([torch.full((n, *x.shape[1:]), fill, dtype=x.dtype, device='cuda') if n else x
                          for n in (5, 0, behind)])

    want, lse = torch.empty_like(padded(q, 0.0)), torch.empty(4, sum(lq) + 5 + behind, device='cuda')
    ext.prompt_attention(padded(q, 0.0), padded(k, 0.0), padded(v, 0.0), want, cq, ck, 0.2, lse=lse)
    end = 5 + sum(lq)
    _check(q, k, v, want[5:end], lse[:, 5:end], lq, lk, 0.2, True)

    nan = float('nan')
    q2, k2, v2 = padded(q, nan), padded(k, nan), padded(v, nan)
    a, b = int(ck[1]), int(ck[2])
    k2[a:b], v2[a:b] = nan, float('inf')  # the whole middle sequence
    out = torch.full_like(q2, 7.0)
    lse2 = torch.full((4, q2.size(0)), 7.0, device='cuda')
    ext.prompt_attention(q2, k2, v2, out, cq, ck, 0.2, lse=lse2)
    assert bool((out[:5] == 7).all() and (out[end:] == 7).all() and (lse2[:, :5] == 7).all() and (lse2[:, end:] == 7).all())
    for i in (0, 2):
        rows = slice(int(cq[i]), int(cq[i + 1]))
        assert torch.equal(out[rows], want[rows]) and torch.equal(lse2[:, rows], lse[:, rows])
    assert bool(out[int(cq[1]):int(cq[2])].isnan().all())
    assert ext.device_error() == 0


def test_prompt_attention_bad_offsets(ext):
    """Offsets out of range or out of order leave their sequences out and set the error bit."""
    q, k, v = _make([64, 64], [64, 64], 2, 2, 'fp16', fused=False)
    good = torch.empty_like(q)
    ext.prompt_attention(q, k, v, good, _cu([64, 64]), _cu([64, 64]), 0.1)
    ext.device_error()
    for cq, ck in (([0, 64, 200], [0, 64, 128]), ([0, 64, 128], [0, 64, 300]), ([0, 64, 10], [0, 64, 128]),
                   ([0, 64, 128], [0, 64, -5])):
        out = torch.full_like(q, 3.0)
        ext.prompt_attention(q, k, v, out, torch.tensor(cq, device='cuda'), torch.tensor(ck, device='cuda'), 0.1)
        assert ext.device_error() == 2
        assert torch.equal(out[:64], good[:64]) and bool((out[64:] == 3).all())


def test_prompt_attention_many_sequences(ext):
    """More sequences than one scan step of the item search, empty ones among them."""
    lens = [(i * 37) % 50 for i in range(100)]
    q, k, v = _make(lens, lens, 4, 4, 'fp16')
    out, lse = torch.empty(sum(lens), 4, 64, dtype=q.dtype, device='cuda'), torch.empty(4, sum(lens), device='cuda')
    ext.prompt_attention(q, k, v, out, _cu(lens), _cu(lens), 0.125, lse=lse)
    _check(q, k, v, out, lse, lens, lens, 0.125, True)


def test_prompt_attention_single_token_matches_decode_attention(ext):
    """The single-token form against decode_attention on the same cache: both are within the test's bound of the exact
    result, and the layout [heads, max_len, 64] of the decoder's cache is read in place."""
    g = torch.Generator(device='cuda').manual_seed(1)
    kc, vc = (torch.randn(20, 1500, 64, device='cuda', generator=g).half() for _ in range(2))
    q = torch.randn(20, 64, device='cuda', generator=g).half()
    out, lse = torch.empty(1, 20, 64, dtype=torch.float16, device='cuda'), torch.empty(20, 1, device='cuda')
    k, v = kc.transpose(0, 1), vc.transpose(0, 1)
    ext.prompt_attention(q[None], k, v, out, _cu([1]), _cu([1500]), 0.125, lse=lse)
    _check(q[None], k, v, out, lse, [1], [1500], 0.125, True)
    ref = torch.empty(1280, dtype=torch.float16, device='cuda')
    m, l, acc = (torch.empty(20 * 24 * n, device='cuda') for n in (1, 1, 64))
    ext.decode_attention(q.view(-1), kc, vc, ref, None, None, None, m, l, acc, 0.125)
    _check(q[None], k, v, ref.view(1, 20, 64), lse, [1], [1500], 0.125, True)


@pytest.mark.parametrize('lq,lk', [([200, 130], [200, 130]), ([1, 1], [900, 1300])])
def test_prompt_attention_captured_and_on_another_stream(ext, lq, lk):
    """Captured; then replayed with other contents and other lengths. And on a side stream."""
    q, k, v = _make(lq, lk, 8, 2, 'fp16', fused=False)
    cq, ck = _cu(lq), _cu(lk)
    out, lse = torch.empty_like(q), torch.empty(8, sum(lq), device='cuda')
    ws = torch.empty(max(16, ext.prompt_attention_workspace(sum(lq), sum(lk), 2, 8, 2)), dtype=torch.uint8, device='cuda')
    ext.prompt_attention(q, k, v, out, cq, ck, 0.125, lse=lse, ws=ws)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ext.prompt_attention(q, k, v, out, cq, ck, 0.125, lse=lse, ws=ws)
    a, b, c = _make(lq, lk, 8, 2, 'fp16', seed=5, fused=False)
    q.copy_(a), k.copy_(b), v.copy_(c)
    other = [lk[1] + 7, lk[0] - 7]
    ck.copy_(_cu(other))
    if lq == lk:
        cq.copy_(_cu(other))
    graph.replay()
    _check(q, k, v, out, lse, other if lq == lk else lq, other, 0.125, True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = torch.empty_like(out)
        ext.prompt_attention(q, k, v, again, cq, ck, 0.125)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(out, again)


def test_prompt_attention_nothing_to_do(ext):
    q = torch.empty(0, 4, 64, dtype=torch.float16, device='cuda')
    ext.prompt_attention(q, q, q, q, _cu([]), _cu([]), 0.1)
    ext.prompt_attention(q, q, q, q, _cu([0, 0]), _cu([0, 0]), 0.1)
    x, out = torch.randn(3, 4, 64, device='cuda').half(), torch.ones(3, 4, 64, device='cuda').half()
    ext.prompt_attention(x, q, q, out, _cu([3]), _cu([0]), 0.1)
    assert not out.any()
    assert ext.device_error() == 0
