"""Embedding of whole transcripts and its gradient (fw_embed_scaled, fw_embed_grad) against 64-bit sums.

Tolerances: the result is rounded once to its type T (half a step, finfo.eps / 2 of the value, or half the smallest
subnormal) from fp32 arithmetic. A sum of m terms in fp32 is off by at most m * 2^-24 * sum |x| (m - 1 additions of
relative error 2^-24 each, plus the scale's product), which is computed per element in 64 bits.
"""

import pytest
import torch

pytestmark = pytest.mark.gpu
TYPES = {'fp16': torch.float16, 'bf16': torch.bfloat16, 'fp32': torch.float32}


def _half_step(t):
    info = torch.finfo(t)
    return info.eps / 2, info.smallest_normal * info.eps / 2


def _close(got, want, err32):
    """|got - want| within one rounding of `want` after an fp32 error of err32."""
    rel, tiny = _half_step(got.dtype)
    bound = (want.abs() + err32) * rel + err32 + tiny
    off = (got.double() - want).abs()
    assert bool((off <= bound).all()), f'{float((off - bound).max())} beyond the bound'


def _gen(seed):
    return torch.Generator(device='cuda').manual_seed(seed)


@pytest.mark.parametrize('n,vocab,hidden,max_pos,scale,dtype', [
    (1, 7, 8, 0, 1.0, 'fp16'), (4, 51866, 1280, 448, 1.0, 'fp16'), (449, 51865, 1280, 448, 35.777, 'bf16'),
    (1201, 300, 80, 100, 8.944, 'fp32'), (33, 101, 7, 0, 2.5, 'fp16'), (70, 50, 1001, 9, 1.0, 'bf16'),
    (5, 3, 1, 2, 0.0, 'fp32'), (2000, 1000, 2049, 0, -1.5, 'fp32'), (0, 10, 64, 0, 1.0, 'fp16')])
def test_embed_scaled(ext, n, vocab, hidden, max_pos, scale, dtype):
    t, g = TYPES[dtype], _gen(n + hidden)
    embed = torch.randn(vocab, hidden, device='cuda', generator=g).to(t)
    ids = torch.randint(vocab, (n,), device='cuda', generator=g)
    pos = at = None
    want = embed.double()[ids] * torch.tensor(scale, dtype=torch.float32).double().item()
    err = want.abs()
    if max_pos:
        pos = torch.randn(max_pos, hidden, device='cuda', generator=g).to(t)
        at = torch.randint(max_pos, (n,), device='cuda', generator=g)
        want = want + pos.double()[at]
        err = err + pos.double()[at].abs()
    out = torch.full((n, hidden), float('nan'), dtype=t, device='cuda')
    ext.embed_scaled(embed, ids, out, scale=scale, pos_embed=pos, positions=at)
    _close(out, want, err * 2.0 ** -23)
    assert ext.device_error() == 0


def test_embed_scaled_matches_embed_pos(ext):
    """With scale 1 it is embed_pos: the same sums, the same rounding."""
    g = _gen(3)
    embed = torch.randn(500, 1280, device='cuda', generator=g).half()
    pos = torch.randn(448, 1280, device='cuda', generator=g).half()
    ids, at = (torch.randint(k, (97,), device='cuda', generator=g) for k in (500, 448))
    a, b = (torch.empty(97, 1280, dtype=torch.float16, device='cuda') for _ in range(2))
    ext.embed_pos(embed, pos, ids, at, a)
    ext.embed_scaled(embed, ids, b, pos_embed=pos, positions=at)
    assert torch.equal(a, b)


def test_embed_scaled_unaligned_views(ext):
    """Tables and outputs that do not start on 16 bytes take the element-wise path."""
    g = _gen(4)
    store = torch.randn(1 + 60 * 64, device='cuda', generator=g).half()
    embed = store[1:].view(60, 64)
    ids = torch.randint(60, (31,), device='cuda', generator=g)
    out = torch.empty(1 + 31 * 64, dtype=torch.float16, device='cuda')[1:].view(31, 64)
    ext.embed_scaled(embed, ids, out, scale=3.0)
    assert torch.equal(out, (embed[ids].float() * 3.0).half())


def test_embed_scaled_flags_bad_ids(ext):
    from flash_whisper_b200._lib import lib  # noqa: F401
    ext.device_error()
    embed = torch.randn(10, 64, device='cuda').half()
    out = torch.empty(3, 64, dtype=torch.float16, device='cuda')
    ext.embed_scaled(embed, torch.tensor([-1, 4, 10], device='cuda'), out)
    assert ext.device_error() == 2
    assert torch.equal(out, embed[[0, 4, 9]])


def _grad(dout, ids, vocab, scale, padding, base=None):
    keep = (ids != padding) & (ids >= 0) & (ids < vocab)
    rows, at = dout[keep].double() * scale, ids[keep]
    want = torch.zeros(vocab, dout.size(1), dtype=torch.float64, device='cuda')
    size = torch.zeros_like(want)
    want.index_put_((at,), rows, accumulate=True)
    size.index_put_((at,), rows.abs(), accumulate=True)
    terms = torch.bincount(at, minlength=vocab)[:, None] + 2
    if base is not None:
        want, size = want + base.double(), size + base.double().abs()
    return want, size * terms * 2.0 ** -24


CASES = [  # n, vocab, hidden, scale, padding, dtype, ids
    (1, 7, 8, 1.0, -1, 'fp16', 'uniform'), (27, 51866, 1280, 1.0, -1, 'fp16', 'zipf'),
    (3584, 51866, 1280, 1.0, 50257, 'fp16', 'zipf'), (2048, 300, 80, 8.944, 5, 'bf16', 'uniform'),
    (2049, 300, 80, 8.944, -1, 'fp32', 'uniform'), (9001, 65536, 64, 0.5, 0, 'bf16', 'zipf'),
    (8192, 255, 48, 1.0, -1, 'fp32', 'one'), (8193, 70000, 24, 1.0, -1, 'fp32', 'zipf'),
    (333, 256, 7, 2.0, 255, 'fp16', 'uniform'), (5000, 17, 1001, 1.0, -1, 'bf16', 'uniform'),
    (32749, 51866, 128, 11.314, -1, 'bf16', 'zipf'), (700, 1, 8, 1.0, -1, 'fp32', 'uniform'),
    (640, 9, 8, 1.0, 3, 'fp32', 'padding'), (0, 33, 16, 1.0, -1, 'fp16', 'uniform')]


def _ids(kind, n, vocab, padding, g):
    if kind == 'uniform':
        return torch.randint(vocab, (n,), device='cuda', generator=g)
    if kind in ('one', 'padding'):
        return torch.full((n,), padding if kind == 'padding' else vocab - 1, device='cuda', dtype=torch.long)
    u = torch.rand(n, device='cuda', generator=g)
    return (torch.exp(u * torch.log(torch.tensor(float(vocab)))).long().clamp(1, vocab) - 1) * 7919 % vocab


@pytest.mark.parametrize('accumulate', [False, True])
@pytest.mark.parametrize('n,vocab,hidden,scale,padding,dtype,kind', CASES)
def test_embed_grad(ext, n, vocab, hidden, scale, padding, dtype, kind, accumulate):
    t, g = TYPES[dtype], _gen(n + vocab)
    ids = _ids(kind, n, vocab, padding, g)
    dout = torch.randn(n, hidden, device='cuda', generator=g).to(t)
    scale = torch.tensor(scale, dtype=torch.float32).double().item()
    base = torch.randn(vocab, hidden, device='cuda', generator=g).to(t) if accumulate else None
    want, err = _grad(dout, ids, vocab, scale, padding, base)
    got = base.clone() if accumulate else torch.full((vocab, hidden), float('nan'), dtype=t, device='cuda')
    ext.embed_grad(dout, ids, got, scale=scale, padding_idx=padding, accumulate=accumulate)
    _close(got, want, err)
    again = base.clone() if accumulate else torch.empty_like(got)
    ext.embed_grad(dout, ids, again, scale=scale, padding_idx=padding, accumulate=accumulate)
    assert torch.equal(got, again), 'two runs differ'
    assert ext.device_error() == 0


def test_embed_grad_accumulates_positions_and_leaves_other_rows(ext):
    """The position table's gradient (ids = positions), added in place; rows that are not named keep their bits, NaN
    among them."""
    g = _gen(9)
    at = torch.arange(300, device='cuda') % 100
    dout = torch.randn(300, 64, device='cuda', generator=g)
    dpos = torch.full((448, 64), float('nan'), device='cuda')
    dpos[:100] = 1.0
    ext.embed_grad(dout, at, dpos, accumulate=True)
    assert bool(dpos[100:].isnan().all())
    want, err = _grad(dout, at, 448, 1.0, -1, torch.ones(448, 64, device='cuda'))
    _close(dpos[:100], want[:100], err[:100])


def test_embed_grad_unaligned_rows(ext):
    g = _gen(10)
    dout = torch.randn(1 + 50 * 64, device='cuda', generator=g).half()[1:].view(50, 64)
    ids = torch.randint(20, (50,), device='cuda', generator=g)
    got = torch.full((1 + 23 * 64,), 7.0, dtype=torch.float16, device='cuda')
    ext.embed_grad(dout, ids, got[1:].view(23, 64))
    want, err = _grad(dout, ids, 23, 1.0, -1)
    _close(got[1:].view(23, 64), want, err)
    assert float(got[0]) == 7.0


def test_embed_grad_flags_and_skips_bad_ids(ext):
    ext.device_error()
    ids = torch.tensor([0, -5, 3, 10, 3], device='cuda')
    dout = torch.ones(5, 16, device='cuda')
    got = torch.empty(10, 16, device='cuda')
    ext.embed_grad(dout, ids, got)
    assert ext.device_error() == 2
    assert got.sum(1).tolist() == [16.0, 0, 0, 32.0, 0, 0, 0, 0, 0, 0]
    ext.embed_grad(dout, torch.tensor([0, -100, 3, -100, 3], device='cuda'), got, padding_idx=-100)
    assert ext.device_error() == 0  # a padding id outside the vocabulary is no mistake


def test_embed_grad_is_the_derivative(ext):
    """Differences of a linear functional of the forward pass: exact up to fp32 rounding, as the map is linear."""
    g = _gen(11)
    embed = torch.randn(40, 24, device='cuda', generator=g)
    ids = torch.randint(40, (90,), device='cuda', generator=g)
    dout = torch.randn(90, 24, device='cuda', generator=g)
    step = torch.randn(40, 24, device='cuda', generator=g)
    a, b, grad = torch.empty(90, 24, device='cuda'), torch.empty(90, 24, device='cuda'), torch.empty_like(embed)
    ext.embed_scaled(embed, ids, a, scale=3.0)
    ext.embed_scaled(embed + step, ids, b, scale=3.0)
    ext.embed_grad(dout, ids, grad, scale=3.0)
    diff = ((b.double() - a.double()) * dout.double()).sum()
    assert abs(float(diff - (grad.double() * step.double()).sum())) <= 90 * 24 * 3 * 4 * 4 * 2.0 ** -22


def test_embed_captured_and_on_another_stream(ext):
    """Captured with a caller's workspace and replayed on new contents; and called on a side stream."""
    g = _gen(12)
    ids = torch.randint(500, (3000,), device='cuda', generator=g)
    dout = torch.randn(3000, 64, device='cuda', generator=g).half()
    got = torch.empty(500, 64, dtype=torch.float16, device='cuda')
    ws = torch.empty(ext.embed_grad_workspace(3000, 64), dtype=torch.uint8, device='cuda')
    ext.embed_grad(dout, ids, got, ws=ws)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ext.embed_grad(dout, ids, got, ws=ws)
    ids.copy_(torch.randint(500, (3000,), device='cuda', generator=g))
    dout.normal_(generator=g)
    graph.replay()
    want, err = _grad(dout, ids, 500, 1.0, -1)
    _close(got, want, err)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = torch.empty_like(got)
        ext.embed_grad(dout, ids, other)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other, got)
