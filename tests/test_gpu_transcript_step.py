"""The whole-transcript operators run together as a training step of a one-layer decoder uses them: embedding, causal
attention over the packed transcripts, cross entropy over the tied matrix, and back; against the same step in 64 bits.

h = E[ids] + P[pos], a = attention(h as q, k and v, causal), x = h + a, loss = mean cross entropy of x E^T. Every 16-bit
tensor that the step hands from one operator to the next is one rounding (u = finfo.eps / 2 of its values) and each
operator's own result is within a few u of its magnitudes (see their tests); the gradient of the tied table is the sum of
two operators' results, each of which is rounded twice on the way. So the 2-norm of each result's error is held to 8 u
of its norm: at most 8 roundings lie on the longest path from the loss to a gradient (x, dx, p, ds, dq + dk + dv in
two sums, the table's two)."""

import pytest
import torch

pytestmark = pytest.mark.gpu

VOCAB, HEADS, POS = 1000, 4, 64
HIDDEN = 64 * HEADS
LENS = [40, 1, 64, 23]


def _step(ext, table, pos, ids, at, targets, cu):
    n = ids.numel()
    t, dev = table.dtype, table.device
    h = torch.empty(n, HIDDEN, dtype=t, device=dev)
    ext.embed_scaled(table, ids, h, scale=4.0, pos_embed=pos, positions=at)
    q = h.view(n, HEADS, 64)
    a, lse = torch.empty_like(q), torch.empty(HEADS, n, device=dev)
    ext.prompt_attention(q, q, q, a, cu, cu, 0.125, lse=lse)
    x = h + a.view(n, HIDDEN)
    loss, norm = torch.empty(n, device=dev), torch.empty(n, device=dev)
    ext.lm_head_loss(x, table, targets, loss, norm)
    kept = (targets != -100).float()
    g = kept / kept.sum()
    dx, dtable = torch.empty_like(x), torch.empty_like(table)
    ext.lm_head_loss_grad(x, table, targets, norm, g, dx, dtable)
    dq, dk, dv = (torch.empty_like(q) for _ in range(3))
    ext.prompt_attention_grad(q, q, q, a, dx.view(n, HEADS, 64), lse, cu, cu, 0.125, dq, dk, dv)
    dh = (dx.float() + (dq.float() + dk.float() + dv.float()).view(n, HIDDEN)).to(t)
    ext.embed_grad(dh, ids, dtable, scale=4.0, accumulate=True)
    dpos = torch.empty_like(pos)
    ext.embed_grad(dh, at, dpos)
    return loss, dtable, dpos


def _exact(table, pos, ids, at, targets):
    table, pos = table.double().requires_grad_(), pos.double().requires_grad_()
    h = table[ids] * 4.0 + pos[at]
    parts, first = [], 0
    for n in LENS:
        q = h[first:first + n].view(n, HEADS, 64).transpose(0, 1)
        s = (q @ q.transpose(1, 2) * 0.125).masked_fill(
            torch.ones(n, n, dtype=torch.bool, device='cuda').triu(1), float('-inf'))
        parts.append((torch.softmax(s, 2) @ q).transpose(0, 1).reshape(n, HIDDEN))
        first += n
    x = h + torch.cat(parts)
    loss = torch.nn.functional.cross_entropy(x @ table.T, targets, ignore_index=-100, reduction='none')
    (loss.sum() / (targets != -100).sum()).backward()
    return loss.detach(), table.grad, pos.grad


@pytest.mark.parametrize('t', [torch.float16, torch.bfloat16])
def test_training_step(ext, t):
    g = torch.Generator(device='cuda').manual_seed(2)
    table = (torch.randn(VOCAB, HIDDEN, device='cuda', generator=g) * 0.1).to(t)
    pos = (torch.randn(POS, HIDDEN, device='cuda', generator=g) * 0.1).to(t)
    n = sum(LENS)
    ids = torch.randint(VOCAB, (n,), device='cuda', generator=g)
    at = torch.cat([torch.arange(x, device='cuda') for x in LENS])
    targets = torch.randint(VOCAB, (n,), device='cuda', generator=g)
    targets[::7] = -100
    cu = torch.tensor([0] + LENS, device='cuda').cumsum(0)
    got = _step(ext, table, pos, ids, at, targets, cu)
    assert ext.device_error() == 0
    u = torch.finfo(t).eps / 2
    for have, want, name in zip(got, _exact(table, pos, ids, at, targets), ('loss', 'table', 'positions')):
        off = float((have.double() - want).norm() / want.norm())
        assert off <= 8 * u, f'{name}: {off / u} half steps'


def test_training_step_captured(ext):
    """The whole step as one CUDA graph (scratch from the graph's pool), replayed on new tokens."""
    g = torch.Generator(device='cuda').manual_seed(3)
    table = (torch.randn(VOCAB, HIDDEN, device='cuda', generator=g) * 0.1).half()
    pos = (torch.randn(POS, HIDDEN, device='cuda', generator=g) * 0.1).half()
    n = sum(LENS)
    ids, targets = (torch.randint(VOCAB, (n,), device='cuda', generator=g) for _ in range(2))
    at = torch.cat([torch.arange(x, device='cuda') for x in LENS])
    cu = torch.tensor([0] + LENS, device='cuda').cumsum(0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _step(ext, table, pos, ids, at, targets, cu)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = _step(ext, table, pos, ids, at, targets, cu)
    for x in (ids, targets):
        x.copy_(torch.randint(VOCAB, (n,), device='cuda', generator=g))
    graph.replay()
    want = _step(ext, table, pos, ids, at, targets, cu)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
