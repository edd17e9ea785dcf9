"""Whole-transcript operators at the edges of their range: tensors past 2^31 elements, calls that overlap on two
streams, workspaces of exactly the asked size with guard bytes behind them, and the sizes at which one kernel takes over
from another."""

import pytest
import torch

from tests.test_gpu_embed import _close, _grad
from tests.test_gpu_loss import _check_grad as _check_loss_grad
from tests.test_gpu_loss import _inputs, _logit_error, _want
from tests.test_gpu_prompt import _check, _cu, _make
from tests.test_gpu_prompt_grad import _check_grad

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('lq,causal', [([1, 1], True), ([200, 300], True), ([40, 150], False)])
def test_prompt_attention_far_into_a_long_cache(ext, lq, causal):
    """Heads-first caches of 8 x 5,000,000 rows (2.56e9 elements): rows and heads whose offsets pass 32 bits."""
    rows, heads, lk = 5_000_000, 8, [333, 1001]
    first = [4_000_037, 4_998_000]
    cache = torch.empty(2, heads, rows, 64, dtype=torch.float16, device='cuda')
    q, k, v = _make(lq, lk, heads, heads, 'fp16', fused=False)
    at = 0
    for a, n in zip(first, lk):
        cache[0, :, a:a + n] = k[at:at + n].transpose(0, 1)
        cache[1, :, a:a + n] = v[at:at + n].transpose(0, 1)
        at += n
    # the sequences' rows do not follow one another in the cache: one call for each
    out, lse = torch.empty_like(q), torch.empty(heads, sum(lq), device='cuda')
    kc, vc = cache[0].transpose(0, 1), cache[1].transpose(0, 1)
    at = 0
    for i, (a, n) in enumerate(zip(first, lk)):
        part = slice(at, at + lq[i])
        o, l = torch.empty_like(q[part]), torch.empty(heads, lq[i], device='cuda')
        ext.prompt_attention(q[part], kc, vc, o, _cu([lq[i]]), torch.tensor([a, a + n], device='cuda'), 0.125,
                             causal=causal, lse=l)
        out[part], lse[:, part] = o, l
        at += lq[i]
    assert ext.device_error() == 0
    _check(q, k, v, out, lse, lq, lk, 0.125, causal)
    if lq[0] == 1:
        return
    dout = torch.randn(q.shape, device='cuda').half()
    dcache = torch.empty_like(cache)
    grads = [torch.empty_like(x) for x in (q, k, v)]
    at = ak = 0
    for i, (a, n) in enumerate(zip(first, lk)):
        part = slice(at, at + lq[i])
        dcache[:, :, a - 3:a] = 7.0
        dcache[:, :, a + n:a + n + 3] = 7.0
        ext.prompt_attention_grad(q[part], kc, vc, out[part], dout[part], lse[:, part].contiguous(), _cu([lq[i]]),
                                  torch.tensor([a, a + n], device='cuda'), 0.125, grads[0][part],
                                  dcache[0].transpose(0, 1), dcache[1].transpose(0, 1), causal=causal)
        grads[1][ak:ak + n], grads[2][ak:ak + n] = (dcache[j, :, a:a + n].transpose(0, 1) for j in (0, 1))
        assert bool((dcache[:, :, a - 3:a] == 7).all() and (dcache[:, :, a + n:a + n + 3] == 7).all())
        at, ak = at + lq[i], ak + n
    _check_grad(q, k, v, dout, grads, lq, lk, 0.125, causal)


def test_embedding_tables_past_32_bits(ext):
    """A table of 1,700,000 x 1280 (2.18e9 elements): lookup and dense gradient of rows at its end."""
    vocab, hidden, n = 1_700_000, 1280, 777
    table = torch.zeros(vocab, hidden, dtype=torch.bfloat16, device='cuda')
    ids = vocab - 1 - torch.randint(300, (n,), device='cuda')
    table[-300:] = torch.randn(300, hidden, device='cuda')
    out = torch.empty(n, hidden, dtype=torch.bfloat16, device='cuda')
    ext.embed_scaled(table, ids, out, scale=2.0)
    assert torch.equal(out, (table[ids].float() * 2).bfloat16())
    got = torch.full_like(table, float('nan'))
    ext.embed_grad(out, ids, got)
    want, err = _grad(out, ids - (vocab - 300), 300, 1.0, -1)
    _close(got[-300:], want, err)
    assert not got[:-300].any()


def test_loss_over_a_matrix_past_32_bits(ext):
    """1,700,000 rows of 1280, zero but for the last 400: the zero rows each add exp(0), and get the gradient
    g exp(-lse) h."""
    vocab, hidden, n = 1_700_000, 1280, 5
    w = torch.zeros(vocab, hidden, dtype=torch.float16, device='cuda')
    w[-400:] = torch.randn(400, hidden, device='cuda') * 0.1
    h = torch.randn(n, hidden, device='cuda').half()
    targets = vocab - 1 - torch.arange(n, device='cuda') * 7
    loss, lse = torch.empty(n, device='cuda'), torch.empty(n, device='cuda')
    ext.lm_head_loss(h, w, targets, loss, lse)
    z = h.double() @ w[-400:].double().T
    want = torch.log(torch.exp(z).sum(1) + (vocab - 400))
    err = _logit_error(h, w[-400:])
    assert bool(((lse.double() - want).abs() <= err).all())
    at = z.gather(1, (targets - (vocab - 400))[:, None])[:, 0]
    assert bool(((loss.double() - (want - at)).abs() <= 2 * err).all())
    g = torch.rand(n, device='cuda') + 0.5
    dh, dw = torch.empty_like(h), torch.empty_like(w)
    ext.lm_head_loss_grad(h, w, targets, lse, g, dh, dw)
    dz = torch.exp(z - want[:, None])
    dz[torch.arange(n), targets - (vocab - 400)] -= 1.0
    dz *= g.double()[:, None]
    exact = dz.T @ h.double()
    # roundings of p - [t], of the scaled copy of h and of the result, over magnitudes; fp16 subnormals (2^-25) of all
    size = dz.abs().T @ h.double().abs()
    assert bool(((dw[-400:].double() - exact).abs() <= 4 * 2.0 ** -11 * size + 2.0 ** -24).all())
    zero = (g.double() * torch.exp(-want)) @ h.double()
    assert bool(((dw[:-400:9973].double() - zero).abs() <= 2.0 ** -24 + 4 * 2.0 ** -11 * zero.abs()).all())


@pytest.mark.parametrize('rows,kv_heads,group', [(8, 2, 1), (9, 2, 1), (2, 2, 4), (3, 2, 4), (1, 3, 8), (1, 2, 9), (4, 5, 2)])
def test_prompt_attention_around_the_few_rows_rule(ext, rows, kv_heads, group):
    """Row counts on both sides of the rule by which single tokens leave the tensor core, one sequence far longer in
    queries than the average, and one without any."""
    lq = [rows] * 6 + [0, rows * 7 if rows > 1 else 1]
    lk = [n + 150 for n in lq]
    for i in range(2):
        lens_q = lq if i == 0 else [0] * 7 + [sum(lq)]
        lens_k = lk if i == 0 else [70] * 7 + [sum(lq) + 900]
        q, k, v = _make(lens_q, lens_k, kv_heads * group, kv_heads, 'bf16', fused=False)
        out, lse = torch.empty_like(q), torch.empty(q.size(1), q.size(0), device='cuda')
        ext.prompt_attention(q, k, v, out, _cu(lens_q), _cu(lens_k), 0.15, lse=lse)
        _check(q, k, v, out, lse, lens_q, lens_k, 0.15, True)
        dout = torch.randn(q.shape, device='cuda').bfloat16()
        grads = [torch.empty_like(x) for x in (q, k, v)]
        ext.prompt_attention_grad(q, k, v, out, dout, lse, _cu(lens_q), _cu(lens_k), 0.15, *grads)
        _check_grad(q, k, v, dout, grads, lens_q, lens_k, 0.15, True)


def test_workspaces_of_exactly_the_asked_size(ext):
    """Guard bytes behind each operator's scratch stay as they are."""

    def scratch(need):
        ws = torch.full((need + 4096,), 0xA5, dtype=torch.uint8, device='cuda')
        return ws, ws[:need]

    guards = []
    ids, dout = torch.randint(500, (9000,), device='cuda'), torch.randn(9000, 72, device='cuda')
    full, ws = scratch(ext.embed_grad_workspace(9000, 72))
    ext.embed_grad(dout, ids, torch.empty(500, 72, device='cuda'), ws=ws)
    guards.append(full[ws.numel():])
    h, w, targets = _inputs(300, 5000, 136, 'fp16')
    loss, lse, g = (torch.rand(300, device='cuda') for _ in range(3))
    full, ws = scratch(ext.lm_head_loss_workspace(300, 5000))
    ext.lm_head_loss(h, w, targets, loss, lse, ws=ws)
    guards.append(full[ws.numel():])
    full, ws = scratch(ext.lm_head_loss_grad_workspace(300, 5000, 136))
    dh, dw = torch.empty_like(h), torch.empty_like(w)
    ext.lm_head_loss_grad(h, w, targets, lse, g, dh, dw, ws=ws)
    _check_loss_grad(h, w, targets, g, lse, dh, dw)
    guards.append(full[ws.numel():])
    for lq in ([1, 1, 2], [130, 1, 77]):
        lk = [700, 90, 4000]
        q, k, v = _make(lq, lk, 4, 2, 'fp16', fused=False)
        out, l = torch.empty_like(q), torch.empty(4, sum(lq), device='cuda')
        need = ext.prompt_attention_workspace(sum(lq), sum(lk), 3, 4, 2)
        full, ws = scratch(need)
        ext.prompt_attention(q, k, v, out, _cu(lq), _cu(lk), 0.125, lse=l, ws=ws)
        _check(q, k, v, out, l, lq, lk, 0.125, True)
        guards.append(full[need:])
        full, ws = scratch(ext.prompt_attention_grad_workspace(sum(lq), sum(lk), 3, 4, 2))
        ext.prompt_attention_grad(q, k, v, out, out, l, _cu(lq), _cu(lk), 0.125, *(torch.empty_like(x) for x in (q, k, v)),
                                  ws=ws)
        guards.append(full[ws.numel():])
    assert all(bool((x == 0xA5).all()) for x in guards)


def test_calls_that_overlap_on_two_streams(ext):
    """Every operator on two streams at once, each call with scratch of its own: the bits of a call alone."""
    lens = [300, 77, 410]
    q, k, v = _make(lens, lens, 8, 2, 'bf16', fused=False)
    cu, n = _cu(lens), sum(lens)
    h, w, targets = _inputs(n, 9000, 512, 'bf16')
    ids = torch.randint(9000, (n,), device='cuda')
    g = torch.rand(n, device='cuda')

    def step():
        out, lse = torch.empty_like(q), torch.empty(8, n, device='cuda')
        ext.prompt_attention(q, k, v, out, cu, cu, 0.125, lse=lse)
        grads = [torch.empty_like(x) for x in (q, k, v)]
        ext.prompt_attention_grad(q, k, v, out, out, lse, cu, cu, 0.125, *grads)
        loss, norm = torch.empty(n, device='cuda'), torch.empty(n, device='cuda')
        ext.lm_head_loss(h, w, targets, loss, norm)
        dh, dw = torch.empty_like(h), torch.empty_like(w)
        ext.lm_head_loss_grad(h, w, targets, norm, g, dh, dw)
        table = torch.empty_like(w)
        ext.embed_grad(dh, ids, table, scale=3.0)
        return [out, lse, *grads, loss, norm, dh, dw, table]

    want = step()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [None, None]
    for _ in range(3):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i] = step()
    torch.cuda.synchronize()
    assert ext.device_error() == 0
    for have in got:
        assert all(torch.equal(a, b) for a, b in zip(want, have))


def test_loss_forward_with_every_target_and_width(ext):
    """Targets in every column of a narrow matrix whose last tile is cut at each width in turn."""
    for vocab in (1, 31, 32, 33, 127, 128, 129, 255, 257, 383, 385):
        h, w, _ = _inputs(vocab, vocab, 64, 'fp16', lean=0.0)
        targets = torch.arange(vocab, device='cuda')
        loss, lse = torch.empty(vocab, device='cuda'), torch.empty(vocab, device='cuda')
        ext.lm_head_loss(h, w, targets, loss, lse)
        want_loss, want_lse, _, _ = _want(h, w, targets)
        err = _logit_error(h, w)
        assert bool(((lse.double() - want_lse).abs() <= err).all() and ((loss.double() - want_loss).abs() <= 2 * err).all())


@pytest.mark.parametrize('singles,longer,group', [(127, [600], 1), (70, [65, 64, 300], 1), (300, [17, 16, 900], 4),
                                                  (8, [64], 1), (400, [300, 33, 32], 1), (90, [3, 2, 16, 17], 2)])
@pytest.mark.parametrize('kv_heads', [2, 20])
def test_prompt_attention_prompts_among_single_tokens(ext, singles, longer, group, kv_heads):
    """Few rows on average, some sequences with many: on both sides of the length that tiles take over."""
    lq = [1] * singles
    for i, n in enumerate(longer):
        lq.insert((37 * i + 5) % singles, n)
    lk = [n + (53 * i) % 400 for i, n in enumerate(lq)]
    q, k, v = _make(lq, lk, kv_heads * group, kv_heads, 'fp16', fused=False)
    out, lse = torch.full_like(q, float('nan')), torch.full((q.size(1), q.size(0)), float('nan'), device='cuda')
    ext.prompt_attention(q, k, v, out, _cu(lq), _cu(lk), 0.15, lse=lse)
    assert ext.device_error() == 0
    if kv_heads == 20:  # every head is alike: check four of them
        heads = [0, 7 * group, 13 * group + group - 1, 20 * group - 1]
        keep = [h // group for h in heads]
        q, k, v, out, lse = q[:, heads], k[:, keep], v[:, keep], out[:, heads], lse[heads]
    _check(q, k, v, out, lse, lq, lk, 0.15, True)


def test_prompt_attention_masked_keys_of_any_finite_size(ext):
    """What a later key holds reaches no earlier query, however large it is."""
    q, k, v = _make([200], [200], 2, 2, 'bf16', fused=False)
    outs = []
    for fill in (1.0, torch.finfo(torch.bfloat16).max):
        v[100:] = fill
        k[100:] = fill if fill == 1.0 else 1e30
        out = torch.empty_like(q)
        ext.prompt_attention(q, k, v, out, _cu([200]), _cu([200]), 0.125)
        outs.append(out)
    assert torch.equal(outs[0][:100], outs[1][:100])


@pytest.mark.parametrize('lq,group', [([2] * 5 + [0], 1), ([3] * 5, 1), ([1] * 6, 2), ([1] * 6, 3), ([1, 0, 5, 0, 1, 1], 1),
                                      ([2, 2, 3, 2, 1], 1), ([1], 1), ([1, 1], 1)])
@pytest.mark.parametrize('dtype', ['fp16', 'bf16'])
def test_prompt_attention_of_one_to_three_rows(ext, lq, group, dtype):
    """On both sides of two rows; keys from none to several tiles of 32, cut anywhere by the warps and splits."""
    for base in (0, 1, 31, 33, 260, 1500):
        lk = [base + 13 * i if base else max(n - 1, 0) for i, n in enumerate(lq)]
        q, k, v = _make(lq, lk, 3 * group, 3, dtype, fused=False)
        out, lse = torch.full_like(q, float('nan')), torch.full((q.size(1), q.size(0)), float('nan'), device='cuda')
        ext.prompt_attention(q, k, v, out, _cu(lq), _cu(lk), 0.2, lse=lse)
        assert ext.device_error() == 0
        _check(q, k, v, out, lse, lq, lk, 0.2, True)


@pytest.mark.parametrize('n,vocab,hidden', [(300, 5000, 136), (300, 5000, 128), (2000, 40001, 64), (2000, 40001, 72),
                                            (1, 33, 64), (65, 200, 192)])
def test_loss_grad_with_scratch_of_nan(ext, n, vocab, hidden):
    """Whole and cut chunks of 64, several pieces and splits; the scratch holds NaN before the call."""
    h, w, targets = _inputs(n, vocab, hidden, 'bf16', seed=3)
    loss, lse = torch.empty(n, device='cuda'), torch.empty(n, device='cuda')
    ext.lm_head_loss(h, w, targets, loss, lse,
                     ws=torch.full((ext.lm_head_loss_workspace(n, vocab),), 255, dtype=torch.uint8, device='cuda'))
    assert bool(((lse.double() - _want(h, w, targets)[1]).abs() <= _logit_error(h, w)).all())
    g = torch.rand(n, device='cuda')
    dh, dw = torch.full_like(h, float('nan')), torch.full_like(w, float('nan'))
    ws = torch.full((ext.lm_head_loss_grad_workspace(n, vocab, hidden),), 255, dtype=torch.uint8, device='cuda')
    ext.lm_head_loss_grad(h, w, targets, lse, g, dh, dw, ws=ws)
    assert ext.device_error() == 0
    _check_loss_grad(h, w, targets, g, lse, dh, dw)


@pytest.mark.parametrize('lq,lk', [([1, 1], [3000, 700]), ([5, 130, 0], [900, 131, 40]), ([300, 1], [300, 1])])
@pytest.mark.parametrize('dtype', ['fp16', 'bf16'])
def test_prompt_attention_with_scratch_of_nan(ext, lq, lk, dtype):
    q, k, v = _make(lq, lk, 4, 2, dtype, fused=False)
    out, lse = torch.full_like(q, float('nan')), torch.empty(4, sum(lq), device='cuda')
    sizes = (sum(lq), sum(lk), len(lq), 4, 2)
    ws = torch.full((ext.prompt_attention_workspace(*sizes) + 16,), 255, dtype=torch.uint8, device='cuda')
    ext.prompt_attention(q, k, v, out, _cu(lq), _cu(lk), 0.125, lse=lse, ws=ws)
    _check(q, k, v, out, lse, lq, lk, 0.125, True)
    dout = torch.randn(q.shape, device='cuda').to(q.dtype)
    grads = [torch.full_like(x, float('nan')) for x in (q, k, v)]
    ws = torch.full((ext.prompt_attention_grad_workspace(*sizes),), 255, dtype=torch.uint8, device='cuda')
    ext.prompt_attention_grad(q, k, v, out, dout, lse, _cu(lq), _cu(lk), 0.125, *grads, ws=ws)
    assert ext.device_error() == 0
    _check_grad(q, k, v, dout, grads, lq, lk, 0.125, True)


def test_embed_grad_with_scratch_of_nan(ext):
    for n in (1, 40, 9000):
        ids, dout = torch.randint(300, (n,), device='cuda'), torch.randn(n, 72, device='cuda')
        ws = torch.full((ext.embed_grad_workspace(n, 72),), 255, dtype=torch.uint8, device='cuda')
        got, again = (torch.full((300, 72), float('nan'), device='cuda') for _ in range(2))
        ext.embed_grad(dout, ids, got, ws=ws)
        ext.embed_grad(dout, ids, again)
        want = torch.zeros(300, 72, dtype=torch.float64, device='cuda').index_add_(0, ids, dout.double())
        # n additions in fp32 at most, each off by half a step of the sum of magnitudes
        size = torch.zeros(300, 72, dtype=torch.float64, device='cuda').index_add_(0, ids, dout.double().abs())
        assert torch.equal(got, again) and bool(((got.double() - want).abs() <= n * 2.0 ** -24 * size).all())


@pytest.mark.parametrize('lq,lk', [([1] * 60 + [200], [300] * 61), ([1] * 9 + [70], [5000] * 10)])
def test_prompt_among_single_tokens_captured_and_replayed(ext, lq, lk):
    """Both launches (and the join of the key splits) in a graph, replayed over new contents."""
    q, k, v = _make(lq, lk, 1, 1, 'fp16', fused=False)
    cu_q, cu_k, out = _cu(lq), _cu(lk), torch.empty_like(q)
    lse = torch.empty(1, sum(lq), device='cuda')
    ws = torch.empty(ext.prompt_attention_workspace(sum(lq), sum(lk), len(lq), 1, 1) + 16, dtype=torch.uint8,
                     device='cuda')

    def step():
        ext.prompt_attention(q, k, v, out, cu_q, cu_k, 0.125, lse=lse, ws=ws)

    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
        step()
    for seed in (1, 2):
        for x, y in zip((q, k, v), _make(lq, lk, 1, 1, 'fp16', seed=seed, fused=False)):
            x.copy_(y)
        out.fill_(float('nan'))
        graph.replay()
        _check(q, k, v, out, lse, lq, lk, 0.125, True)
    assert ext.device_error() == 0
