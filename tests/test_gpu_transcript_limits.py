"""Whole-transcript operators where their promises end: long walks beside other work, offsets that are wrong in the middle,
values near the ends of fp16. Tolerances are those of test_gpu_prompt.py, test_gpu_prompt_grad.py and test_gpu_loss.py."""

import pytest
import torch

from tests.test_gpu_loss import _check_grad as _check_loss_grad
from tests.test_gpu_loss import _inputs, _logit_error
from tests.test_gpu_prompt import _check, _cu, _make
from tests.test_gpu_prompt_grad import _check_grad, _run, _within

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('lens,heads,kv_heads,dtype', [([2048], 8, 1, 'fp16'), ([1000, 1500, 90], 4, 4, 'bf16')])
def test_prompt_attention_grad_long_walks_repeat_beside_other_work(ext, lens, heads, kv_heads, dtype):
    """Items of many steps, whose warps hand over to the products step by step, while another stream keeps the memory
    and the SMs busy: within the bounds, and the same bits in every run."""
    q, k, v = _make(lens, lens, heads, kv_heads, dtype)
    dout = torch.randn(q.shape, device='cuda').to(q.dtype)
    cu = _cu(lens)
    out, lse, want = _run(ext, q, k, v, dout, cu, cu, 0.125, True)
    _check_grad(q, k, v, dout, want, lens, lens, 0.125, True)
    side, big = torch.cuda.Stream(), torch.zeros(1 << 26, device='cuda')
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(8):
        with torch.cuda.stream(side):
            big.mul_(0.5).add_(1.0)
        grads = [torch.full(x.shape, float('nan'), dtype=x.dtype, device='cuda') for x in (q, k, v)]
        ext.prompt_attention_grad(q, k, v, out, dout, lse, cu, cu, 0.125, *grads)
        assert all(torch.equal(a, b) for a, b in zip(grads, want))
    torch.cuda.current_stream().wait_stream(side)
    assert ext.device_error() == 0


def _offsets(*x):
    return torch.tensor(x, device='cuda')


# (cu_q, cu_k, the sequences that stay good): a bad offset in front of good sequences, in either array
MIDDLE = [([0, 64, 3000, 128, 192], [0, 64, 128, 192, 256], [0, 3]), ([0, 64, 128, 192], [0, 70, 5000, 200], [0]),
          ([0, 3000, 3, 4], [0, 10, 20, 150], [2]), ([0, 64, 128, 128, 192], [0, 64, -1, 150, 256], [0, 3]),
          ([-7, 3, 40, 192], [0, 30, 90, 256], [1, 2]), ([5, 3, 9, 192], [0, 30, 90, 256], [1, 2])]


@pytest.mark.parametrize('cu_q,cu_k,good', MIDDLE)
@pytest.mark.parametrize('rows_k', [256, 4096])
@pytest.mark.parametrize('dtype', ['fp16', 'bf16'])
def test_prompt_attention_good_sequences_behind_bad_offsets(ext, cu_q, cu_k, good, rows_k, dtype):
    """Whether the keys are split and joined (as the rows of an average sequence suggest) or not: the good sequences are
    computed, the rows of the others stay."""
    rows_q, heads, kv_heads = 192, 4, 2
    q, k, v = _make([rows_q], [rows_k], heads, kv_heads, dtype, fused=False)
    assert (ext.prompt_attention_workspace(rows_q, rows_k, len(cu_q) - 1, heads, kv_heads) > 0) == (rows_k == 4096)
    out, lse = torch.full_like(q, 3.0), torch.full((heads, rows_q), 3.0, device='cuda')
    ws = torch.full((ext.prompt_attention_workspace(rows_q, rows_k, len(cu_q) - 1, heads, kv_heads) + 16,), 255,
                    dtype=torch.uint8, device='cuda')
    ext.device_error()
    ext.prompt_attention(q, k, v, out, _offsets(*cu_q), _offsets(*cu_k), 0.125, lse=lse, ws=ws)
    assert ext.device_error() == 2
    left = torch.ones(rows_q, dtype=torch.bool, device='cuda')
    for b in good:
        rq, rk = slice(cu_q[b], cu_q[b + 1]), slice(cu_k[b], cu_k[b + 1])
        _check(q[rq], k[rk], v[rk], out[rq], lse[:, rq], [rq.stop - rq.start], [rk.stop - rk.start], 0.125, True)
        left[rq] = False
    assert bool((out[left] == 3).all()) and bool((lse[:, left] == 3).all())


@pytest.mark.parametrize('cu_q,cu_k,good', MIDDLE)
@pytest.mark.parametrize('dtype', ['fp16', 'bf16'])
def test_prompt_attention_grad_good_sequences_behind_bad_offsets(ext, cu_q, cu_k, good, dtype):
    """As above, with scratch of NaN and with NaN in what belongs to no good sequence."""
    rows_q, rows_k, heads, kv_heads = 192, 256, 4, 2
    q, k, v = _make([rows_q], [rows_k], heads, kv_heads, dtype, fused=False)
    dout = torch.randn(q.shape, device='cuda').to(q.dtype)
    out, lse = torch.full_like(q, float('nan')), torch.full((heads, rows_q), float('nan'), device='cuda')
    spans = [(slice(cu_q[b], cu_q[b + 1]), slice(cu_k[b], cu_k[b + 1])) for b in good]
    no_q, no_k = (torch.ones(n, dtype=torch.bool, device='cuda') for n in (rows_q, rows_k))
    for rq, rk in spans:
        o, l = torch.empty_like(q[rq]), torch.empty(heads, rq.stop - rq.start, device='cuda')
        ext.prompt_attention(q[rq], k[rk], v[rk], o, _cu([o.size(0)]), _cu([rk.stop - rk.start]), 0.125, lse=l)
        out[rq], lse[:, rq] = o, l
        no_q[rq] = no_k[rk] = False
    q[no_q], dout[no_q], k[no_k], v[no_k] = (float('nan'),) * 4
    need = ext.prompt_attention_grad_workspace(rows_q, rows_k, len(cu_q) - 1, heads, kv_heads)
    ws = torch.full((need,), 255, dtype=torch.uint8, device='cuda')
    grads = [torch.full_like(x, 3.0) for x in (q, k, v)]
    ext.device_error()
    ext.prompt_attention_grad(q, k, v, out, dout, lse, _offsets(*cu_q), _offsets(*cu_k), 0.125, *grads, ws=ws)
    assert ext.device_error() == 2
    for rq, rk in spans:
        _check_grad(q[rq], k[rk], v[rk], dout[rq], [grads[0][rq], grads[1][rk], grads[2][rk]], [rq.stop - rq.start],
                    [rk.stop - rk.start], 0.125, True)
    assert bool((grads[0][no_q] == 3).all() and (grads[1][no_k] == 3).all() and (grads[2][no_k] == 3).all())


def test_prompt_attention_grad_first_sequence_in_front_of_bad_offsets(ext):
    """The sequence in front keeps its gradients, not finite ones only."""
    q, k, v = _make([64, 64], [64, 64], 2, 2, 'fp16', fused=False)
    dout = torch.randn(q.shape, device='cuda').half()
    out, lse, _ = _run(ext, q, k, v, dout, _cu([64, 64]), _cu([64, 64]), 0.1, True)
    for cu_q, cu_k in (([0, 64, 200], [0, 64, 128]), ([0, 64, 128], [0, 64, 300]), ([0, 64, 10], [0, 64, 128]),
                       ([0, 64, 128], [0, 64, -5])):
        grads = [torch.full_like(x, 3.0) for x in (q, k, v)]
        ext.prompt_attention_grad(q, k, v, out, dout, lse, _offsets(*cu_q), _offsets(*cu_k), 0.1, *grads)
        assert ext.device_error() == 2
        # the largest |do| may lie in the other sequence: the bound for this one goes by the call's
        _check_grad(q, k, v, dout, [torch.cat([x[:64], y[64:]]) for x, y in zip(grads, _run(
            ext, q, k, v, dout, _cu([64, 64]), _cu([64, 64]), 0.1, True)[2])], [64, 64], [64, 64], 0.1, True)


@pytest.mark.parametrize('dtype', ['fp16', 'bf16'])
def test_prompt_attention_grad_padded_batch_of_many_sequences(ext, dtype):
    """Rows in front of, and behind, 70 sequences: which belong to no sequence, with offsets in order."""
    lens = [(i * 37) % 23 for i in range(70)]
    n = sum(lens)
    q, k, v = _make([n + 50], [n + 50], 4, 2, dtype, fused=False)
    dout = torch.randn(q.shape, device='cuda').to(q.dtype)
    cu = _cu(lens) + 20
    for x in (q, k, v, dout):
        x[:20], x[n + 20:] = float('nan'), float('nan')
    out, lse = torch.zeros_like(q), torch.zeros(4, n + 50, device='cuda')
    ext.prompt_attention(q, k, v, out, cu, cu, 0.125, lse=lse)
    grads = [torch.full_like(x, 3.0) for x in (q, k, v)]
    ws = torch.full((ext.prompt_attention_grad_workspace(n + 50, n + 50, 70, 4, 2),), 255, dtype=torch.uint8, device='cuda')
    ext.prompt_attention_grad(q, k, v, out, dout, lse, cu, cu, 0.125, *grads, ws=ws)
    assert ext.device_error() == 0
    mid = slice(20, n + 20)
    _check_grad(q[mid], k[mid], v[mid], dout[mid], [x[mid] for x in grads], lens, lens, 0.125, True)
    assert all(bool((x[:20] == 3).all() and (x[n + 20:] == 3).all()) for x in grads)


@pytest.mark.parametrize('rows,lens_k', [(1000, 1000), (1000, 60000), (12, 4000)])
@pytest.mark.parametrize('heads,kv_heads', [(2, 2), (8, 1)])
def test_prompt_attention_sequence_behind_sequences_that_share_rows(ext, rows, lens_k, heads, kv_heads):
    """Offsets that go back over and over: the sequence behind them still has its tiles, with and without split keys.
    Its gradient too."""
    last, cut_k = rows // 10, lens_k - lens_k // 10
    cu_q = _offsets(*[0, rows - last] * 20, rows)
    cu_k = _offsets(*[0, cut_k] * 20, lens_k)
    q, k, v = _make([rows], [lens_k], heads, kv_heads, 'bf16', fused=False)
    out, lse = torch.full_like(q, 3.0), torch.full((heads, rows), 3.0, device='cuda')
    sizes = (rows, lens_k, 40, heads, kv_heads)
    ws = torch.full((ext.prompt_attention_workspace(*sizes) + 16,), 255, dtype=torch.uint8, device='cuda')
    ext.device_error()
    ext.prompt_attention(q, k, v, out, cu_q, cu_k, 0.125, lse=lse, ws=ws)
    assert ext.device_error() == 2
    rq, rk = slice(rows - last, rows), slice(cut_k, lens_k)
    size = [last], [lens_k - cut_k]
    _check(q[rq], k[rk], v[rk], out[rq], lse[:, rq], *size, 0.125, True)
    dout = torch.randn(q.shape, device='cuda').bfloat16()
    grads = [torch.full_like(x, 3.0) for x in (q, k, v)]
    ws = torch.full((ext.prompt_attention_grad_workspace(*sizes),), 255, dtype=torch.uint8, device='cuda')
    ext.prompt_attention_grad(q, k, v, out, dout, lse, cu_q, cu_k, 0.125, *grads, ws=ws)
    assert ext.device_error() == 2
    _check_grad(q[rq], k[rk], v[rk], dout[rq], [grads[0][rq], grads[1][rk], grads[2][rk]], *size, 0.125, True)


def test_prompt_attention_sequences_out_of_their_order(ext):
    """Good sequences that do not share rows, the later rows first: computed, or left as they were."""
    q, k, v = _make([192], [192], 4, 2, 'fp16', fused=False)
    cu = _offsets(128, 192, 0, 70, 128)
    out, lse = torch.full_like(q, 3.0), torch.full((4, 192), 3.0, device='cuda')
    ext.device_error()
    ext.prompt_attention(q, k, v, out, cu, cu, 0.125, lse=lse)
    assert ext.device_error() == 2
    for first, end, must in ((128, 192, True), (0, 70, False), (70, 128, False)):
        s = slice(first, end)
        if must or not bool((out[s] == 3).all()):
            _check(q[s], k[s], v[s], out[s], lse[:, s], [end - first], [end - first], 0.125, True)


@pytest.mark.parametrize('v_size,do_size,scale', [(4000.0, 1.0, 0.03), (60000.0, 1e-3, 0.02), (300.0, 50.0, 0.03),
                                                 (1e-3, 100.0, 0.1), (65504.0, 4e-4, 0.001)])
@pytest.mark.parametrize('lens', [[3, 2, 1], [200, 5], [140, 300]])
def test_prompt_attention_grad_of_large_values(ext, v_size, do_size, scale, lens):
    """fp16: values of v in the thousands, where do . v is far beyond the largest |do|; nothing overflows that is in range.
    Scores are small, so that no probability is below 2^-11: then the error that p brings (2^-17 p times the sum of |do| |v|, of
    which there are 64) covers half a subnormal step of what is kept, 2^-31 of the largest |do| times the largest |v|."""
    q, k, v = _make(lens, lens, 4, 2, 'fp16', fused=False)
    g = torch.Generator(device='cuda').manual_seed(3)
    v = ((torch.rand(v.shape, device='cuda', generator=g) * 2 - 1) * v_size).half()
    dout = ((torch.rand(q.shape, device='cuda', generator=g) * 2 - 1) * do_size).half()
    cu = _cu(lens)
    _, _, grads = _run(ext, q, k, v, dout, cu, cu, scale, True)
    assert ext.device_error() == 0
    assert all(bool(x.isfinite().all()) for x in grads)
    _check_grad(q, k, v, dout, grads, lens, lens, scale, True)


def test_prompt_attention_grad_largest_value_counts_good_rows_only(ext):
    """What rows of no sequence hold of v does not change a bit; infinities and NaN in a sequence stay there."""
    lens = [60, 30]
    q, k, v = _make([120], [120], 4, 2, 'fp16', fused=False)
    dout = torch.randn(q.shape, device='cuda').half() * 1e-6
    cu = _cu(lens) + 10
    want = _run(ext, q, k, v, dout, cu, cu, 0.125, True)
    for fill in (65504.0, float('inf'), float('nan')):
        v2 = v.clone()
        v2[:10], v2[100:] = fill, fill
        got = _run(ext, q, k, v2, dout, cu, cu, 0.125, True)
        for a, b in zip(got[2], want[2]):
            assert torch.equal(a[10:100], b[10:100])


@pytest.mark.parametrize('top', [0, 12, -8])
@pytest.mark.parametrize('size', [1.0, 0.01, 200.0])
def test_loss_grad_of_unequal_weights(ext, top, size):
    """fp16: weights from 2^top down to 2^(top - 26), and rows so sure of a wrong token that each row of dw comes from one
    row of h: w[i] is row i's token, row 500 + i its target, so dw[i] = g h and dw[500 + i] = -g h. Roundings: p - [t] (u of it
    and 2^-37, half a subnormal step over 2^12), the scaled copy of h (u of it, or half a subnormal step 2^-25 where the
    largest |h g| is kept as at least 2^14, or h as 2^24 times its own), the result (u, or 2^-25); and exp(z) for the others,
    below 2^-40 in sum."""
    n, vocab, hidden, u = 105, 1000, 256, 2.0 ** -11
    gen = torch.Generator(device='cuda').manual_seed(4)
    w = torch.randn(vocab, hidden, device='cuda', generator=gen)
    w = (w / size if size < 1 else w * 0.25).half()
    h = (w[:n].float() * (size * size if size < 1 else 4 * size)).half()
    targets = 500 + torch.arange(n, device='cuda')
    g = 2.0 ** (top - torch.arange(n, device='cuda') / 4.0)
    loss, lse = torch.empty(n, device='cuda'), torch.empty(n, device='cuda')
    ext.lm_head_loss(h, w, targets, loss, lse)
    assert bool((loss > 40).all())
    dh, dw = torch.empty_like(h), torch.full_like(w, float('nan'))
    ext.lm_head_loss_grad(h, w, targets, lse, g, dh, dw)
    assert ext.device_error() == 0
    p = torch.softmax(h.double() @ w.double().T, 1)
    p[torch.arange(n, device='cuda'), targets] -= 1.0
    want = (p * g.double()[:, None]).T @ h.double()
    z_err = 3 * (hidden * 2.0 ** -23 * (h.double().abs() @ w.double().abs().T).amax(1) + 2.0 ** -17)
    gh = g.double()[:, None] * h.double().abs()
    kept = max(2.0 ** -39 * float(gh.max()), 2.0 ** -49 * float(g.max()))
    each = (3 * u + z_err[:, None]) * gh + kept  # of the two rows that row i of h goes to
    bound = torch.full_like(want, 2.0 ** -25) + (2.0 ** -37 + 2.0 ** -40) * gh.sum(0)
    bound[:n] += each
    bound[targets] += each
    # 200 times 2^12 is beyond fp16: such values round to infinity, which _within allows where the bound reaches that far
    _within(dw, want, bound, 'dw')


def test_embedding_of_nearly_2_31_tokens(ext):
    """As many tokens as 32 bits count, rows of one element."""
    n = (1 << 31) - 3
    table = torch.arange(7, device='cuda').bfloat16()[:, None]
    ids = torch.zeros(n, dtype=torch.long, device='cuda')
    ids[-5:], ids[1 << 30] = torch.arange(2, 7, device='cuda'), 1
    out = torch.full((n, 1), 9.0, dtype=torch.bfloat16, device='cuda')
    ext.embed_scaled(table, ids, out, scale=2.0)
    assert ext.device_error() == 0
    assert out[-6:, 0].tolist() == [0, 4, 6, 8, 10, 12] and float(out[1 << 30]) == 2.0
    assert float(out.float().sum()) == 42.0


@pytest.mark.parametrize('size', [100.0, 3000.0, 30000.0])
def test_prompt_attention_grad_with_one_large_value(ext, size):
    """fp16: one element of v far above the rest. The other sequence's ds is off by half a subnormal step more, 2^-37 ||do||
    ||v||, below 2^-18 at 30000; the bound's p e_delta, with e_delta about 2^-6 here, covers that for p above 2^-12, and
    scores of about +-1 over 90 keys leave hardly one below."""
    lens = [90, 140]
    q, k, v = _make(lens, lens, 4, 2, 'fp16', fused=False)
    dout = torch.randn(q.shape, device='cuda').half()
    v[200, 1, 7] = size
    cu = _cu(lens)
    grads = _run(ext, q, k, v, dout, cu, cu, 0.125, True)[2]
    assert ext.device_error() == 0 and all(bool(x.isfinite().all()) for x in grads)
    _check_grad(q, k, v, dout, grads, lens, lens, 0.125, True)
    first = slice(0, 90)
    _check_grad(q[first], k[first], v[first], dout[first], [x[first] for x in grads], lens[:1], lens[:1], 0.125, True)


@pytest.mark.parametrize('n,vocab,hidden', [(300, 2000, 256), (70, 777, 72)])
def test_loss_grad_accumulates_in_fp16(ext, n, vocab, hidden):
    """dw added to what is there, by unequal weights whose copy of h is scaled."""
    h, w, targets = _inputs(n, vocab, hidden, 'fp16')
    loss, lse, g = torch.empty(n, device='cuda'), torch.empty(n, device='cuda'), torch.rand(n, device='cuda') * 3e-3
    ext.lm_head_loss(h, w, targets, loss, lse)
    base = torch.randn(vocab, hidden, device='cuda').half()
    dw = base.clone()
    ext.lm_head_loss_grad(h, w, targets, lse, g, None, dw, accumulate=True)
    _check_loss_grad(h, w, targets, g, lse, None, dw, base=base)
    assert ext.device_error() == 0


@pytest.mark.parametrize('longer', [1, 50])
def test_prompt_attention_many_tokens_with_bad_offsets_among_them(ext, longer):
    """More sequences than the join looks at in one go, some of them prompts, with a bad one in the middle and rows of no
    sequence in front and behind: keys are split, every good sequence is computed."""
    lens = [1] * 200
    lens[20] = lens[160] = longer
    n, lk, bad = sum(lens), 300, 90
    at_q, at_k = _cu(lens) + 7, torch.arange(201, device='cuda') * lk
    q, k, v = _make([n + 30], [200 * lk], 2, 1, 'fp16', fused=False)
    cu_q = at_q.clone()
    cu_q[bad + 1] = 1 << 40  # its end and the next one's begin
    assert ext.prompt_attention_workspace(n + 30, 200 * lk, 200, 2, 1) > 0
    out, lse = torch.full_like(q, 3.0), torch.full((2, n + 30), 3.0, device='cuda')
    ws = torch.full((ext.prompt_attention_workspace(n + 30, 200 * lk, 200, 2, 1),), 255, dtype=torch.uint8, device='cuda')
    ext.device_error()
    ext.prompt_attention(q, k, v, out, cu_q, at_k, 0.125, lse=lse, ws=ws)
    assert ext.device_error() == 2
    left = torch.ones(n + 30, dtype=torch.bool, device='cuda')
    for first, end, size in ((0, bad, lens[:bad]), (bad + 2, 200, lens[bad + 2:])):
        rq, rk = slice(int(at_q[first]), int(at_q[end])), slice(first * lk, end * lk)
        _check(q[rq], k[rk], v[rk], out[rq], lse[:, rq], size, [lk] * len(size), 0.125, True)
        left[rq] = False
    assert bool((out[left] == 3).all()) and bool((lse[:, left] == 3).all())


@pytest.mark.parametrize('n,vocab,hidden', [(5, 226, 1280), (40, 3001, 1280), (100, 1000, 1280), (33, 700, 4096), (300, 900, 1288)])
@pytest.mark.parametrize('dtype', ['fp16', 'bf16'])
def test_loss_of_rows_that_are_sure_of_their_target(ext, n, vocab, hidden, dtype):
    """Rows that leave from 1e-1 to 1e-8 to the other tokens: the loss and p - 1 are small differences of large numbers.

    The target's logit is summed in 256 parts of hidden / 256 terms in fp32 and exactly from there, off by hidden / 256 x
    2^-24 of sum |h w| at most, the others' are off by _logit_error. The loss is log1p of
    others / target, so relative to itself it is off by that, and by 2^-18 for the exponentials; lse is rounded to fp32 (2^-24
    of it, once more for the sum). dz at the target is expm1(z - lse), off by lse's rounding and the relative error of what
    is left; with an lse from elsewhere, by z's error too. Then the 16-bit roundings (see test_gpu_loss.py)."""
    gen = torch.Generator(device='cuda').manual_seed(n + hidden)
    t, u = (torch.float16, 2.0 ** -11) if dtype == 'fp16' else (torch.bfloat16, 2.0 ** -8)
    w = (torch.randn(vocab, hidden, device='cuda', generator=gen) * 1.43 / hidden ** 0.5).to(t)
    targets = torch.randint(vocab, (n,), device='cuda', generator=gen)
    size = torch.linspace(4.0, 12.0, n, device='cuda')[:, None]
    h = (w[targets].float() * size).to(t)
    g = torch.full((n,), 1.0 / n, device='cuda')
    rows = torch.arange(n, device='cuda')
    z = h.double() @ w.double().T
    want_lse = torch.logsumexp(z, 1)
    others = z.clone()
    others[rows, targets] = -float('inf')
    left = torch.exp(torch.logsumexp(others, 1) - want_lse)  # 1 - p without the cancellation
    want_loss = -torch.log1p(-left)
    z_err = (hidden / 256) * 2.0 ** -24 * (h.double().abs() * w[targets].double().abs()).sum(1)
    rel = _logit_error(h, w) * 2 + 2.0 ** -18
    loss, lse = torch.empty(n, device='cuda'), torch.empty(n, device='cuda')
    ext.lm_head_loss(h, w, targets, loss, lse)
    assert bool(((loss.double() - want_loss).abs() <= want_loss * rel).all())
    assert bool(((lse.double() - want_lse).abs() <= z_err + 2.0 ** -23 * want_lse.abs() + left * rel).all())
    dz = torch.exp(z - want_lse[:, None])
    dz[rows, targets] = -left
    want_h, want_w = (dz / n) @ w.double(), (dz / n).T @ h.double()
    for given, off in ((lse, 0.0), (want_lse.float(), z_err)):
        dh, dw = torch.empty_like(h), torch.empty_like(w)
        ext.lm_head_loss_grad(h, w, targets, given, g, dh, dw)
        e = dz.abs() * (u + 1.5 * rel[:, None]) + 2.0 ** -37
        e += dz.abs() * (z_err + 2.0 ** -22 * want_lse.abs())[:, None]  # the others have lse's error
        e[rows, targets] += 2.0 ** -23 * want_lse.abs() + off
        k32 = 8 * 2.0 ** -23
        bound = (e / n) @ w.double().abs() + (dz.abs() / n) @ w.double().abs() * k32 * vocab ** 0.5 + u * want_h.abs()
        tiny = torch.finfo(t).smallest_normal * u
        _within(dh, want_h, bound + tiny, 'dh')
        copy = (dz.abs() / n).T @ h.double().abs() * u if dtype == 'bf16' else 0.0  # 1 / n is the same for all: exact
        bound = (e / n).T @ h.double().abs() + copy + (dz.abs() / n).T @ h.double().abs() * k32 * n ** 0.5 + u * want_w.abs()
        _within(dw, want_w, bound + tiny, 'dw')
    assert ext.device_error() == 0


def test_loss_grad_of_rows_that_are_not_numbers(ext):
    """NaN and infinities in rows that count stay visible; other rows' dh is as it was."""
    for t in (torch.float16, torch.bfloat16):
        h, w, targets = _inputs(90, 700, 128, 'fp16' if t == torch.float16 else 'bf16')
        targets.clamp_(min=0)
        loss, lse, g = torch.empty(90, device='cuda'), torch.empty(90, device='cuda'), torch.ones(90, device='cuda')
        ext.lm_head_loss(h, w, targets, loss, lse)
        want, dh, dw = torch.empty_like(h), torch.empty_like(h), torch.empty_like(w)
        ext.lm_head_loss_grad(h, w, targets, lse, g, want, None)
        h[7, 3], h[50, 9] = float('nan'), float('inf')
        ext.lm_head_loss(h, w, targets, loss, lse)
        assert not bool(loss[7].isfinite()) and not bool(loss[50].isfinite())
        ext.lm_head_loss_grad(h, w, targets, lse, g, dh, dw)
        assert bool(dh[7].isnan().all()) and not bool(dh[50].isfinite().all()) and not bool(dw.isfinite().any())
        rest = torch.ones(90, dtype=torch.bool, device='cuda')
        rest[7] = rest[50] = False
        assert torch.equal(dh[rest], want[rest])
    assert ext.device_error() == 0
