"""The decoder operators that work on whole transcripts (teacher-forced scoring and training), as cases to be timed.

A transcript's tokens go through the token embedding, causal attention over the packed transcripts and the tied
vocabulary matrix with its cross entropy; each of the three comes with its gradient. `run` computes one operator
once: in plain torch operations where `own` is false, by the calls a user makes of flash_whisper_b200.ext where it
is true. Sizes are the ones this package has (hidden 1280, vocabulary 51866, 20 heads of 64, 448 text positions, 8
clips at a time) and generic larger ones.
"""

import math

import torch

own = False

HEAD_DIM = 64
IGNORE = -100
TYPES = {'fp16': torch.float16, 'bf16': torch.bfloat16, 'fp32': torch.float32}
ITEM = {'fp16': 2, 'bf16': 2, 'fp32': 4}


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # the four forced prompt tokens of one clip, with their positions: latency
        {'name': 'embed_prompt', 'op': 'embed', 'n': 4, 'vocab': 51866, 'hidden': 1280, 'max_pos': 448,
         'scale': 1.0, 'dtype': 'fp16'},
        # a large packed training batch, rows scaled by sqrt(hidden), no learned positions
        {'name': 'embed_packed', 'op': 'embed', 'n': 32749, 'vocab': 51866, 'hidden': 1280, 'max_pos': 0,
         'scale': 35.777, 'dtype': 'bf16'},
        # eight transcripts of 448 tokens: the dense gradient of the table
        {'name': 'embed_grad_clips', 'op': 'embed_grad', 'n': 3584, 'vocab': 51866, 'hidden': 1280, 'scale': 1.0,
         'padding': 50257, 'dtype': 'fp16'},
        # a large packed batch without padding
        {'name': 'embed_grad_packed', 'op': 'embed_grad', 'n': 32749, 'vocab': 51866, 'hidden': 1280,
         'scale': 35.777, 'padding': -1, 'dtype': 'bf16'},
        # one short transcript scored: log probabilities of 27 tokens
        {'name': 'loss_transcript', 'op': 'loss', 'n': 27, 'vocab': 51866, 'hidden': 1280, 'dtype': 'fp16'},
        # a large packed batch scored
        {'name': 'loss_packed', 'op': 'loss', 'n': 16381, 'vocab': 51866, 'hidden': 1280, 'dtype': 'bf16'},
        # gradient for two short transcripts (fine-tuning on a few examples)
        {'name': 'loss_grad_transcripts', 'op': 'loss_grad', 'n': 211, 'vocab': 51866, 'hidden': 1280,
         'dtype': 'fp16'},
        # gradient for a packed batch
        {'name': 'loss_grad_packed', 'op': 'loss_grad', 'n': 8189, 'vocab': 51866, 'hidden': 1280, 'dtype': 'bf16'},
        # one new token for each of eight clips over what they have so far: the serving form
        {'name': 'attn_token', 'op': 'attn', 'lq': '1,1,1,1,1,1,1,1', 'lk': '448,1500,1,37,1499,224,700,129',
         'heads': 20, 'kv_heads': 20, 'causal': True, 'dtype': 'fp16'},
        # packed prompts of very different lengths, grouped heads
        {'name': 'attn_packed', 'op': 'attn', 'lq': '4096,1,777,2048,250,4001', 'lk': '4096,1,777,2048,250,4001',
         'heads': 32, 'kv_heads': 8, 'causal': True, 'dtype': 'bf16'},
        # eight ragged transcripts, every head with its own keys
        {'name': 'attn_grad_clips', 'op': 'attn_grad', 'lq': '448,391,27,224,448,1,130,305',
         'lk': '448,391,27,224,448,1,130,305', 'heads': 20, 'kv_heads': 20, 'causal': True, 'dtype': 'fp16'},
        # long packed sequences, grouped heads
        {'name': 'attn_grad_packed', 'op': 'attn_grad', 'lq': '4096,1,777,2048,250,4001',
         'lk': '4096,1,777,2048,250,4001', 'heads': 32, 'kv_heads': 8, 'causal': True, 'dtype': 'bf16'},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(['embed', 'embed_grad', 'loss', 'loss_grad', 'attn', 'attn_grad'])
    dtype = rng.choice(['fp16', 'bf16'])
    if op in ('embed', 'embed_grad'):
        hidden = 8 * _log_int(rng, 8, 256)
        vocab = _log_int(rng, 300, 60000)
        most = 32749 * 1280 // hidden if op == 'embed' else 32000 * 1280 // hidden
        case = {'op': op, 'n': _log_int(rng, 1, min(32749, most)), 'vocab': min(vocab, 51866 * 1280 // hidden),
                'hidden': hidden, 'scale': rng.choice([1.0, round(math.sqrt(hidden), 3)]),
                'dtype': rng.choice(['fp16', 'bf16', 'bf16', 'fp32']) if hidden <= 640 else dtype}
        if op == 'embed':
            return {**case, 'max_pos': rng.choice([0, 448, _log_int(rng, 16, 4096)])}
        return {**case, 'padding': rng.choice([-1, rng.randrange(case['vocab'])])}
    if op in ('loss', 'loss_grad'):
        hidden = rng.choice([384, 512, 768, 1024, 1280, 8 * _log_int(rng, 8, 256)])
        vocab = min(rng.choice([51866, 51865, _log_int(rng, 100, 60000)]), 51866 * 1280 // hidden)
        most = (16381 if op == 'loss' else 8189) * 51866 * 1280
        return {'op': op, 'n': _log_int(rng, 1, min(16381, most // (vocab * hidden))), 'vocab': vocab,
                'hidden': hidden, 'dtype': dtype}
    group = rng.choice([1, 1, 2, 3, 4, 5, 8])
    kv = rng.choice([1, 2, 4, 8, 20]) if group == 1 else rng.choice([1, 2, 4])
    form = rng.choice(['prompt', 'prompt', 'token', 'chunk', 'cross']) if op == 'attn' else rng.choice(
        ['prompt', 'prompt', 'chunk', 'cross'])
    lk = [_log_int(rng, 1, 4096) for _ in range(rng.randint(1, 8))]
    if form == 'prompt':
        lq = list(lk)
    elif form == 'token':
        lq = [1] * len(lk)
    elif form == 'chunk':  # new tokens behind a kept prefix; now and then fewer keys than queries
        lq = [_log_int(rng, 1, max(1, n)) + (rng.choice([0, 0, 0, 5])) for n in lk]
    else:  # transcripts against the frames of their clips
        lq = [_log_int(rng, 1, 448) for _ in lk]
        lk = [rng.choice([1500, n]) for n in lk]
    if rng.random() < 0.2:
        lk[-1] = 0 if form != 'prompt' else lk[-1]
    return {'op': op, 'lq': ','.join(map(str, lq)), 'lk': ','.join(map(str, lk)), 'heads': group * kv,
            'kv_heads': kv, 'causal': form != 'cross', 'dtype': dtype}


# ------------------------------------------------------------------------------------------------ inputs
def _lens(text):
    return [int(x) for x in text.split(',')]


def _gen(seed):
    return torch.Generator(device='cuda').manual_seed(seed)


def _tokens(n, vocab, g):
    """Token ids as text has them: a few very frequent ones, a long tail."""
    u = torch.rand(n, device='cuda', generator=g)
    rank = torch.exp(u * math.log(vocab)).long().clamp_(1, vocab) - 1
    return (rank * 7919) % vocab


def _normal(shape, std, dtype, g):
    return torch.empty(shape, dtype=dtype, device='cuda').normal_(0.0, std, generator=g)


def prepare(case, seed):
    g = _gen(seed)
    op, t = case['op'], TYPES[case['dtype']]
    s = dict(case)
    if op == 'embed':
        n, vocab, hidden = case['n'], case['vocab'], case['hidden']
        s['embed'] = _normal((vocab, hidden), 0.02, t, g)
        s['ids'] = _tokens(n, vocab, g)
        s['pos_embed'] = s['positions'] = None
        if case['max_pos']:
            s['pos_embed'] = _normal((case['max_pos'], hidden), 0.02, t, g)
            s['positions'] = torch.arange(n, device='cuda') % case['max_pos']
    elif op == 'embed_grad':
        n, vocab, hidden = case['n'], case['vocab'], case['hidden']
        s['ids'] = _tokens(n, vocab, g)
        if case['padding'] >= 0:  # the ends of the shorter transcripts
            s['ids'] = torch.where(torch.rand(n, device='cuda', generator=g) < 0.15,
                                   torch.full_like(s['ids'], case['padding']), s['ids'])
        s['dout'] = _normal((n, hidden), 0.1, t, g)
    elif op in ('loss', 'loss_grad'):
        n, vocab, hidden = case['n'], case['vocab'], case['hidden']
        s['w'] = _normal((vocab, hidden), 0.04, t, g)
        s['targets'] = _tokens(n, vocab, g)
        # hidden states that lean towards their targets, as a trained decoder's do
        h = torch.empty(n, hidden, device='cuda').normal_(0.0, 1.0, generator=g)
        h += 5.0 * torch.rand(n, 1, device='cuda', generator=g) * s['w'][s['targets']].float() / 0.04 / 8
        s['h'] = h.to(t)
        s['targets'][torch.rand(n, device='cuda', generator=g) < 0.1] = IGNORE
        if op == 'loss_grad':
            s['lse'] = torch.cat([torch.logsumexp(x.float() @ s['w'].float().T, 1) for x in s['h'].split(2048)])
            kept = (s['targets'] != IGNORE).float()
            s['g'] = kept / kept.sum().clamp(min=1.0)
    else:
        lq, lk = _lens(case['lq']), _lens(case['lk'])
        hq, hk = case['heads'], case['kv_heads']
        if lq == lk:  # self attention: q, k and v are views of the fused projection's output
            qkv = _normal((sum(lq), hq + 2 * hk, HEAD_DIM), 1.0, t, g)
            s['q'], s['k'], s['v'] = qkv[:, :hq], qkv[:, hq:hq + hk], qkv[:, hq + hk:]
        else:
            s['q'] = _normal((sum(lq), hq, HEAD_DIM), 1.0, t, g)
            s['k'] = _normal((sum(lk), hk, HEAD_DIM), 1.0, t, g)
            s['v'] = _normal((sum(lk), hk, HEAD_DIM), 1.0, t, g)
        s['scale'] = 1.5 * HEAD_DIM ** -0.5
        s['cu_q'] = torch.tensor([0] + lq, device='cuda').cumsum(0)
        s['cu_k'] = torch.tensor([0] + lk, device='cuda').cumsum(0)
        s['max_q'], s['max_k'] = max(lq), max(lk)
        if op == 'attn_grad':
            s['out'], s['lse'] = _attention(s)
            s['dout'] = _normal((sum(lq), hq, HEAD_DIM), 0.1, t, g)
    return s


# ------------------------------------------------------------------------------------------------ plain forms
def _embed(s):
    x = s['embed'][s['ids']].float() * s['scale']
    if s['positions'] is not None:
        x = x + s['pos_embed'][s['positions']].float()
    return x.to(s['embed'].dtype)


def _embed_grad(s):
    ids, dout = s['ids'], s['dout']
    rows = dout.float() * s['scale']
    rows = torch.where((ids == s['padding'])[:, None], torch.zeros_like(rows), rows)
    sums = torch.zeros(s['vocab'], s['hidden'], device='cuda').index_add_(0, ids, rows)
    return sums.to(dout.dtype)


def _loss(s):
    z = s['h'].float() @ s['w'].float().T
    top = z.amax(1)
    lse = top + torch.log(torch.exp(z - top[:, None]).sum(1))
    kept = s['targets'] != IGNORE
    at = z.gather(1, s['targets'].clamp(min=0)[:, None])[:, 0]
    return {'loss': torch.where(kept, lse - at, torch.zeros_like(lse)), 'lse': lse}


def _loss_grad(s):
    h, w = s['h'].float(), s['w'].float()
    kept = s['targets'] != IGNORE
    dz = torch.exp(h @ w.T - s['lse'][:, None])
    dz.scatter_add_(1, s['targets'].clamp(min=0)[:, None], torch.full_like(dz[:, :1], -1.0))
    dz *= torch.where(kept, s['g'], torch.zeros_like(s['g']))[:, None]
    return {'dh': (dz @ w).to(s['h'].dtype), 'dw': (dz.T @ h).to(s['w'].dtype)}


def _spread(x, cu, longest):
    """Packed rows [T, H, D] as [B, H, longest, D] in 32 bits, zeros behind each sequence's end."""
    at = cu[:-1, None] + torch.arange(longest, device=x.device)[None]
    x = torch.cat([x, x.new_zeros(1, *x.shape[1:])])
    return x[torch.where(at < cu[1:, None], at, x.shape[0] - 1)].float().transpose(1, 2)


def _packed(x, cu, rows):
    """[B, H, L, ...] back to packed rows [T, H, ...]."""
    row = torch.arange(rows, device=x.device)
    seq = torch.searchsorted(cu, row, right=True) - 1
    return x.transpose(1, 2)[seq, row - cu[seq]]


def _scores(s):
    """Scaled scores [B, Hq, Lq, Lk] with -inf wherever a query does not see a key; and q, k, v spread out."""
    group = s['heads'] // s['kv_heads']
    q = _spread(s['q'], s['cu_q'], s['max_q'])
    k = _spread(s['k'], s['cu_k'], s['max_k']).repeat_interleave(group, 1)
    v = _spread(s['v'], s['cu_k'], s['max_k']).repeat_interleave(group, 1)
    nq, nk = s['cu_q'].diff(), s['cu_k'].diff()
    i, j = torch.arange(s['max_q'], device='cuda')[:, None], torch.arange(s['max_k'], device='cuda')[None]
    seen = (j[None] < nk[:, None, None]) & (i[None] < nq[:, None, None])
    if s['causal']:  # the last query sees the last key
        seen = seen & (j[None] <= i[None] + (nk - nq)[:, None, None])
    z = (q @ k.transpose(2, 3)).mul_(s['scale']).masked_fill_(~seen[:, None], -math.inf)
    return z, q, k, v


def _attention(s):
    z, _, _, v = _scores(s)
    top = z.amax(3, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    e = z.sub_(top).exp_()
    total = e.sum(3, keepdim=True)
    out = (e @ v) / torch.where(total == 0, torch.ones_like(total), total)
    lse = (top + torch.log(total))[..., 0]
    rows = s['q'].shape[0]
    return _packed(out, s['cu_q'], rows).to(s['q'].dtype), _packed(lse, s['cu_q'], rows).T.contiguous()


def _attention_grad(s):
    group, hk = s['heads'] // s['kv_heads'], s['kv_heads']
    z, q, k, v = _scores(s)
    lse = _spread(s['lse'].T[:, :, None], s['cu_q'], s['max_q'])
    p = z.sub_(torch.where(lse == -math.inf, torch.zeros_like(lse), lse)).exp_()
    dout = _spread(s['dout'], s['cu_q'], s['max_q'])
    delta = (dout * _spread(s['out'], s['cu_q'], s['max_q'])).sum(3, keepdim=True)
    dv = p.transpose(2, 3) @ dout
    dz = (dout @ v.transpose(2, 3)).sub_(delta).mul_(p).mul_(s['scale'])
    dq, dk = dz @ k, dz.transpose(2, 3) @ q
    b, _, n, d = dk.shape
    dk, dv = dk.view(b, hk, group, n, d).sum(2), dv.view(b, hk, group, n, d).sum(2)
    t, nq, nk = s['q'].dtype, s['q'].shape[0], s['k'].shape[0]
    return {'dq': _packed(dq, s['cu_q'], nq).to(t), 'dk': _packed(dk, s['cu_k'], nk).to(t),
            'dv': _packed(dv, s['cu_k'], nk).to(t)}


# ------------------------------------------------------------------------------------------------ one pass
def _run_own(s):
    from flash_whisper_b200.ext import load_ext
    ext, op = load_ext(), s['op']
    if op == 'embed':
        out = torch.empty(s['n'], s['hidden'], dtype=s['embed'].dtype, device='cuda')
        ext.embed_scaled(s['embed'], s['ids'], out, scale=s['scale'], pos_embed=s['pos_embed'],
                         positions=s['positions'])
        return out
    if op == 'embed_grad':
        dembed = torch.empty(s['vocab'], s['hidden'], dtype=s['dout'].dtype, device='cuda')
        ext.embed_grad(s['dout'], s['ids'], dembed, scale=s['scale'], padding_idx=s['padding'])
        return dembed
    if op == 'loss':
        loss, lse = torch.empty(s['n'], device='cuda'), torch.empty(s['n'], device='cuda')
        ext.lm_head_loss(s['h'], s['w'], s['targets'], loss, lse, ignore_index=IGNORE)
        return {'loss': loss, 'lse': lse}
    if op == 'loss_grad':
        dh, dw = torch.empty_like(s['h']), torch.empty_like(s['w'])
        ext.lm_head_loss_grad(s['h'], s['w'], s['targets'], s['lse'], s['g'], dh, dw, ignore_index=IGNORE)
        return {'dh': dh, 'dw': dw}
    q, k, v = s['q'], s['k'], s['v']
    if op == 'attn':
        out = torch.empty(q.shape, dtype=q.dtype, device='cuda')
        lse = torch.empty(q.shape[1], q.shape[0], device='cuda')
        ext.prompt_attention(q, k, v, out, s['cu_q'], s['cu_k'], s['scale'], causal=s['causal'], lse=lse)
        return {'out': out, 'lse': lse}
    dq, dk, dv = (torch.empty(x.shape, dtype=x.dtype, device='cuda') for x in (q, k, v))
    ext.prompt_attention_grad(q, k, v, s['out'], s['dout'], s['lse'], s['cu_q'], s['cu_k'], s['scale'], dq, dk, dv,
                              causal=s['causal'])
    return {'dq': dq, 'dk': dk, 'dv': dv}


def run(state):
    if own:
        return _run_own(state)
    op = state['op']
    if op == 'embed':
        return _embed(state)
    if op == 'embed_grad':
        return _embed_grad(state)
    if op == 'loss':
        return _loss(state)
    if op == 'loss_grad':
        return _loss_grad(state)
    if op == 'attn':
        out, lse = _attention(state)
        return {'out': out, 'lse': lse}
    return _attention_grad(state)


# ------------------------------------------------------------------------------------------------ what it costs
def _seen(nq, nk, causal):
    """How many (query, key) pairs one sequence has; causal query i sees i + 1 + nk - nq keys."""
    rows = min(nq, nk)
    return rows * (2 * nk - rows + 1) // 2 if causal else nq * nk


def _pairs(case):
    return sum(_seen(nq, nk, case['causal']) for nq, nk in zip(_lens(case['lq']), _lens(case['lk'])))


def work(case):
    op, size = case['op'], ITEM[case['dtype']]
    if op == 'embed':
        n, hidden = case['n'], case['hidden']
        rows = n + min(n, case['vocab']) + min(n, case['max_pos'])
        return {'bytes': rows * hidden * size + 8 * n * (2 if case['max_pos'] else 1), 'flops': 2 * n * hidden}
    if op == 'embed_grad':
        n, vocab, hidden = case['n'], case['vocab'], case['hidden']
        return {'bytes': (n + vocab) * hidden * size + 8 * n, 'flops': 2 * n * hidden}
    if op in ('loss', 'loss_grad'):
        n, vocab, hidden = case['n'], case['vocab'], case['hidden']
        moved = (n + vocab) * hidden * size + 8 * n
        if op == 'loss':
            return {'bytes': moved + 8 * n, 'flops': 2 * n * vocab * hidden}
        return {'bytes': moved + 8 * n + (n + vocab) * hidden * size, 'flops': 6 * n * vocab * hidden}
    nq, nk, hq, hk = sum(_lens(case['lq'])), sum(_lens(case['lk'])), case['heads'], case['kv_heads']
    q, kv = nq * hq * HEAD_DIM * size, nk * hk * HEAD_DIM * size
    if op == 'attn':
        return {'bytes': 2 * q + 2 * kv + 4 * nq * hq, 'flops': 4 * HEAD_DIM * hq * _pairs(case)}
    return {'bytes': 4 * q + 4 * kv + 4 * nq * hq, 'flops': 10 * HEAD_DIM * hq * _pairs(case)}


# ------------------------------------------------------------------------------------------------ 64 bits
def exact(case, seed):
    s, op = prepare(case, seed), case['op']
    if op == 'embed':
        x = s['embed'].double().index_select(0, s['ids']) * case['scale']
        return x if s['positions'] is None else x + s['pos_embed'].double().index_select(0, s['positions'])
    if op == 'embed_grad':
        kept = s['ids'] != case['padding']
        dembed = torch.zeros(case['vocab'], case['hidden'], dtype=torch.float64, device='cuda')
        dembed.index_put_((s['ids'][kept],), s['dout'][kept].double(), accumulate=True)
        return dembed * case['scale']
    if op in ('loss', 'loss_grad'):
        w, targets = s['w'].double(), s['targets']
        if op == 'loss':
            loss, lse = [], []
            for h, t in zip(s['h'].split(1024), targets.split(1024)):
                logp = torch.log_softmax(h.double() @ w.T, 1)
                loss.append(torch.nn.functional.nll_loss(logp, t, ignore_index=IGNORE, reduction='none'))
                lse.append((h.double() @ w[0]) - logp[:, 0])
            return {'loss': torch.cat(loss), 'lse': torch.cat(lse)}
        dh, dw = [], torch.zeros_like(w)
        for h, t, g in zip(s['h'].split(1024), targets.split(1024), s['g'].split(1024)):
            h = h.double()
            dz = torch.softmax(h @ w.T, 1)
            kept = (t != IGNORE).nonzero()[:, 0]
            dz[kept, t[kept]] -= 1.0
            dz *= (g.double() * (t != IGNORE))[:, None]
            dh.append(dz @ w)
            dw += dz.T @ h
        return {'dh': torch.cat(dh), 'dw': dw}
    q, k, v = s['q'].double(), s['k'].double(), s['v'].double()
    group, scale = case['heads'] // case['kv_heads'], s['scale']
    out, lse = torch.zeros_like(q), torch.full((case['heads'], q.shape[0]), -math.inf, device='cuda', dtype=q.dtype)
    dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    a = b = 0
    for nq, nk in zip(_lens(case['lq']), _lens(case['lk'])):
        first = max(0, nq - nk) if case['causal'] else 0  # the queries before it see nothing
        for h in range(case['heads'] if nk and nq > first else 0):
            x, y, z = q[a + first:a + nq, h], k[b:b + nk, h // group], v[b:b + nk, h // group]
            score = x @ y.T * scale
            if case['causal']:
                score += torch.full_like(score, -math.inf).triu(nk - (nq - first) + 1)
            top = torch.logsumexp(score, 1)
            p = torch.exp(score - top[:, None])
            o = p @ z
            out[a + first:a + nq, h], lse[h, a + first:a + nq] = o, top
            if op == 'attn_grad':
                do = s['dout'][a + first:a + nq, h].double()
                ds = p * (do @ z.T - (do * o).sum(1, keepdim=True)) * scale
                dq[a + first:a + nq, h] = ds @ y
                dk[b:b + nk, h // group] += ds.T @ x
                dv[b:b + nk, h // group] += p.T @ do
        a, b = a + nq, b + nk
    return {'out': out, 'lse': lse} if op == 'attn' else {'dq': dq, 'dk': dk, 'dv': dv}
