"""Kernel boundary for PyTorch callers: the drop-in for the reference's custom/ext.py.

`load_ext()` returns an object exposing the reference's four kernels with the same names, argument
order and error behaviour as its pybind module (custom/kernels/whisper_kernels.cu:278-363, loaded by
custom/ext.py:13-18):

    add_layernorm(h, x, gamma, beta, y, eps)
    decode_attention(q, k, v, out, len_state, k_new, v_new, part_m, part_l, part_acc, scale)
    lm_head_argmax(h, w, suppress, best)
    argmax_finalize(best, tokens, state, cur, max_pos)

plus the fused decode, log-mel and encoder ops of this package. Each method validates dtype,
device, contiguity and shape like the reference's TORCH_CHECKs (RuntimeError with the same
messages), then calls the C ABI of libflashwhisper.so with raw pointers on the current CUDA
stream. There is no CPU path: without a CUDA tensor the checks fail.
"""

import ctypes
import functools

import torch

from . import _lib

HIDDEN, HEAD_DIM, SPLIT_KEYS = 1280, 64, 64


def _stream():
    return ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)


def _ptr(t):
    return ctypes.c_void_p(t.data_ptr()) if t is not None else ctypes.c_void_p(0)


def _check(cond, msg):
    if not cond:
        raise RuntimeError(msg)


def _check_half(t, name):
    _check(t.is_cuda and t.is_contiguous() and t.dtype == torch.float16, f'{name} must be contiguous CUDA fp16')


def _check_cuda(t, dtype, name, what):
    _check(t.is_cuda and t.is_contiguous() and t.dtype == dtype, f'{name} must be contiguous CUDA {what}')


_DTYPES = {torch.float16: _lib.FW_F16, torch.bfloat16: _lib.FW_BF16, torch.float32: _lib.FW_F32}
_HALF_TYPES = (torch.float16, torch.bfloat16)


# The whole-transcript operators' checks and calls. They cost as much as a small operator takes on the GPU, so messages
# are made only where they are raised, devices are compared by index, and pointers are passed as plain integers.
def _check_typed(t, dtype, dev, name):
    """A contiguous tensor of this type on CUDA device `dev`."""
    if t.dtype is not dtype or dev < 0 or t.get_device() != dev or not t.is_contiguous():
        where = f'on cuda:{dev}' if dev >= 0 else 'on a CUDA device'
        raise RuntimeError(f'{name} must be contiguous CUDA {str(dtype)[6:]} {where}')


def _check_ints(t, n, dev, name):
    if t.dtype is not torch.long or dev < 0 or t.get_device() != dev or t.numel() != n or not t.is_contiguous():
        raise RuntimeError(f'{name} must be contiguous CUDA int64 [{n}] on cuda:{dev}')


def _check_fp32(t, n, dev, name):
    if t.dtype is not torch.float32 or t.get_device() != dev or t.numel() != n or not t.is_contiguous():
        raise RuntimeError(f'{name} must be contiguous CUDA fp32 [{n}] on cuda:{dev}')


def _check_lse(t, heads, rows, dev):
    """Rows before heads would be as many numbers in another order."""
    _check_fp32(t, heads * rows, dev, 'lse')
    if t.shape != (heads, rows):
        more = [n for n in t.shape if n != 1]
        if len(more) < 2 or more == [heads, rows]:
            return  # flat, or with dimensions of 1 besides
        raise RuntimeError(f'lse must be [heads, rows_q] = [{heads}, {rows}]')


def _check_sizes(*sizes):
    """The library takes these in 32 bits, to which they would be cut silently."""
    if max(sizes) > 0x7fffffff:
        raise RuntimeError(f'sizes must be below 2^31, not {max(sizes)}')


@functools.lru_cache(maxsize=1024)
def _workspace_bytes(name, *sizes):
    _check_sizes(*sizes)
    need = ctypes.c_int64(0)
    _lib.call(name, *sizes, ctypes.byref(need))
    return need.value


def _workspace(ws, need, dev):
    """The caller's scratch after a check of its size, or (None) scratch of the device's current stream."""
    if ws is None:
        return torch.empty(need, dtype=torch.uint8, device=f'cuda:{dev}') if need else None
    if (ws.dtype is not torch.uint8 or ws.get_device() != dev or ws.numel() < need or not ws.is_contiguous()):
        raise RuntimeError(f'ws must be contiguous CUDA uint8 on cuda:{dev} of at least {need} bytes')
    return ws


def _address(t):
    return 0 if t is None else t.data_ptr()


def _size(ws):
    return 0 if ws is None else ws.numel()


def _call_on(dev, name, *args):
    """Calls fw_<name> on device `dev`, whichever is current, and its current stream."""
    if torch.cuda.current_device() != dev:
        with torch.cuda.device(dev):
            return _lib.call(name, *args, torch._C._cuda_getCurrentRawStream(dev))
    return _lib.call(name, *args, torch._C._cuda_getCurrentRawStream(dev))


class Ext:
    """Reference-compatible kernel module backed by libflashwhisper.so."""

    SPLIT_KEYS = SPLIT_KEYS

    def __init__(self):
        self.lib = _lib.lib()

    # ---- reference surface -----------------------------------------------------------------
    def add_layernorm(self, h, x, gamma, beta, y, eps):
        """h += x (stored back in fp16) when x is given, then y = LayerNorm(h)."""
        for t, n in ((h, 'h'), (gamma, 'gamma'), (beta, 'beta'), (y, 'y')):
            _check_half(t, n)
        _check(h.numel() == HIDDEN, f'hidden size must be {HIDDEN}')
        if x is not None:
            _check_half(x, 'x')
        _lib.call('fw_add_layernorm', _ptr(h), _ptr(x), _ptr(gamma), _ptr(beta), _ptr(y), HIDDEN, float(eps),
                  _stream())

    def decode_attention(self, q, k, v, out, len_state, k_new, v_new, part_m, part_l, part_acc, scale):
        """Split-K single-query attention; self attention (len_state given) also writes k_new/v_new."""
        for t, n in ((q, 'q'), (k, 'k'), (v, 'v'), (out, 'out')):
            _check_half(t, n)
        _check(k.dim() == 3 and k.size(2) == HEAD_DIM and k.shape == v.shape, 'k, v must be [heads, max_len, 64]')
        heads, max_len = k.size(0), k.size(1)
        splits = -(-max_len // SPLIT_KEYS)
        _check(q.numel() == heads * HEAD_DIM and out.numel() == heads * HEAD_DIM, 'q, out must be [heads * 64]')
        _check((k_new is None) == (v_new is None) == (len_state is None),
               'len_state, k_new and v_new must be given together')
        if k_new is not None:
            _check_half(k_new, 'k_new')
            _check_half(v_new, 'v_new')
            _check(k_new.numel() == heads * HEAD_DIM and v_new.numel() == heads * HEAD_DIM,
                   'k_new, v_new must be [heads, 64]')
            _check(len_state.is_cuda and len_state.dtype == torch.long, 'len_state must be CUDA int64')
        for t in (part_m, part_l, part_acc):
            _check(t.is_cuda and t.is_contiguous() and t.dtype == torch.float32,
                   'workspace must be contiguous CUDA fp32')
        _check(part_m.numel() >= heads * splits and part_l.numel() >= heads * splits
               and part_acc.numel() >= heads * splits * HEAD_DIM, f'workspace too small for {splits} splits')
        _lib.call('fw_decode_attention', _ptr(q), _ptr(k), _ptr(v), _ptr(out), _ptr(len_state), _ptr(k_new),
                  _ptr(v_new), _ptr(part_m), part_m.numel(), _ptr(part_l), part_l.numel(), _ptr(part_acc),
                  part_acc.numel(), heads, max_len, float(scale), _stream())

    def decode_attention_noalloc(self, q, k, v, out, len_state, k_new, v_new, scale):
        """decode_attention without a workspace: the split partials live in the library's fixed device
        array (heads * ceil(max_len / 64) <= 2048; calls that overlap on the GPU race on it)."""
        for t, n in ((q, 'q'), (k, 'k'), (v, 'v'), (out, 'out')):
            _check_half(t, n)
        _check(k.dim() == 3 and k.size(2) == HEAD_DIM and k.shape == v.shape, 'k, v must be [heads, max_len, 64]')
        heads, max_len = k.size(0), k.size(1)
        _check(q.numel() == heads * HEAD_DIM and out.numel() == heads * HEAD_DIM, 'q, out must be [heads * 64]')
        _check((k_new is None) == (v_new is None) == (len_state is None),
               'len_state, k_new and v_new must be given together')
        if k_new is not None:
            _check_half(k_new, 'k_new')
            _check_half(v_new, 'v_new')
            _check(k_new.numel() == heads * HEAD_DIM and v_new.numel() == heads * HEAD_DIM,
                   'k_new, v_new must be [heads, 64]')
            _check(len_state.is_cuda and len_state.dtype == torch.long, 'len_state must be CUDA int64')
        _lib.call('fw_decode_attention_noalloc', _ptr(q), _ptr(k), _ptr(v), _ptr(out), _ptr(len_state), _ptr(k_new),
                  _ptr(v_new), heads, max_len, float(scale), _stream())

    def lm_head_argmax(self, h, w, suppress, best):
        """best <- max(best, packed key of the unsuppressed argmax of fp16(w @ h))."""
        _check_half(h, 'h')
        _check_half(w, 'w')
        _check(h.numel() == HIDDEN and w.dim() == 2 and w.size(1) == HIDDEN, f'hidden size must be {HIDDEN}')
        _check(suppress.dtype == torch.bool and suppress.numel() == w.size(0) and suppress.is_cuda
               and suppress.is_contiguous(), 'suppress must be bool [vocab]')
        _check(best.dtype == torch.long and best.numel() == 1 and best.is_cuda, 'best must be int64 [1]')
        _lib.call('fw_lm_head_argmax', _ptr(h), _ptr(w), _ptr(suppress), w.size(0), HIDDEN, _ptr(best), _stream())

    def lm_quantize(self, w):
        """(wq int8 [vocab, 1280], rp fp32 [vocab, 4]): the int8 LM head and per-row bounds that
        lm_head_argmax_q and the decode step's pruned argmax stream instead of w."""
        _check_half(w, 'w')
        _check(w.dim() == 2 and w.size(1) == HIDDEN, f'hidden size must be {HIDDEN}')
        wq = torch.empty(w.shape, dtype=torch.int8, device=w.device)
        rp = torch.empty(w.size(0), 4, dtype=torch.float32, device=w.device)
        _lib.call('fw_lm_quantize', _ptr(w), w.size(0), HIDDEN, _ptr(wq), _ptr(rp), _stream())
        return wq, rp

    def lm_head_argmax_q(self, h, w, wq, rp, suppress, best):
        """As lm_head_argmax (same key), streaming the lm_quantize output and recomputing exactly
        only the rows that can still win."""
        _check_half(h, 'h')
        _check_half(w, 'w')
        _check(h.numel() == HIDDEN and w.dim() == 2 and w.size(1) == HIDDEN, f'hidden size must be {HIDDEN}')
        _check(wq.dtype == torch.int8 and wq.shape == w.shape and wq.is_cuda and wq.is_contiguous(),
               'wq must be int8 like w')
        _check(rp.dtype == torch.float32 and rp.shape == (w.size(0), 4) and rp.is_cuda and rp.is_contiguous(),
               'rp must be fp32 [vocab, 4]')
        _check(suppress.dtype == torch.bool and suppress.numel() == w.size(0) and suppress.is_cuda
               and suppress.is_contiguous(), 'suppress must be bool [vocab]')
        _check(best.dtype == torch.long and best.numel() == 1 and best.is_cuda, 'best must be int64 [1]')
        _lib.call('fw_lm_head_argmax_q', _ptr(h), _ptr(w), _ptr(wq), _ptr(rp), _ptr(suppress), w.size(0), HIDDEN,
                  _ptr(best), _stream())

    def argmax_finalize(self, best, tokens, state, cur, max_pos):
        """Appends the decoded token, feeds it back, advances the position and resets best."""
        _check(tokens.dtype == torch.long and state.dtype == torch.long and cur.dtype == torch.long,
               'tokens, state and cur must be int64')
        _check(best.dtype == torch.long and best.numel() == 1, 'best must be int64 [1]')
        for t in (best, tokens, state, cur):
            _check(t.is_cuda and t.is_contiguous(), 'tokens, state and cur must be int64')
        _lib.call('fw_argmax_finalize', _ptr(best), _ptr(tokens), tokens.numel(), _ptr(state), _ptr(cur),
                  int(max_pos), _stream())

    # ---- fused / stand-alone decode ops ------------------------------------------------------
    def embed_pos(self, embed, pos_embed, ids, positions, out):
        """out[i] = fp16(embed[ids[i]] + pos_embed[positions[i]])."""
        for t, n in ((embed, 'embed'), (pos_embed, 'pos_embed'), (out, 'out')):
            _check_half(t, n)
        for t, n in ((ids, 'ids'), (positions, 'positions')):
            _check_cuda(t, torch.long, n, 'int64')
        n = ids.numel()
        _check(positions.numel() == n and out.numel() == n * embed.size(1) and pos_embed.size(1) == embed.size(1),
               'embed_pos: shape mismatch')
        _lib.call('fw_embed_pos', _ptr(embed), _ptr(pos_embed), _ptr(ids), _ptr(positions), _ptr(out), n,
                  embed.size(0), pos_embed.size(0), embed.size(1), _stream())

    def gelu(self, x, y):
        _check_half(x, 'x')
        _check_half(y, 'y')
        _check(x.numel() == y.numel(), 'gelu: x and y must have the same size')
        _lib.call('fw_gelu', _ptr(x), _ptr(y), x.numel(), _stream())

    def argmax_f16(self, logits, suppress, key, out_index):
        """out_index = first argmax of unsuppressed fp16 logits; key is an int64 scratch word (0)."""
        _check_half(logits, 'logits')
        if suppress is not None:
            _check(suppress.dtype == torch.bool and suppress.numel() == logits.numel() and suppress.is_cuda,
                   'suppress must be bool [n]')
        _check_cuda(key, torch.long, 'key', 'int64')
        _check_cuda(out_index, torch.long, 'out_index', 'int64')
        _lib.call('fw_argmax_f16', _ptr(logits), logits.numel(), _ptr(suppress), _ptr(key), _ptr(out_index),
                  _stream())

    def ln_gemv(self, h, gamma, beta, eps, w, b, out, act=0):
        """out = act(w @ LayerNorm(h) + b); act 0 none, 1 exact GELU."""
        for t, n in ((h, 'h'), (gamma, 'gamma'), (beta, 'beta'), (w, 'w'), (out, 'out')):
            _check_half(t, n)
        _check(h.numel() == HIDDEN and w.dim() == 2 and w.size(1) == HIDDEN, f'hidden size must be {HIDDEN}')
        _check(out.numel() == w.size(0), 'ln_gemv: out must have w.size(0) elements')
        if b is not None:
            _check_half(b, 'b')
        _lib.call('fw_ln_gemv', _ptr(h), _ptr(gamma), _ptr(beta), float(eps), _ptr(w), _ptr(b), _ptr(out),
                  w.size(0), HIDDEN, int(act), _stream())

    def gemv_residual(self, x, w, b, h):
        """h = fp16(h + fp16(w @ x + b))."""
        for t, n in ((x, 'x'), (w, 'w'), (h, 'h')):
            _check_half(t, n)
        _check(w.dim() == 2 and w.size(1) == x.numel() and h.numel() == w.size(0), 'gemv_residual: shape mismatch')
        if b is not None:
            _check_half(b, 'b')
        _lib.call('fw_gemv_residual', _ptr(x), x.numel(), _ptr(w), _ptr(b), _ptr(h), w.size(0), _stream())

    # ---- front end and encoder ---------------------------------------------------------------
    def log_mel(self, wave, filters, scratch, clip_max, out, layout=0):
        """fp16 log-mel of fp32 wave [batch, n_samples]; layout 0 [b,128,T], 1 [b,T+2,128] padded."""
        _check_cuda(wave, torch.float32, 'wave', 'fp32')
        _check_cuda(filters, torch.float32, 'filters', 'fp32')
        _check_cuda(scratch, torch.float32, 'scratch', 'fp32')
        _check(clip_max.is_cuda and clip_max.dtype == torch.int32, 'clip_max must be CUDA int32')
        _check_half(out, 'out')
        wave2 = wave.view(-1, wave.size(-1))
        batch, n = wave2.shape
        frames = n // 160
        _check(filters.shape == (201, 128), 'filters must be [201, 128]')
        _check(scratch.numel() >= batch * 128 * frames and clip_max.numel() >= batch, 'log_mel: scratch too small')
        want = batch * 128 * frames if layout == 0 else batch * (frames + 2) * 128
        _check(out.numel() == want, 'log_mel: output has the wrong size')
        _lib.call('fw_log_mel', _ptr(wave2), batch, n, _ptr(filters), _ptr(scratch), _ptr(clip_max), _ptr(out),
                  int(layout), _stream())

    def gemm(self, a, b, bias, c, epilogue=_lib.FW_EPI_BIAS, r=None, scale=1.0, scale_cols=0, m=None):
        """c = epilogue(a @ b.T + bias) on tcgen05 tensor cores."""
        _check_half(a, 'a')
        _check_half(b, 'b')
        _check_half(c, 'c')
        m = a.size(0) if m is None else m
        n, k = b.shape
        ldc = c.stride(0) if c.dim() == 2 else 0
        ldr = r.stride(0) if r is not None else 0
        _lib.call('fw_gemm_f16', _ptr(a), a.stride(0), _ptr(b), b.stride(0), _ptr(bias), _ptr(c), ldc, _ptr(r), ldr,
                  m, n, k, int(epilogue), float(scale), int(scale_cols), _stream())

    def conv1d_k3(self, x_padded, w_taps, bias, out, stride, epilogue=_lib.FW_EPI_BIAS_GELU, r=None, m=None):
        """Conv1d(k=3, pad=1) over a zero-padded time-major input as an implicit tcgen05 GEMM."""
        _check_half(x_padded, 'x')
        _check_half(w_taps, 'w')
        rows, ch = x_padded.shape
        n = w_taps.size(0)
        m = (rows - 2 + stride - 1) // stride if m is None else m
        ldr = r.stride(0) if r is not None else 0
        _lib.call('fw_conv1d_k3_f16', _ptr(x_padded), ch, rows, int(stride), _ptr(w_taps), _ptr(bias), _ptr(out),
                  out.stride(0), _ptr(r), ldr, m, n, int(epilogue), _stream())

    def layernorm_rows(self, x, g, b, y, eps):
        for t, n in ((x, 'x'), (g, 'g'), (b, 'b'), (y, 'y')):
            _check_half(t, n)
        _lib.call('fw_layernorm_rows', _ptr(x), _ptr(g), _ptr(b), _ptr(y), x.size(0), x.size(1), float(eps),
                  _stream())

    def encoder_attention(self, qkv, out, heads, kcol=HIDDEN, vcol=2 * HIDDEN, vt=None):
        """vt: optional fp16 scratch [heads * 64, round_up(seq, 8)] for V transposed (allocated if None)."""
        _check_half(qkv, 'qkv')
        _check_half(out, 'out')
        if vt is None:
            vt = torch.empty(int(heads) * 64, -(-qkv.size(0) // 8) * 8, dtype=torch.float16, device=qkv.device)
        _check_half(vt, 'vt')
        _lib.call('fw_encoder_attention', _ptr(qkv), qkv.stride(0), int(kcol), int(vcol), _ptr(out), qkv.size(0),
                  int(heads), _ptr(vt), _stream())

    # ---- whole transcripts ---------------------------------------------------------------------
    # These take the tensors' own device, whichever is current, and its current stream. `ws` is uint8
    # scratch of at least the matching *_workspace bytes; without it scratch is allocated on that stream.
    def embed_scaled(self, embed, ids, out, scale=1.0, pos_embed=None, positions=None):
        """out[i] = embed[ids[i]] * scale (+ pos_embed[positions[i]]) in fp16, bf16 or fp32."""
        dtype, dev, n = embed.dtype, embed.get_device(), ids.numel()
        _check(dtype in _DTYPES, 'embed must be fp16, bf16 or fp32')
        _check_typed(embed, dtype, dev, 'embed')
        _check_typed(out, dtype, dev, 'out')
        _check_ints(ids, n, dev, 'ids')
        _check(embed.dim() == 2 and embed.numel() > 0, 'embed must be [vocab, hidden]')
        vocab, hidden = embed.shape
        max_pos = pos_at = positions_at = 0
        if pos_embed is not None and positions is not None:
            _check_typed(pos_embed, dtype, dev, 'pos_embed')
            _check_ints(positions, n, dev, 'positions')
            max_pos = pos_embed.size(0)
            _check(pos_embed.dim() == 2 and max_pos > 0 and pos_embed.size(1) == hidden,
                   'pos_embed must be [max_pos, hidden]')
            pos_at, positions_at = pos_embed.data_ptr(), positions.data_ptr()
        else:
            _check(pos_embed is positions, 'pos_embed and positions must be given together')
        _check(out.numel() == n * hidden, 'embed_scaled: out must be [n, hidden]')
        _check_sizes(n, vocab, max_pos, hidden)
        _call_on(dev, 'fw_embed_scaled', embed.data_ptr(), pos_at, ids.data_ptr(), positions_at, out.data_ptr(), n,
                 vocab, max_pos, hidden, scale, _DTYPES[dtype])

    def embed_grad_workspace(self, n, hidden):
        return _workspace_bytes('fw_embed_grad_workspace', int(n), int(hidden))

    def embed_grad(self, dout, ids, dembed, scale=1.0, padding_idx=-1, accumulate=False, ws=None):
        """dembed[v] = (dembed[v] if accumulate) + scale * sum of dout[i] over ids[i] == v != padding_idx, summed in
        fp32 in an order that only the ids decide. With ids = positions and scale 1 it is the position table's gradient."""
        dtype, dev, n = dembed.dtype, dembed.get_device(), ids.numel()
        _check(dtype in _DTYPES, 'dembed must be fp16, bf16 or fp32')
        _check_typed(dembed, dtype, dev, 'dembed')
        _check_typed(dout, dtype, dev, 'dout')
        _check_ints(ids, n, dev, 'ids')
        _check(dembed.dim() == 2 and dembed.numel() > 0, 'dembed must be [vocab, hidden]')
        vocab, hidden = dembed.shape
        _check(dout.numel() == n * hidden, 'embed_grad: dout must be [n, hidden]')
        _check_sizes(n, vocab, hidden)
        ws = _workspace(ws, self.embed_grad_workspace(n, hidden), dev)
        _call_on(dev, 'fw_embed_grad', dout.data_ptr(), ids.data_ptr(), dembed.data_ptr(), n, vocab, hidden, scale,
                 padding_idx, 1 if accumulate else 0, _DTYPES[dtype], _address(ws), _size(ws))

    @staticmethod
    def _rows(t, dtype, dev, shape, name):
        """[rows, heads, 64] of this type, strided over rows and heads, as a C descriptor."""
        if (t.dtype is not dtype or t.get_device() != dev or t.shape != shape
                or (t.stride(2) != 1 and t.numel() > 0)):
            raise RuntimeError(f'{name} must be CUDA {str(dtype)[6:]} [{shape[0]}, {shape[1]}, {shape[2]}] on '
                               f'cuda:{dev}, its last dimension contiguous')
        token, head, _ = t.stride()
        # a dimension of one element has no stride of its own
        if shape[1] <= 1:
            head = HEAD_DIM
        return _lib.Rows(t.data_ptr(), token if shape[0] > 1 else shape[1] * head, head)

    def _check_prompt(self, q, k, v, cu_q, cu_k):
        _check(q.dtype in _HALF_TYPES, 'q must be fp16 or bf16')
        _check(q.dim() == 3 and k.dim() == 3, 'q and k must be [rows, heads, 64]')
        rows_q, heads, _ = q.shape
        rows_k, kv_heads, _ = k.shape
        _check(heads > 0 and kv_heads > 0 and heads % kv_heads == 0, 'heads must be a multiple of kv_heads')
        dev, seqs = q.get_device(), max(cu_q.numel() - 1, 0)
        _check_ints(cu_q, seqs + 1, dev, 'cu_q')
        _check_ints(cu_k, seqs + 1, dev, 'cu_k')
        _check_sizes(seqs, heads, kv_heads)
        return dev, (rows_q, heads, HEAD_DIM), (rows_k, kv_heads, HEAD_DIM), seqs

    def prompt_attention_workspace(self, rows_q, rows_k, seqs, heads, kv_heads):
        return _workspace_bytes('fw_prompt_attention_workspace', int(rows_q), int(rows_k), int(seqs), int(heads),
                                int(kv_heads))

    def prompt_attention(self, q, k, v, out, cu_q, cu_k, scale, causal=True, lse=None, ws=None):
        """Attention over packed sequences: q, out [rows_q, heads, 64], k, v [rows_k, kv_heads, 64] (fp16 or bf16, rows
        and heads strided); sequence b has the rows cu_q[b]:cu_q[b + 1] and cu_k[b]:cu_k[b + 1] (int64). causal: the
        last query sees the last key. lse: fp32 [heads, rows_q] or None."""
        dev, like_q, like_k, seqs = self._check_prompt(q, k, v, cu_q, cu_k)
        dtype, ref = q.dtype, ctypes.byref
        rq, ro = self._rows(q, dtype, dev, like_q, 'q'), self._rows(out, dtype, dev, like_q, 'out')
        rk, rv = self._rows(k, dtype, dev, like_k, 'k'), self._rows(v, dtype, dev, like_k, 'v')
        rows_q, heads, rows_k, kv_heads = like_q[0], like_q[1], like_k[0], like_k[1]
        if lse is not None:
            _check_lse(lse, heads, rows_q, dev)
        ws = _workspace(ws, self.prompt_attention_workspace(rows_q, rows_k, seqs, heads, kv_heads), dev)
        _call_on(dev, 'fw_prompt_attention', ref(rq), ref(rk), ref(rv), ref(ro), _address(lse), cu_q.data_ptr(),
                 cu_k.data_ptr(), seqs, rows_q, rows_k, heads, kv_heads, scale, 1 if causal else 0, _DTYPES[dtype],
                 _address(ws), _size(ws))

    def prompt_attention_grad_workspace(self, rows_q, rows_k, seqs, heads, kv_heads):
        return _workspace_bytes('fw_prompt_attention_grad_workspace', int(rows_q), int(rows_k), int(seqs), int(heads),
                                int(kv_heads))

    def prompt_attention_grad(self, q, k, v, out, dout, lse, cu_q, cu_k, scale, dq, dk, dv, causal=True, ws=None):
        """Gradient of prompt_attention: dq like q, dk and dv like k and v, for dout, from the forward's out and lse."""
        dev, like_q, like_k, seqs = self._check_prompt(q, k, v, cu_q, cu_k)
        dtype, ref = q.dtype, ctypes.byref
        rq, ro, rd, rdq = (self._rows(t, dtype, dev, like_q, name)
                           for t, name in ((q, 'q'), (out, 'out'), (dout, 'dout'), (dq, 'dq')))
        rk, rv, rdk, rdv = (self._rows(t, dtype, dev, like_k, name)
                            for t, name in ((k, 'k'), (v, 'v'), (dk, 'dk'), (dv, 'dv')))
        rows_q, heads, rows_k, kv_heads = like_q[0], like_q[1], like_k[0], like_k[1]
        _check_lse(lse, heads, rows_q, dev)
        ws = _workspace(ws, self.prompt_attention_grad_workspace(rows_q, rows_k, seqs, heads, kv_heads), dev)
        _call_on(dev, 'fw_prompt_attention_grad', ref(rq), ref(rk), ref(rv), ref(ro), ref(rd), lse.data_ptr(),
                 cu_q.data_ptr(), cu_k.data_ptr(), seqs, rows_q, rows_k, heads, kv_heads, scale, 1 if causal else 0,
                 _DTYPES[dtype], ref(rdq), ref(rdk), ref(rdv), _address(ws), _size(ws))

    def _check_loss(self, h, w, targets):
        dtype, dev = h.dtype, h.get_device()
        _check(dtype in _HALF_TYPES, 'h must be fp16 or bf16')
        _check_typed(h, dtype, dev, 'h')
        _check_typed(w, dtype, dev, 'w')
        _check(h.dim() == 2 and w.dim() == 2 and w.size(1) == h.size(1) and w.size(0) > 0 and w.size(1) > 0,
               'h must be [n, hidden], w [vocab, hidden]')
        _check_ints(targets, h.size(0), dev, 'targets')
        _check_sizes(*h.shape, *w.shape)
        return dev, h.size(0), w.size(0), h.size(1)

    def lm_head_loss_workspace(self, n, vocab):
        return _workspace_bytes('fw_lm_head_loss_workspace', int(n), int(vocab))

    def lm_head_loss(self, h, w, targets, loss, lse, ignore_index=-100, ws=None):
        """loss[i] = lse[i] - h[i] . w[targets[i]] (0 where targets[i] == ignore_index), lse[i] = log sum_v
        exp(h[i] . w[v]), both fp32 [n]; h, w fp16 or bf16. The logits are never stored."""
        dev, n, vocab, hidden = self._check_loss(h, w, targets)
        _check_fp32(loss, n, dev, 'loss')
        _check_fp32(lse, n, dev, 'lse')
        ws = _workspace(ws, self.lm_head_loss_workspace(n, vocab), dev)
        _call_on(dev, 'fw_lm_head_loss', h.data_ptr(), w.data_ptr(), targets.data_ptr(), loss.data_ptr(),
                 lse.data_ptr(), n, vocab, hidden, ignore_index, _DTYPES[h.dtype], _address(ws), _size(ws))

    def lm_head_loss_grad_workspace(self, n, vocab, hidden):
        return _workspace_bytes('fw_lm_head_loss_grad_workspace', int(n), int(vocab), int(hidden))

    def lm_head_loss_grad(self, h, w, targets, lse, g, dh, dw, ignore_index=-100, accumulate=False, ws=None):
        """Gradient of sum_i g[i] loss[i] of lm_head_loss: dh like h, dw like w (either may be None); accumulate adds
        to dw. lse is lm_head_loss's, g fp32 [n]."""
        dev, n, vocab, hidden = self._check_loss(h, w, targets)
        _check_fp32(lse, n, dev, 'lse')
        _check_fp32(g, n, dev, 'g')
        for t, like, name in ((dh, h, 'dh'), (dw, w, 'dw')):
            if t is not None:
                _check_typed(t, h.dtype, dev, name)
                _check(t.shape == like.shape, 'dh must be shaped like h, dw like w')
        _check(dh is not None or dw is not None, 'at least one of dh and dw is required')
        ws = _workspace(ws, self.lm_head_loss_grad_workspace(n, vocab, hidden), dev)
        _call_on(dev, 'fw_lm_head_loss_grad', h.data_ptr(), w.data_ptr(), targets.data_ptr(), lse.data_ptr(),
                 g.data_ptr(), _address(dh), _address(dw), n, vocab, hidden, ignore_index, 1 if accumulate else 0,
                 _DTYPES[h.dtype], _address(ws), _size(ws))

    def decoder_step(self, desc, steps=1):
        _lib.call('fw_decoder_step', ctypes.byref(desc), int(steps), _stream())

    def batch_decoder_step(self, desc, steps=1):
        """`steps` decode steps of every clip of a batched decoder descriptor (_lib.BatchDecoder)."""
        _lib.call('fw_batch_decoder_step', ctypes.byref(desc), int(steps), _stream())

    def batch_decoder_launch(self, desc, layer, block):
        """One launch of the batched step (0 qkv, 1 self attention, 2 out_proj, 3 cross q, 4 cross
        attention, 5 cross out_proj, 6 fc1, 7 fc2, 8 LM head)."""
        _lib.call('fw_batch_decoder_launch', ctypes.byref(desc), int(layer), int(block), _stream())

    def decoder_launch(self, desc, layer, block):
        """One launch of the decode step (block 0 self, 1 cross, 2 fc1, 3 fc2, 4 LM head)."""
        _lib.call('fw_decoder_launch', ctypes.byref(desc), int(layer), int(block), _stream())

    def decoder_step_trace(self, desc, trace):
        """One decode step that also records each block's output into `trace` (fp16, at least
        n_layers * TRACE_LAYER + 1280 elements; layout in include/flash_whisper.h)."""
        _check_half(trace, 'trace')
        need = desc.n_layers * _lib.TRACE_LAYER + HIDDEN
        if trace.numel() < need:
            raise RuntimeError(f'trace must hold at least {need} fp16 elements')
        _lib.call('fw_decoder_step_trace', ctypes.byref(desc), _ptr(trace), _stream())

    def encoder_forward(self, desc):
        _lib.call('fw_encoder_forward', ctypes.byref(desc), _stream())

    def device_error(self, clear=True):
        bits = ctypes.c_uint(0)
        _lib.call('fw_device_error', ctypes.byref(bits), int(clear))
        return bits.value


_EXT = None


def load_ext(verbose=False):
    """Returns the kernel module (the library is built ahead of time by flash_whisper_b200.build)."""
    global _EXT
    if _EXT is None:
        _EXT = Ext()
    return _EXT
