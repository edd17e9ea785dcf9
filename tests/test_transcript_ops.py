"""CPU tests of the whole-transcript operators' refusals: the C entry points reject bad sizes, types, alignment and
workspaces before anything touches a GPU, and the wrappers reject tensors that are not on one."""

import ctypes

import pytest
import torch

from flash_whisper_b200 import _lib
from flash_whisper_b200.ext import Ext

P = ctypes.c_void_p(256)
ODD = ctypes.c_void_p(257)


def _refused(name, args, status, text):
    lib = _lib.lib()
    assert getattr(lib, name)(*args) == status, lib.fw_last_error_string()
    assert text in lib.fw_last_error_string().decode(), lib.fw_last_error_string()


@pytest.mark.parametrize('args,status,text', [
    ((None, None, P, None, P, 4, 10, 0, 64, 1.0, 0, None), 1, 'required'),
    ((P, None, None, None, P, 4, 10, 0, 64, 1.0, 0, None), 1, 'required'),
    ((P, P, P, None, P, 4, 10, 5, 64, 1.0, 0, None), 4, 'given together'),
    ((P, None, P, None, P, -1, 10, 0, 64, 1.0, 0, None), 2, 'bad sizes'),
    ((P, None, P, None, P, 4, 0, 0, 64, 1.0, 0, None), 2, 'bad sizes'),
    ((P, P, P, P, P, 4, 10, 0, 64, 1.0, 0, None), 2, 'bad sizes'),
    ((P, None, P, None, P, 4, 10, 0, 64, 1.0, 3, None), 4, 'dtype'),
    ((ODD, None, P, None, P, 4, 10, 0, 64, 1.0, 1, None), 3, 'aligned'),
])
def test_embed_scaled_refuses(args, status, text):
    _refused('fw_embed_scaled', args, status, text)


@pytest.mark.parametrize('args,status,text', [
    ((P, P, None, 4, 10, 64, 1.0, -1, 0, 0, P, 1 << 20, None), 1, 'required'),
    ((P, P, P, 4, 10, 64, 1.0, -1, 0, 0, None, 1 << 20, None), 1, 'required'),
    ((P, P, P, 4, 10, 0, 1.0, -1, 0, 0, P, 1 << 20, None), 2, 'bad sizes'),
    ((P, P, P, 4, (1 << 30) + 1, 64, 1.0, -1, 0, 0, P, 1 << 20, None), 2, 'bad sizes'),
    ((P, P, P, 4, 10, 64, 1.0, -1, 0, 7, P, 1 << 20, None), 4, 'dtype'),
    ((P, P, ODD, 4, 10, 64, 1.0, -1, 0, 2, P, 1 << 20, None), 3, 'aligned'),
    ((P, P, P, 4, 10, 64, 1.0, -1, 0, 0, ODD, 1 << 20, None), 3, 'workspace'),
    ((P, P, P, 4, 10, 64, 1.0, -1, 0, 0, P, 100, None), 2, 'workspace too small'),
])
def test_embed_grad_refuses(args, status, text):
    _refused('fw_embed_grad', args, status, text)


def test_nothing_to_do_needs_no_gpu():
    lib = _lib.lib()
    assert lib.fw_embed_scaled(P, None, None, None, None, 0, 10, 0, 64, 1.0, 0, None) == 0
    assert lib.fw_embed_grad(None, None, P, 0, 10, 64, 1.0, -1, 1, 0, None, 0, None) == 0


def test_embed_wrappers_refuse_cpu_tensors():
    ext = Ext()
    h, ids = torch.zeros(4, 64, dtype=torch.float16), torch.zeros(4, dtype=torch.long)
    with pytest.raises(RuntimeError, match='embed must be contiguous CUDA float16'):
        ext.embed_scaled(h, ids, h)
    with pytest.raises(RuntimeError, match='dembed must be contiguous CUDA float16'):
        ext.embed_grad(h, ids, h)
    with pytest.raises(RuntimeError, match='fp16, bf16 or fp32'):
        ext.embed_scaled(h.double(), ids, h)
    assert ext.embed_grad_workspace(100, 64) > 0
    with pytest.raises(RuntimeError, match='bad sizes'):
        ext.embed_grad_workspace(-1, 64)


@pytest.mark.parametrize('args,status,text', [
    ((None, P, P, P, P, 4, 10, 64, -100, 0, P, 1 << 20, None), 1, 'required'),
    ((P, P, P, None, P, 4, 10, 64, -100, 0, P, 1 << 20, None), 1, 'loss and lse'),
    ((P, P, P, P, P, 4, 10, 60, -100, 0, P, 1 << 20, None), 2, 'multiple of 8'),
    ((P, P, P, P, P, 4, 0, 64, -100, 0, P, 1 << 20, None), 2, 'n and vocab'),
    ((P, P, P, P, P, (1 << 22) + 1, 10, 64, -100, 0, P, 1 << 20, None), 2, 'n and vocab'),
    ((P, P, P, P, P, 4, 10, 64, -100, 2, P, 1 << 20, None), 4, 'dtype'),
    ((P, ODD, P, P, P, 4, 10, 64, -100, 0, P, 1 << 20, None), 3, '16-byte aligned'),
    ((P, P, P, P, P, 400, 1000, 64, -100, 0, P, 100, None), 2, 'workspace too small'),
])
def test_lm_head_loss_refuses(args, status, text):
    _refused('fw_lm_head_loss', args, status, text)


@pytest.mark.parametrize('args,status,text', [
    ((P, P, P, None, P, P, P, 4, 10, 64, -100, 0, 0, P, 1 << 30, None), 1, 'lse and g'),
    ((P, P, P, P, P, None, None, 4, 10, 64, -100, 0, 0, P, 1 << 30, None), 1, 'at least one of dh and dw'),
    ((P, P, P, P, P, P, ODD, 4, 10, 64, -100, 0, 0, P, 1 << 30, None), 3, '16-byte aligned'),
    ((P, P, P, P, P, P, P, 4, 10, 65544, -100, 0, 0, P, 1 << 30, None), 2, 'hidden'),
    ((P, P, P, P, P, P, P, 4, 10, 64, -100, 0, 0, P, 100, None), 2, 'workspace too small'),
])
def test_lm_head_loss_grad_refuses(args, status, text):
    _refused('fw_lm_head_loss_grad', args, status, text)


def test_loss_wrappers_refuse():
    ext = Ext()
    h, t, f = torch.zeros(4, 64, dtype=torch.float16), torch.zeros(4, dtype=torch.long), torch.zeros(4)
    with pytest.raises(RuntimeError, match='h must be contiguous CUDA float16'):
        ext.lm_head_loss(h, h, t, f, f)
    with pytest.raises(RuntimeError, match='h must be fp16 or bf16'):
        ext.lm_head_loss_grad(h.float(), h, t, f, f, h, h)
    assert ext.lm_head_loss_workspace(0, 10) == 0
    assert ext.lm_head_loss_grad_workspace(100, 1000, 64) > 100 * 64 * 2
    with pytest.raises(RuntimeError, match='n and vocab'):
        ext.lm_head_loss_workspace(1, 0)


def test_lm_head_loss_grad_scratch_is_bounded():
    """A piece of the vocabulary at a time: the scratch does not grow with n * vocab."""
    ext = Ext()
    assert ext.lm_head_loss_grad_workspace(8192, 51866, 1280) < 200 << 20
    assert ext.lm_head_loss_grad_workspace(65536, 51866, 1280) < 65536 * 51866  # half a byte a logit


def _rows(ptr=256, token=640, head=64):
    return ctypes.byref(_lib.Rows(ptr, token, head))


def _attn(**changed):
    a = dict(q=_rows(), k=_rows(), v=_rows(), out=_rows(), lse=P, cu_q=P, cu_k=P, seqs=2, rows_q=100, rows_k=100,
             heads=10, kv_heads=10, scale=0.125, causal=1, dtype=0, ws=P, ws_bytes=1 << 40)
    assert set(changed) <= set(a)
    a.update(changed)
    return (*a.values(), None)


def _attn_grad(**changed):
    a = dict(q=_rows(), k=_rows(), v=_rows(), out=_rows(), dout=_rows(), lse=P, cu_q=P, cu_k=P, seqs=2, rows_q=100,
             rows_k=100, heads=10, kv_heads=10, scale=0.125, causal=1, dtype=0, dq=_rows(), dk=_rows(), dv=_rows(),
             ws=P, ws_bytes=1 << 40)
    assert set(changed) <= set(a)
    a.update(changed)
    return (*a.values(), None)


@pytest.mark.parametrize('changed,status,text', [
    (dict(q=None), 1, 'required'), (dict(k=_rows(ptr=0)), 1, 'k is required'), (dict(cu_k=None), 1, 'cu_q and cu_k'),
    (dict(seqs=-1), 2, 'bad sizes'), (dict(rows_k=1 << 30), 2, 'bad sizes'), (dict(kv_heads=3), 2, 'multiple of kv_heads'),
    (dict(heads=0), 2, 'multiple of kv_heads'), (dict(heads=1290, kv_heads=10), 2, 'at most 128 times'),
    (dict(scale=0.0), 4, 'positive'), (dict(scale=-1.0), 4, 'positive'), (dict(scale=float('nan')), 4, 'positive'),
    (dict(scale=float('inf')), 4, 'positive'), (dict(dtype=2), 4, 'dtype'), (dict(v=_rows(ptr=264)), 3, '16 bytes'),
    (dict(q=_rows(token=644)), 3, 'multiple of 8'), (dict(k=_rows(head=32)), 2, 'overlapping'),
    (dict(v=_rows(token=64, head=64)), 2, 'overlapping'), (dict(k=_rows(token=-640)), 2, 'overlapping'),
])
def test_prompt_attention_refuses(changed, status, text):
    _refused('fw_prompt_attention', _attn(**changed), status, text)
    _refused('fw_prompt_attention_grad', _attn_grad(**changed), status, text)


def test_prompt_attention_refuses_small_workspaces():
    _refused('fw_prompt_attention', _attn(rows_q=2, ws_bytes=10, rows_k=4096, heads=1, kv_heads=1), 2, 'workspace too')
    _refused('fw_prompt_attention', _attn(rows_q=2, ws=None, rows_k=4096, heads=1, kv_heads=1), 3, 'workspace')
    _refused('fw_prompt_attention_grad', _attn_grad(ws_bytes=10), 2, 'workspace too')
    _refused('fw_prompt_attention_grad', _attn_grad(ws=None), 3, 'workspace')
    _refused('fw_prompt_attention_grad', _attn_grad(lse=None), 1, 'lse')
    _refused('fw_prompt_attention_grad', _attn_grad(dk=_rows(ptr=8)), 3, 'dk must start')


def test_prompt_wrappers_refuse():
    ext = Ext()
    q, cu = torch.zeros(4, 2, 64, dtype=torch.float16), torch.tensor([0, 4])
    with pytest.raises(RuntimeError, match='cu_q must be contiguous CUDA int64'):
        ext.prompt_attention(q, q, q, q, cu, cu, 0.1)
    with pytest.raises(RuntimeError, match='q must be fp16 or bf16'):
        ext.prompt_attention(q.float(), q, q, q, cu, cu, 0.1)
    with pytest.raises(RuntimeError, match='multiple of kv_heads'):
        ext.prompt_attention_grad(q, torch.zeros(4, 3, 64), q, q, q, q, cu, cu, 0.1, q, q, q)
    with pytest.raises(RuntimeError, match='rows, heads, 64'):
        ext.prompt_attention(q[0], q, q, q, cu, cu, 0.1)
    assert ext.prompt_attention_workspace(11173, 11173, 6, 32, 8) == 0  # enough query tiles: no key splits
    assert ext.prompt_attention_workspace(1, 4096, 1, 1, 1) > 0  # one token: the keys are split


def test_rows_struct_matches_header():
    assert ctypes.sizeof(_lib.Rows) == 24 and _lib.Rows.token.offset == 8 and _lib.Rows.head.offset == 16


def test_prompt_attention_refuses_what_overflows():
    for scale in (2.5e38, 3.4e38):  # times log2 e no longer finite
        _refused('fw_prompt_attention', _attn(scale=scale), 4, 'positive and finite')
        _refused('fw_prompt_attention_grad', _attn_grad(scale=scale), 4, 'positive and finite')
    wide = _rows(token=1 << 35, head=(1 << 35) - 64)  # neither rows behind heads nor heads behind rows
    _refused('fw_prompt_attention', _attn(k=wide, rows_k=(1 << 29) + 1), 2, 'overlapping')


@pytest.mark.parametrize('vocab,hidden', [(1, 8), (33, 64), (5003, 384), (51866, 1280), (1 << 22, 1280)])
def test_loss_scratch_grows_with_rows_and_stays_bounded(vocab, hidden):
    """Over the rows' whole range, kernels and pieces changing on the way: never more than dz's 112 MB (or one tile of 256
    columns), 16 parts of dh's sums and the copy of h; and the forward's 8 bytes a row and half tile, or a CTA."""
    ext = Ext()
    for n in (1, 2, 31, 32, 33, 64, 65, 211, 1024, 2047, 4096, 8189, 16381, 100001):
        most = max(112 << 20, n * 256 * 2) + n * hidden * (16 * 4 + 2) + 4096
        assert n * hidden * 6 < ext.lm_head_loss_grad_workspace(n, vocab, hidden) <= most
        assert 8 * n <= ext.lm_head_loss_workspace(n, vocab) <= 8 * n * max(148, 2 * -(-vocab // 256))
