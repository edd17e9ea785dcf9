"""CPU tests of what the whole-transcript wrappers refuse although sizes and pointers alone would do: stand-ins for CUDA
tensors, and a library call that is not made."""

import ctypes
import math

import pytest
import torch

from flash_whisper_b200 import _lib
from flash_whisper_b200 import ext as ext_module
from flash_whisper_b200.ext import Ext


class Stub:
    """What the wrappers ask of a contiguous tensor on cuda:0, of any size."""

    def __init__(self, *shape, dtype=torch.float16):
        self.shape, self.dtype = torch.Size(shape), dtype

    def get_device(self):
        return 0

    def is_contiguous(self):
        return True

    def dim(self):
        return len(self.shape)

    def size(self, i):
        return self.shape[i]

    def numel(self):
        return math.prod(self.shape)

    def stride(self, i=None):
        steps = tuple(math.prod(self.shape[j + 1:]) for j in range(len(self.shape)))
        return steps if i is None else steps[i]

    def data_ptr(self):
        return 256


def ints(*shape):
    return Stub(*shape, dtype=torch.long)


def floats(*shape):
    return Stub(*shape, dtype=torch.float32)


def scratch():
    return Stub(1 << 45, dtype=torch.uint8)


@pytest.fixture
def calls(monkeypatch):
    made = []
    monkeypatch.setattr(ext_module, '_call_on', lambda dev, name, *args: made.append(name))
    return made


@pytest.mark.parametrize('shape', [(30, 4), (1, 30, 4), (2, 60), (30, 2, 2)])
def test_lse_with_rows_before_heads_is_refused(calls, shape):
    ext, q, cu = Ext(), Stub(30, 4, 64), ints(3)
    for good in ((4, 30), (120,), (1, 4, 30), (120, 1)):
        ext.prompt_attention(q, q, q, q, cu, cu, 0.125, lse=floats(*good), ws=scratch())
        ext.prompt_attention_grad(q, q, q, q, q, floats(*good), cu, cu, 0.125, q, q, q, ws=scratch())
    assert len(calls) == 8
    with pytest.raises(RuntimeError, match=r'lse must be \[heads, rows_q\] = \[4, 30\]'):
        ext.prompt_attention(q, q, q, q, cu, cu, 0.125, lse=floats(*shape), ws=scratch())
    with pytest.raises(RuntimeError, match=r'lse must be \[heads, rows_q\]'):
        ext.prompt_attention_grad(q, q, q, q, q, floats(*shape), cu, cu, 0.125, q, q, q, ws=scratch())
    assert len(calls) == 8


FAR = (1 << 32) + 4  # 4 in 32 bits


def test_sizes_past_32_bits_are_refused(calls):
    ext, f = Ext(), floats(4)
    few, many = Stub(4, 8), Stub(FAR, 8)
    cases = [
        lambda: ext.embed_scaled(few, ints(FAR), many),
        lambda: ext.embed_scaled(many, ints(4), few),
        lambda: ext.embed_scaled(few, ints(4), few, pos_embed=many, positions=ints(4)),
        lambda: ext.embed_scaled(Stub(4, FAR), ints(4), Stub(4, FAR)),
        lambda: ext.embed_grad(many, ints(FAR), few, ws=scratch()),
        lambda: ext.embed_grad(few, ints(4), many, ws=scratch()),
        lambda: ext.lm_head_loss(few, many, ints(4), f, f, ws=scratch()),
        lambda: ext.lm_head_loss(many, few, ints(FAR), floats(FAR), floats(FAR), ws=scratch()),
        lambda: ext.lm_head_loss_grad(few, many, ints(4), f, f, few, many, ws=scratch()),
        lambda: ext.prompt_attention(Stub(4, 2, 64), Stub(4, 2, 64), Stub(4, 2, 64), Stub(4, 2, 64), ints(FAR + 1),
                                     ints(FAR + 1), 0.1, ws=scratch()),
        lambda: ext.embed_grad_workspace(FAR, 8),
        lambda: ext.lm_head_loss_workspace(4, FAR),
        lambda: ext.lm_head_loss_grad_workspace(4, 4, FAR),
        lambda: ext.prompt_attention_workspace(4, 4, FAR, 2, 2),
    ]
    for i, case in enumerate(cases):
        with pytest.raises(RuntimeError, match='below 2'):
            case()
            pytest.fail(f'case {i} was not refused')
    assert not calls


def test_embedding_sizes_at_the_end_of_32_bits():
    """Scratch for more tokens than the operator takes would come out negative; rows of 2^30 elements and more would
    overflow the kernels' column counts."""
    ext, lib, p = Ext(), _lib.lib(), ctypes.c_void_p(256)
    assert ext.embed_grad_workspace(1 << 30, 8) > 4 << 32
    for n in ((1 << 30) + 1, (1 << 31) - 1):
        with pytest.raises(RuntimeError, match='bad sizes'):
            ext.embed_grad_workspace(n, 8)
    assert lib.fw_embed_scaled(p, None, p, None, p, 4, 1, 0, (1 << 30) + 1, 1.0, 1, None) == 2
    # refused before anything is launched, so without a GPU too
    assert lib.fw_embed_grad(p, p, p, 4, 1, 1 << 30, 1.0, -1, 0, 1, p, 1 << 62, None) == 2
    assert b'hidden is too large' in lib.fw_last_error_string()
