"""Whole-transcript operators where their promises end: long walks beside other work, offsets that are wrong in the middle,
values near the ends of fp16. Tolerances are those of test_gpu_prompt.py, test_gpu_prompt_grad.py and test_gpu_loss.py."""

import pytest
import torch

from tests.test_gpu_prompt import _check, _cu, _make
from tests.test_gpu_prompt_grad import _check_grad, _run

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
