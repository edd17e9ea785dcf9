"""Whole-transcript operators where their promises end: long walks beside other work, offsets that are wrong in the middle,
values near the ends of fp16. Tolerances are those of test_gpu_prompt.py, test_gpu_prompt_grad.py and test_gpu_loss.py."""

import pytest
import torch

from tests.test_gpu_prompt import _cu, _make
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
