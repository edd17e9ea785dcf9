"""The hand-over of the attention gradient's softmax warps (csrc/fw_prompt_grad.cu) in every order of events, on the CPU.

A warp waits for X of a step, waits for Y, gives Y back, stores P and dS and arrives at p_full; the Y warp forms the next Y
once all have given theirs back; the products' warp waits for p_full of a step before it reads what the warps stored, and then
forms X of the step after the next. Barriers are counters: the wait for the n-th use of one is over once n times as many
arrivals as it has warps have come. How many p_full barriers the steps go round on is read from the kernel."""

import re
from collections import deque
from pathlib import Path

import pytest

SOURCE = Path(__file__).resolve().parent.parent / 'flash_whisper_b200' / 'csrc' / 'fw_prompt_grad.cu'


def _read_too_early(bars, warps, steps):
    """Whether the products' warp can pass p_full of a step that some warp has not stored yet."""
    # (step, part) of each warp; steps of Y, of the products, of X formed; arrivals at each p_full, at y_free
    start = (((0, 0),) * warps, 0, 0, 2, (0,) * bars, 0)
    seen, todo = {start}, deque([start])
    while todo:
        at, y, done, x, p, free = todo.popleft()
        out = []
        for w, (j, part) in enumerate(at):
            if j == steps:
                continue
            if part == 0 and x > j:
                move = (j, 1), p, free
            elif part == 1 and y > j:
                move = (j, 2), p, free + 1
            elif part == 2:
                move = (j + 1, 0), tuple(n + (b == j % bars) for b, n in enumerate(p)), free
            else:
                continue
            out.append((at[:w] + move[:1] + at[w + 1:], y, done, x, *move[1:]))
        if y < steps and free >= warps * y:
            out.append((at, y + 1, done, x, p, free))
        if done < steps and p[done % bars] >= warps * (done // bars + 1):
            if any(j <= done for j, _ in at):
                return True
            out.append((at, y, done + 1, done + 3, p, free))
        for s in out:
            if s not in seen:
                seen.add(s)
                todo.append(s)
    assert any(s[2] == steps for s in seen), 'the steps never end'
    return False


@pytest.mark.parametrize('warps', [2, 3])
def test_gradient_products_wait_for_every_warp_of_their_step(warps):
    text = SOURCE.read_text()
    declared = re.search(r'__shared__[^;]*\bp_full(?:\[(\d+)\])?\s*[,;]', text)
    bars = int(declared.group(1) or 1)
    assert not _read_too_early(bars, warps, 6)
    assert re.search(r'mbar_wait_warp\(&p_full\[j & 1\], \(j >> 1\) & 1u\)', text) and 'g.p_full + (j & 1)' in text
    assert _read_too_early(1, warps, 6)  # what one barrier would allow
