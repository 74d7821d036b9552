"""Attention with score rules, drafted trees and acceptance at the ends of what their calls allow: streams,
lengths, positions, counts and arguments that the tests beside this file do not reach."""
from __future__ import annotations

import copy

import numpy as np
import pytest

from test_scores import PAIR_HALF, Batch, compare


def of_streams(b, n):
    """Batch b's first n sequences, on the same cache."""
    c, rows = copy.copy(b), int(b.rows[:n].sum())
    c.cached, c.rows, c.streams, c.q, c.k, c.v = b.cached[:n], b.rows[:n], b.streams[:n], b.q[:rows], b.k[:rows], b.v[:rows]
    return c


@pytest.mark.gpu
@pytest.mark.parametrize("scored", [True, False])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_first_token_calls_on_a_side_stream_beside_a_busy_default_stream(ptts, cuda, dtype, scored):
    """The merge counters of a cache's first token call, and of one with more rows, are zeros before its rows
    are cut and joined, whatever the default stream has to do. Bounds as for attend_scored's f32 outputs."""
    import torch
    side = torch.cuda.Stream()
    all43 = Batch(ptts, cuda, [5000, 3000, 700] + [900 + 9 * i for i in range(40)], [1] * 43, dtype=dtype, seed=2)
    a = torch.randn(8192, 8192, device=cuda).bfloat16()
    c = torch.empty_like(a)
    got = []
    for b in (of_streams(all43, 3), all43):
        out = torch.empty(len(b.q), 512, device=cuda)
        torch.cuda.synchronize()
        for _ in range(60):  # tens of milliseconds
            torch.mm(a, a, out=c)
        args = (b.kv, 0, b.q, b.k, b.v, b.streams, b.rows)
        ptts.attend_scored(*args, softcap=9.0, out=out, stream=side) if scored else ptts.attend(*args, out=out, stream=side)
        side.synchronize()
        got.append((out.clone(), *b.want(softcap=9.0 if scored else 0.0, half_p=PAIR_HALF)))
    all43.kv.check()
    for out, want, bound in got:
        compare(out, want, bound)
