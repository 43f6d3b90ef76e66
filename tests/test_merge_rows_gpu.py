"""Merges of enough tokens that a thread holds several rows (two of up to four states, four of up to two), at token
counts on both sides of where that begins and with a last block that is not full.  Tolerances and the definition in 64
bits are test_merge_gpu's."""
import math

import pytest
import torch

from dual_b200 import ops
from test_merge_gpu import DEV, close, make, merged64

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float32
# tokens from which on: bf16 1,184 (up to four states) and 2,368 (up to two), fp32 592 and 1,184
CASES = [(T, n, BF) for T in (1183, 1184, 1185, 1999) for n in (3, 4)]
CASES += [(T, n, BF) for T in (1185, 2367, 2368, 2369, 2371, 5001) for n in (1, 2)]
CASES += [(T, n, FP) for T in (591, 592, 593, 997) for n in (3, 4)]
CASES += [(T, n, FP) for T in (593, 1183, 1184, 1185, 1187, 2503) for n in (1, 2)]
CASES += [(2369, 5, BF), (1185, 5, FP)]


@pytest.mark.parametrize("out_dtype", [BF, FP])
@pytest.mark.parametrize("T,n,dtype", CASES)
def test_many_tokens(T, n, dtype, out_dtype):
    """A quarter of the rows of each state unseen (NaN there), and some that no state saw."""
    states, lses = make(T, n, dtype, seed=T + n)
    for l in lses:
        l[T // 2], l[-1, 5] = -math.inf, -math.inf
    out = torch.full((T, 32, 128), 5.0, dtype=out_dtype, device=DEV)
    lse = torch.full((T, 32), 5.0, dtype=FP, device=DEV)
    ops.merge_attention_states(states, lses, out, lse)
    assert bool((out[T // 2] == 0).all()) and bool((out[-1, 5] == 0).all())
    close(out, lse, merged64(states, lses))


@pytest.mark.parametrize("T,n,dtype", [(2369, 2, BF), (2371, 2, BF), (1185, 4, BF), (1187, 3, BF), (1185, 2, FP),
                                       (593, 4, FP)])
def test_many_tokens_in_place(T, n, dtype):
    """The output and its log-sum-exp in the place of a state's: threads past the last row read it once more."""
    for which in range(n):
        for _ in range(5):
            states, lses = make(T, n, dtype, seed=which)
            want = merged64(states, lses)
            ops.merge_attention_states(states, lses, states[which], lses[which])
            close(states[which], lses[which], want)


@pytest.mark.parametrize("T,n", [(2369, 2), (1185, 3)])
def test_many_tokens_strided(T, n):
    """States side by side in one buffer and in the second half of wider rows; the output between them."""
    g = torch.Generator(device=DEV).manual_seed(T)
    buf = torch.empty((T, 3, 32, 128), dtype=BF, device=DEV).normal_(generator=g)
    wide = torch.empty((T, 32, 256), dtype=BF, device=DEV).normal_(generator=g)
    states = [buf[:, 0], wide[:, :, 128:], buf[:, 2]][:n]
    lses = [torch.empty((T, 32), device=DEV).normal_(generator=g) for _ in states]
    want, kept, kept_wide = merged64(states, lses), buf.clone(), wide.clone()
    ops.merge_attention_states(states, lses, buf[:, 1])
    close(buf[:, 1], None, want)
    assert torch.equal(buf[:, ::2], kept[:, ::2]) and torch.equal(wide, kept_wide)


@pytest.mark.parametrize("T,n", [(40, 2), (2369, 2), (1185, 3)])
def test_side_by_side_within_a_head(T, n):
    """States and output in one buffer [T, 32, n + 1, 128]."""
    g = torch.Generator(device=DEV).manual_seed(T)
    buf = torch.empty((T, 32, n + 1, 128), dtype=BF, device=DEV).normal_(generator=g)
    states, out = list(buf.unbind(2)[:n]), buf[:, :, n]
    lses = [torch.empty((T, 32), device=DEV).normal_(generator=g) for _ in states]
    want, kept = merged64(states, lses), buf.clone()
    ops.merge_attention_states(states, lses, out)
    close(out, None, want)
    assert torch.equal(buf[:, :, :n], kept[:, :, :n])
