"""Joining partial attention states by their base-2 log-sum-exps, against the formula in 64 bits.

Tolerance, element by element: the weights are exp2 of a difference (rounded, a few 2^-23 of the weight
in all), at most eight products and sums and one division follow: less than 2^-20 of
sum_i share_i |O_i|, and a bf16 output is off by at most 2^-8 of its value more.  The log-sum-exp is
rounded once (2^-24 of it) after log2 of a sum that is off by less than 2^-20 of itself.
"""
import itertools
import math

import pytest
import torch

from dual_b200 import ops
from oracle import attention as OA

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


def merged64(states, lses):
    o, l = torch.stack([s.double() for s in states]), torch.stack(lses).double()
    top = l.amax(0)
    top = torch.where(top == -math.inf, 0.0, top)
    w = torch.exp2(l - top)
    total = w.sum(0)
    share = w / torch.where(total > 0, total, 1.0)
    terms = torch.where(w[..., None] > 0, share[..., None] * o, 0.0)
    return terms.sum(0), terms.abs().sum(0), top + torch.log2(total)


def close(out, lse, want):
    ref, size, ref_lse = want
    half_step = 2.0 ** -8 if out.dtype == torch.bfloat16 else 2.0 ** -24
    off = (out.double() - ref).abs()
    assert bool((off <= half_step * ref.abs() + 2.0 ** -20 * size).all()), float(off.max())
    if lse is not None:
        seen = ref_lse > -math.inf
        assert bool((lse[~seen] == -math.inf).all())
        off = (lse.double() - ref_lse)[seen].abs()
        assert bool((off <= 2.0 ** -23 * ref_lse[seen].abs() + 2.0 ** -20).all()), float(off.max())


def make(T, n, dtype, seed, empty=True):
    g = torch.Generator(device=DEV).manual_seed(seed)
    mk = lambda *s: torch.empty(s, dtype=torch.float32, device=DEV).normal_(generator=g)  # noqa: E731
    states = [mk(T, 32, 128).to(dtype) for _ in range(n)]
    lses = [4 * mk(T, 32) + 9 for _ in range(n)]
    if empty and T:
        for s, l in zip(states, lses):  # rows no key reached: whatever their values are, they count nothing
            gone = torch.rand((T, 32), generator=g, device=DEV) < 0.25
            l[gone] = -math.inf
            s[gone] = float("nan")
    return states, lses


@pytest.mark.parametrize("T,n", [(1, 1), (1, 2), (5, 2), (33, 3), (257, 8), (1000, 5)])
@pytest.mark.parametrize("dtype,out_dtype", list(itertools.product([torch.bfloat16, torch.float32], repeat=2)))
def test_merge_matches_64_bits(T, n, dtype, out_dtype):
    states, lses = make(T, n, dtype, seed=T + n)
    out = torch.empty((T, 32, 128), dtype=out_dtype, device=DEV)
    lse = torch.empty((T, 32), dtype=torch.float32, device=DEV)
    ops.merge_attention_states(states, lses, out, lse)
    close(out, lse, merged64(states, lses))


def test_rows_that_no_state_saw_are_zero():
    states, lses = make(4, 3, torch.bfloat16, seed=1, empty=False)
    for s, l in zip(states, lses):
        l[1] = -math.inf
        s[1] = float("inf")
    out = torch.full((4, 32, 128), 5.0, dtype=torch.bfloat16, device=DEV)
    lse = torch.zeros((4, 32), dtype=torch.float32, device=DEV)
    ops.merge_attention_states(states, lses, out, lse)
    assert bool((out[1] == 0).all()) and bool((lse[1] == -math.inf).all())
    close(out, lse, merged64(states, lses))


def test_far_apart_and_large_log_sum_exps():
    """Weights from 1 to below the smallest float, and log-sum-exps whose powers overflow."""
    states, lses = make(6, 4, torch.float32, seed=2, empty=False)
    for i, l in enumerate(lses):
        l.add_(torch.tensor([0.0, 60.0 * i, -400.0 * i, 5000.0, -5000.0, 150.0 * i], device=DEV)[:, None])
    out = torch.empty((6, 32, 128), dtype=torch.float32, device=DEV)
    lse = torch.empty((6, 32), dtype=torch.float32, device=DEV)
    ops.merge_attention_states(states, lses, out, lse)
    # log-sum-exps of about 5000 are themselves only known to 2^-12: the weights follow from the given values
    close(out, lse, merged64(states, lses))


@pytest.mark.parametrize("which", [0, 2])
def test_in_place(which):
    states, lses = make(70, 3, torch.bfloat16, seed=3)
    want = merged64(states, lses)
    ops.merge_attention_states(states, lses, states[which], lses[which])
    close(states[which], lses[which], want)


def test_strided_states_and_output_without_lse():
    """States side by side in one buffer, the output between them; a head stride of its own."""
    g = torch.Generator(device=DEV).manual_seed(7)
    buf = torch.empty((21, 3, 32, 128), dtype=torch.bfloat16, device=DEV).normal_(generator=g)
    wide = torch.empty((21, 32, 256), dtype=torch.bfloat16, device=DEV).normal_(generator=g)
    states = [buf[:, 0], wide[:, :, 128:], buf[:, 2]]
    lses = [torch.randn((21, 32), device=DEV) for _ in states]
    want, kept = merged64(states, lses), buf.clone()
    ops.merge_attention_states(states, lses, buf[:, 1])
    close(buf[:, 1], None, want)
    assert torch.equal(buf[:, 0], kept[:, 0]) and torch.equal(buf[:, 2], kept[:, 2])


def test_not_a_number_stays_in_its_row():
    states, lses = make(3, 2, torch.bfloat16, seed=5, empty=False)
    states[0][1, 4, 9] = float("nan")
    lses[1][2, 7] = float("nan")
    out = torch.empty((3, 32, 128), dtype=torch.bfloat16, device=DEV)
    lse = torch.empty((3, 32), dtype=torch.float32, device=DEV)
    ops.merge_attention_states(states, lses, out, lse)
    bad = torch.zeros((3, 32, 128), dtype=torch.bool, device=DEV)
    bad[1, 4, 9] = True
    bad[2, 7] = True
    assert torch.equal(out.isnan(), bad)
    assert bool(lse[2, 7].isnan()) and int(lse.isnan().sum()) == 1


def test_matches_the_oracle_merge_and_replays():
    states, lses = make(12, 2, torch.bfloat16, seed=6, empty=False)
    out = torch.empty((12, 32, 128), dtype=torch.bfloat16, device=DEV)
    lse = torch.empty((12, 32), dtype=torch.float32, device=DEV)
    graph = torch.cuda.CUDAGraph()
    stream = torch.cuda.Stream(DEV)
    stream.wait_stream(torch.cuda.current_stream(DEV))
    with torch.cuda.graph(graph, stream=stream):
        ops.merge_attention_states(states, lses, out, lse)
    for _ in range(2):
        states[0].normal_()
        lses[1].normal_()
        graph.replay()
        ref, ref_lse = OA.merge_states(states[0], lses[0], states[1], lses[1])
        torch.testing.assert_close(out.float(), ref, atol=2e-3, rtol=1e-2)
        torch.testing.assert_close(lse, ref_lse, atol=2e-3, rtol=1e-2)


def test_no_tokens():
    empty = torch.empty((0, 32, 128), dtype=torch.bfloat16, device=DEV)
    ops.merge_attention_states([empty], [torch.empty((0, 32), device=DEV)], empty.clone())
