"""Entries whose score is -inf (an infinite key) count nothing, wherever they stand: whole tiles of them, in front of
the finite ones or behind, a whole prefix, all of a request's own entries.  A request of which every score is -inf is
one without entries: output 0, log-sum-exp -inf, as where states are merged.

Tolerance as in test_shared_prefix_gpu, over the finite entries, the weights being bf16 pairs.
"""
import math

import pytest
import torch

from dual_b200 import ops
from test_shared_prefix_gpu import Case, DEV, LOG2E, SCALE

pytestmark = pytest.mark.gpu
INF = float("inf")


def gone_rows(c, gone):
    """Keys of the entries `gone` (a list of (first, last) among all rows) infinite, opposite to every query."""
    c.q[..., 0] = c.q[..., 0].abs() + 0.125
    dead = torch.zeros(c.rows_k.shape[0], dtype=torch.bool, device=DEV)
    for first, last in gone:
        dead[first:last] = True
    c.rows_k[dead, :, 0] = -INF
    c.put()
    return dead


def check(c, dead, out, lse):
    own0 = sum(c.prefixes)
    for grp in range(len(c.sizes)):
        for b in range(int(c.gi[grp]), int(c.gi[grp + 1])):
            rows = torch.cat([torch.arange(int(c.pi[grp]), int(c.pi[grp + 1])),
                              torch.arange(own0 + int(c.ii[b]), own0 + int(c.ii[b + 1]))]).to(DEV)
            rows = rows[~dead[rows]]
            if rows.numel() == 0:
                assert not bool(out[b].any()) and bool((lse[b] == -INF).all()), b
                continue
            k, v, q = c.rows_k[rows].double(), c.rows_v[rows].double(), c.q[b].double().view(8, 4, 128)
            score = torch.einsum("hgd,lhd->hgl", q, k) * SCALE
            share = score.softmax(-1)
            ref = torch.einsum("hgl,lhd->hgd", share, v).reshape(32, 128)
            size = torch.einsum("hgl,lhd->hgd", share, v.abs()).reshape(32, 128)
            ref_lse = (score.logsumexp(-1) * LOG2E).reshape(32)
            S = (torch.einsum("hgd,lhd->hgl", q.abs(), k.abs()).amax(-1) * SCALE * LOG2E).reshape(32).clamp(min=1)
            tol = 2.0 ** -15 * S + 2.0 ** -16 + rows.numel() / 16 * 2.0 ** -23
            off = (out[b].double() - ref).abs()
            assert bool((off <= 2.0 ** -8 * ref.abs() + tol[:, None] * size).all()), (b, float(off.max()))
            off = (lse[b].double() - ref_lse).abs()
            assert bool((off <= 2.0 ** -15 * S + 2.0 ** -23 * ref_lse.abs()).all()), (b, float(off.max()))


@pytest.mark.parametrize("batch", [1, 20, 32, 33, 64])
@pytest.mark.parametrize("first,last", [(0, 128), (0, 256), (128, 256), (0, 300), (100, 500), (512, 700), (0, 699), (0, 700)])
@pytest.mark.parametrize("num_ctas", [1, 0])
def test_part_of_a_prefix(batch, first, last, num_ctas):
    c = Case([batch], [700], [i % 3 for i in range(batch)], seed=batch + first)
    dead = gone_rows(c, [(first, last)])
    out, lse = c.run(num_ctas)
    assert c.status == 0
    check(c, dead, out, lse)


@pytest.mark.parametrize("prefix", [0, 90])
@pytest.mark.parametrize("num_ctas", [1, 3, 0])
def test_own_entries(prefix, num_ctas):
    """Tiles of 16: a first one, one in between, a last, all, and none, one request each."""
    c = Case([5], [prefix], [40, 60, 33, 48, 20], seed=3)
    at = [prefix, prefix + 40, prefix + 100, prefix + 133, prefix + 181]
    dead = gone_rows(c, [(at[0], at[0] + 16), (at[1] + 16, at[1] + 48), (at[2] + 32, at[2] + 33), (at[3], at[3] + 48)])
    out, lse = c.run(num_ctas)
    assert c.status == 0
    check(c, dead, out, lse)


def test_nothing_but_infinite_keys():
    c = Case([2, 40], [200, 1300], [5] * 42, banks=2, remote=0.2, seed=4)
    dead = gone_rows(c, [(0, c.rows_k.shape[0])])
    out, lse = c.run()
    assert c.status == 0
    check(c, dead, out, lse)


def test_positive_infinity_and_not_a_number_are_not_hidden():
    """A score of +inf has no softmax, nor has NaN: its request's heads are NaN, the others keep their results."""
    c = Case([3], [400], [20, 20, 20], seed=5)
    gone_rows(c, [])
    c.rows_k[400 + 17, 2, 0] = INF
    c.rows_k[420:440, 5, 3] = float("nan")
    c.put()
    out, lse = c.run(1)
    bad = torch.zeros((3, 32), dtype=torch.bool, device=DEV)
    bad[0, 8:12] = bad[1, 20:24] = True
    assert torch.equal(out.isnan().all(-1), bad) and torch.equal(out.isnan().any(-1), bad)
    c.check(out, lse, rows=[2])


def test_states_of_infinite_keys_merge():
    c = Case([6], [300], [10] * 6, seed=6)
    dead = gone_rows(c, [(0, 300)])
    only_prefix, no_own = Case.__new__(Case), torch.zeros(7, dtype=torch.int32)
    only_prefix.__dict__.update(c.__dict__, suffixes=[0] * 6, ii=no_own, own_pages=c.own_pages[:0])
    only_own = Case.__new__(Case)
    only_own.__dict__.update(c.__dict__, prefixes=[0], pi=torch.zeros(2, dtype=torch.int32), prefix_pages=c.prefix_pages[:0])
    a, la = only_prefix.run()
    b, lb = only_own.run()
    out, lse = torch.empty_like(a), torch.empty_like(la)
    ops.merge_attention_states([a, b], [la, lb], out, lse)
    whole, whole_lse = c.run()
    check(c, dead, whole, whole_lse)
    assert torch.equal(out, b) and torch.equal(lse, lb) and bool((la == -math.inf).all())
