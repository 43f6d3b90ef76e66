"""The host plan of a decode with shared prefixes, and what that decode refuses (no GPU)."""
import ctypes as C
import random

import pytest
import torch

from dual_b200 import SharedPrefixDecodeWrapper, _lib, ops


def read(plan):
    w = plan.tolist()
    ctas, segments, requests, blocks = w[1:5]
    assert 1 <= w[7] <= ctas
    at = 8 + 12 * ctas
    more = [w[at + 8 * i:at + 8 * i + 8] for i in range(segments)]
    cta, seg = [0], []
    for c in reversed(range(ctas)):  # a CTA's record holds its first segment, the others stand behind the records
        count, second, _, _, *first = w[8 + 12 * c:20 + 12 * c]
        mine = [first] + more[second:second + count - 1] if count else []
        assert len(mine) == count
        deep = all(s[1] <= 32 for s in mine)
        assert all(bool(s[6] & 2) == deep for s in mine)
        seg += mine
        cta.append(len(seg))
    assert len(more) == sum(max(0, b - a - 1) for a, b in zip(cta, cta[1:]))
    at += 8 * segments
    req = [w[at + 2 * i:at + 2 * i + 2] for i in range(requests)]
    at = (at + 2 * requests + 3) // 4 * 4
    job = [w[at + 4 * i:at + 4 * i + 4] for i in range(8 * blocks)]
    assert at + 32 * blocks == len(w)
    return w[5] | (w[6] << 32), cta, seg, req, job


@pytest.mark.parametrize("seed", range(40))
def test_segments_cover_every_prefix_once_and_states_do_not_overlap(seed):
    rng = random.Random(seed)
    groups = rng.randint(1, 6)
    sizes = [rng.choice([0, 1, 3, 32, 33, 64, 65, 130]) for _ in range(groups)]
    prefixes = [rng.choice([0, 1, 127, 128, 129, 500, 5000]) for _ in range(groups)]
    gi, pi = [0], [0]
    for s, p in zip(sizes, prefixes):
        gi.append(gi[-1] + s)
        pi.append(pi[-1] + p)
    plan = ops.shared_prefix_plan(gi, pi, rng.choice([1, 2, 3, 20, 148]), rng.choice([-1, 0, 1, 300, 100000]))
    size, cta, seg, req, job = read(plan)
    assert cta[0] == 0 and cta[-1] == len(seg) and cta == sorted(cta) and len(req) == gi[-1]
    seen, places = {}, []
    for tok0, ntok, head, first, last, off, flags, _ in seg:
        assert first < last and 0 < ntok <= 64
        places.append((off, off + 132 * ntok))
        for t in range(tok0, tok0 + ntok):
            seen.setdefault((t, head), []).append((first, last, off, t - tok0, flags))
    places.sort()
    assert all(a[1] <= b[0] for a, b in zip(places, places[1:])) and (not places or places[-1][1] <= size)
    for g in range(groups):
        for t in range(gi[g], gi[g + 1]):
            for h in range(8):
                mine = sorted(seen.get((t, h), []))
                if prefixes[g] == 0:
                    assert not mine and req[t][0] == -1
                    continue
                assert mine[0][0] == pi[g] and mine[-1][1] == pi[g + 1]
                assert all(a[1] == b[0] for a, b in zip(mine, mine[1:]))
                block, local = req[t]
                off, count, ntok, _ = job[block * 8 + h]
                assert count == len(mine)
                for i, m in enumerate(mine):
                    assert m[2] == off + i * 132 * ntok and m[3] == local
    assert ops.shared_prefix_workspace_size(plan) >= 16 * size + 8 * 132 * 16 * (gi[-1] + len(cta) - 1)


def loads(plan):
    """What each CTA has of the prefixes, in the planner's ns, and the CTAs that have own entries only."""
    words = plan.tolist()
    _, cta, seg, _, _ = read(plan)
    ns = []
    for a, b in zip(cta, cta[1:]):
        tiles = lambda s: -(-(s[4] - s[3]) // 128) * (1350 if s[1] <= 32 else 2400)  # noqa: E731
        ns.append(5000 + sum(3000 + tiles(s) for s in seg[a:b]) if b > a else 0)
    return ns, words[7]


@pytest.mark.parametrize("batch,prefix", [(16, 32768), (64, 32768), (200, 32768), (300, 500)])
def test_work_is_even(batch, prefix):
    """No CTA has more than its start, the even share of what there is, a tile and a segment."""
    ns, own = loads(ops.shared_prefix_plan([0, batch], [0, prefix], 148, 0))
    assert own == 148 and max(ns) <= 5000 + sum(max(0, n - 5000) for n in ns) / 148 + 2400 + 3000


@pytest.mark.parametrize("batch,prefix,entries", [(16, 32768, 2000), (64, 32768, 16000), (64, 4096, 2000), (3, 500, 60)])
def test_own_entries_get_their_share_of_the_ctas(batch, prefix, entries):
    """Apart from the prefixes' CTAs, and done at about the same time where there are many of them."""
    ns, own = loads(ops.shared_prefix_plan([0, batch], [0, prefix], 148, entries))
    assert own < 148 and all(n == 0 for n in sorted(ns)[:own])
    own_ns = (entries // 16 + batch // 2 + 1) * 1100 + batch * 700
    assert 4000 + own_ns / own <= max(ns) + 3000 + 2400
    # not known: every CTA does both
    assert loads(ops.shared_prefix_plan([0, batch], [0, prefix], 148))[1] == 148


def test_plan_refusals():
    for gi, pi, said in [([0, 2, 1], [0, 5, 6], "negative"), ([0, 2], [0, -1], "negative"), ([1, 2], [0, 5], "start at 0"),
                         ([0, 2], [3, 5], "start at 0")]:
        with pytest.raises(_lib.DualError, match=said):
            ops.shared_prefix_plan(gi, pi, 8)
    with pytest.raises(ValueError, match="one entry per group"):
        ops.shared_prefix_plan([0, 2], [0, 1, 2], 8)
    with pytest.raises(ValueError, match="integers"):
        ops.shared_prefix_plan(torch.tensor([0.0, 2.0]), [0, 1], 8)
    with pytest.raises(_lib.DualError, match="plan"):
        ops.shared_prefix_plan([0, 2], [0, 5], -3)
    with pytest.raises(_lib.DualError, match="not a shared-prefix plan"):
        ops.shared_prefix_workspace_size(torch.zeros(40, dtype=torch.int32))
    good = ops.shared_prefix_plan([0, 2], [0, 5], 8)
    with pytest.raises(_lib.DualError, match="not a shared-prefix plan"):
        ops.shared_prefix_workspace_size(good[:-1])
    # a list too short for the plan is left alone
    lib, n, few = _lib.load(), C.c_int64(0), torch.full((4,), -9, dtype=torch.int32)
    gi, pi = torch.tensor([0, 2], dtype=torch.int32), torch.tensor([0, 5], dtype=torch.int32)
    assert lib.dual_shared_prefix_plan(gi.data_ptr(), pi.data_ptr(), 1, 8, -1, few.data_ptr(), 4, C.byref(n)) == 0
    assert n.value == good.numel() and few.tolist() == [-9] * 4


def decode_args(B=3, capacity=10):
    bf = torch.bfloat16
    plan = ops.shared_prefix_plan([0, B], [0, 4], 8)
    return dict(q=torch.zeros((B, 32, 128), dtype=bf), k_local=torch.zeros((capacity + 1, 8, 128), dtype=bf),
                v_local=torch.zeros((capacity + 1, 8, 128), dtype=bf), local_capacity=capacity, peer_k=[], peer_v=[],
                prefix_indices=torch.zeros(4, dtype=torch.int32), kv_indptr=torch.zeros(B + 1, dtype=torch.int32),
                unified_indices=torch.zeros(1, dtype=torch.int32), sm_scale=0.1, plan=plan,
                out=torch.zeros((B, 32, 128), dtype=bf), lse=None,
                workspace=torch.zeros(ops.shared_prefix_workspace_size(plan), dtype=torch.uint8), num_ctas=8)


@pytest.mark.parametrize("change,said", [
    (dict(q=torch.zeros((3, 16, 128), dtype=torch.bfloat16)), "q must"),
    (dict(q=torch.zeros((3, 32, 128))), "q must"),
    (dict(out=torch.zeros((4, 32, 128), dtype=torch.bfloat16)), "out must"),
    (dict(prefix_indices=torch.zeros(4, dtype=torch.int64)), "prefix_indices must"),
    (dict(unified_indices=torch.zeros(8, dtype=torch.int32)[::2]), "unified_indices must"),
    (dict(kv_indptr=torch.zeros(3, dtype=torch.int32)), "kv_indptr too short"),
    (dict(plan=torch.zeros((4, 4), dtype=torch.int32)), "plan must"),
    (dict(lse=torch.zeros((3, 16))), "lse must"),
    (dict(local_capacity=11), "local_capacity"),
    (dict(v_local=torch.zeros((9, 8, 128), dtype=torch.bfloat16)), "pools must share"),
    (dict(peer_k=[torch.zeros((2, 8, 128), dtype=torch.bfloat16)]), "count mismatch"),
    (dict(peer_k=[torch.zeros((2, 8, 128), dtype=torch.bfloat16)] * 9,
          peer_v=[torch.zeros((2, 8, 128), dtype=torch.bfloat16)] * 9), "at most 8"),
    (dict(workspace=torch.zeros((64, 64), dtype=torch.uint8)[:, ::2]), "workspace must"),
    (dict(), "CUDA tensors"),
])
def test_decode_refusals(change, said):
    with pytest.raises(ValueError, match=said):
        ops.shared_prefix_decode(**{**decode_args(), **change})


def test_c_abi_refusals_come_before_any_launch():
    lib = _lib.load()
    two = (C.c_void_p * 8)(*[16] * 8)

    def call(q=256, qs=4096, qh=128, k=256, stride=2048, capacity=9, peers=0, pstride=2048, slots=4, prefix=16, n_prefix=4,
             kv=16, idx=16, n_idx=4, batch=2, scale=0.1, plan=256, words=104, out=256, os=4096, oh=128, ws=256,
             bytes_=1 << 24, ctas=8):
        rc = lib.dual_shared_prefix_decode(q, qs, qh, k, 256, stride, capacity, two, two, peers, pstride, slots, prefix,
                                           n_prefix, kv, idx, n_idx, batch, scale, plan, words, out, os, oh, None, ws,
                                           bytes_, ctas, -1, None)
        return rc, lib.dual_last_error().decode()

    assert call(batch=0) == (0, "")
    for change, code, said in [
            (dict(batch=-1), 1, "batch"), (dict(q=None), 1, "null"), (dict(plan=None), 1, "null"), (dict(ws=None), 1, "null"),
            (dict(prefix=None), 1, "index list"), (dict(idx=None), 1, "index list"), (dict(peers=9), 1, "num_peers"),
            (dict(stride=2040), 1, "slot stride"), (dict(capacity=-1), 1, "local_capacity"), (dict(qh=132), 1, "q/out"),
            (dict(out=264), 1, "q/out"), (dict(peers=2, pstride=1024), 1, "peer banks"), (dict(peers=1, slots=0), 1, "peer banks"),
            (dict(scale=0.0), 1, "sm_scale"), (dict(scale=float("nan")), 1, "sm_scale"), (dict(words=4), 1, "plan"),
            (dict(plan=260), 1, "plan"), (dict(words=103), 1, "for 8 CTAs"), (dict(ctas=0), 1, "num_ctas"), (dict(bytes_=1000), 3, "workspace too small"),
            (dict(ws=320), 1, "256-byte")]:
        rc, msg = call(**change)
        assert rc == code and said in msg, (change, rc, msg)


def test_wrapper_refusals():
    ws = torch.zeros(1 << 20, dtype=torch.uint8)
    with pytest.raises(ValueError, match="NHD"):
        SharedPrefixDecodeWrapper(ws, "HND")
    with pytest.raises(ValueError, match="graphs need"):
        SharedPrefixDecodeWrapper(ws, use_cuda_graph=True)
    w = SharedPrefixDecodeWrapper(ws, num_ctas=8)
    lists = (torch.zeros(4, dtype=torch.int32), torch.zeros(4, dtype=torch.int32), torch.zeros(0, dtype=torch.int32))
    with pytest.raises(ValueError, match="32 q heads"):
        w.plan([0, 3], [0, 4], *lists, 16, 8, 128, 1)
    with pytest.raises(ValueError, match="requests"):
        w.plan([0, 5], [0, 4], *lists, 32, 8, 128, 1)
    with pytest.raises(ValueError, match="shorter"):
        w.plan([0, 3], [0, 40], *lists, 32, 8, 128, 1)
    with pytest.raises(ValueError, match="too small"):
        SharedPrefixDecodeWrapper(ws[:4096], num_ctas=8).plan([0, 3], [0, 4], *lists, 32, 8, 128, 1)
    with pytest.raises(RuntimeError, match="plan"):
        w.run(torch.zeros((3, 32, 128), dtype=torch.bfloat16), (lists[0], lists[0]))
