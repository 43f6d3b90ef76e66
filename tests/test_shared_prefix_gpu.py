"""Decode of batches whose requests share prefixes, against attention over the joined lists in 64 bits.

Tolerance, element by element, with share_j the softmax weights and S = max_j scale log2(e) sum_d |q_d K_jd|:
  * a score is a sum of 128 products in fp32, off by at most 128 x 2^-23 S = 2^-16 S, so a weight and the sum
    below it are off by 2 ln 2 x 2^-16 S < 2^-15 S of themselves (the exponential's 2^-22 and the scale's
    rounding, 2^-23 S, are in that: S is at least 1 here);
  * P enters P V in bf16 (2^-8 of each weight) on prefixes of 1,024 entries and more, and as a bf16 pair (2^-16)
    otherwise;
  * P V adds 16 entries at a time to an fp32 sum: L / 16 additions, each off by at most 2^-23;
  * the output is rounded to bf16: 2^-8 of it.
The first three are relative to sum_j share_j |V_j|.  The LSE is off by 2^-15 S and a rounding.
"""
import math

import pytest
import torch

from dual_b200 import SharedPrefixDecodeWrapper, _lib, ops

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
SCALE = 128 ** -0.5
LOG2E = 1 / math.log(2)


def indptr(lengths):
    return torch.tensor([0] + list(lengths)).cumsum(0).to(torch.int32)


class Case:
    """Inputs with every row that no list names NaN, part of the rows on supplier banks."""

    def __init__(self, sizes, prefixes, suffixes, banks=0, remote=0.0, seed=0, q_std=1.0, capacity=None):
        g = self.g = torch.Generator(device=DEV).manual_seed(seed)
        self.sizes, self.prefixes, self.suffixes = sizes, prefixes, suffixes
        total = sum(prefixes) + sum(suffixes)
        far = torch.rand(total, generator=g, device=DEV) < (remote if banks else 0.0)
        n_far = int(far.sum())
        self.C = capacity or (total - n_far) + 37
        slots = n_far // max(banks, 1) + 3
        nan = lambda *s: torch.full(s, float("nan"), dtype=torch.bfloat16, device=DEV)  # noqa: E731
        self.k, self.v = nan(self.C + 1, 8, 128), nan(self.C + 1, 8, 128)
        self.k[0], self.v[0] = 0, 0  # the dummy slot is finite
        self.bk, self.bv = [nan(slots, 8, 128) for _ in range(banks)], [nan(slots, 8, 128) for _ in range(banks)]
        pages = torch.empty(total, dtype=torch.int32, device=DEV)
        pages[~far] = (torch.randperm(self.C, generator=g, device=DEV)[:total - n_far] + 1).int()
        pages[far] = (torch.randperm(max(banks, 1) * slots, generator=g, device=DEV)[:n_far] + self.C + 1).int()
        self.rows_k = torch.empty((total, 8, 128), dtype=torch.bfloat16, device=DEV).normal_(generator=g)
        self.rows_v = torch.empty((total, 8, 128), dtype=torch.bfloat16, device=DEV).normal_(generator=g)
        self.far, self.pages = far, pages
        self.put()
        self.prefix_pages, self.own_pages = pages[:sum(prefixes)].clone(), pages[sum(prefixes):].clone()
        self.gi, self.pi, self.ii = indptr(sizes), indptr(prefixes), indptr(suffixes)
        self.q = torch.empty((sum(sizes), 32, 128), dtype=torch.bfloat16, device=DEV).normal_(0, q_std, generator=g)

    def put(self):
        """The rows into the places that the pages name."""
        far, pages, C = self.far, self.pages.long(), self.C
        for pool, banks, rows in ((self.k, self.bk, self.rows_k), (self.v, self.bv, self.rows_v)):
            pool[pages[~far]] = rows[~far]
            for i, bank in enumerate(banks):
                here = far & ((pages - C - 1) % len(banks) == i)
                bank[(pages[here] - C - 1) // len(banks)] = rows[here]

    def peers(self):
        return [t for pair in zip(self.bk, self.bv) for t in pair]

    def plan(self, num_ctas=0, own=None):
        return ops.shared_prefix_plan(self.gi, self.pi, num_ctas, sum(self.suffixes) if own is None else own)

    def run(self, num_ctas=0, q=None, out=None, workspace=None, own=None):
        plan = self.plan(num_ctas, own)
        q = self.q if q is None else q
        B = q.shape[0]
        out = torch.full((B, 32, 128), 7.0, dtype=torch.bfloat16, device=DEV) if out is None else out
        lse = torch.full((B, 32), 7.0, dtype=torch.float32, device=DEV)
        ws = workspace
        if ws is None:  # partial states start as NaN: any that is read without being written shows
            ws = torch.full((ops.shared_prefix_workspace_size(plan) // 4,), float("nan"), dtype=torch.float32, device=DEV)
        ops.status_clear(ws)
        ops.shared_prefix_decode(q, self.k, self.v, self.C, self.bk, self.bv, self.prefix_pages, self.ii.to(DEV),
                                 self.own_pages, SCALE, plan.to(DEV), out, lse, ws, num_ctas)
        torch.cuda.synchronize()
        self.status = int(ws.view(torch.int32)[0])
        return out, lse

    def expect(self, q=None):
        q = self.q if q is None else q
        B = q.shape[0]
        ref = torch.zeros((B, 32, 128), dtype=torch.float64, device=DEV)
        size, lse = torch.zeros_like(ref), torch.full((B, 32), -math.inf, dtype=torch.float64, device=DEV)
        tol = torch.zeros((B, 32), dtype=torch.float64, device=DEV)  # relative, of weights and sums
        slack = torch.zeros((B, 32), dtype=torch.float64, device=DEV)  # of the log-sum-exp
        own0 = sum(self.prefixes)
        for grp, prefix in enumerate(self.prefixes):
            for b in range(int(self.gi[grp]), int(self.gi[grp + 1])):
                rows = torch.cat([torch.arange(int(self.pi[grp]), int(self.pi[grp + 1])),
                                  torch.arange(own0 + int(self.ii[b]), own0 + int(self.ii[b + 1]))]).to(DEV)
                if rows.numel() == 0:
                    continue
                k, v = self.rows_k[rows].double(), self.rows_v[rows].double()
                qb = q[b].double().view(8, 4, 128)
                score = torch.einsum("hgd,lhd->hgl", qb, k) * SCALE
                share = score.softmax(-1)
                ref[b] = torch.einsum("hgl,lhd->hgd", share, v).reshape(32, 128)
                size[b] = torch.einsum("hgl,lhd->hgd", share, v.abs()).reshape(32, 128)
                lse[b] = (score.logsumexp(-1) * LOG2E).reshape(32)
                S = (torch.einsum("hgd,lhd->hgl", qb.abs(), k.abs()).amax(-1) * SCALE * LOG2E).reshape(32)
                slack[b] = 2.0 ** -15 * S.clamp(min=1)
                tol[b] = slack[b] + (2.0 ** -8 if prefix >= 1024 else 2.0 ** -16) + rows.numel() / 16 * 2.0 ** -23
        return ref, size, lse, tol, slack

    def check(self, out, lse, q=None, rows=None):
        ref, size, ref_lse, tol, slack = self.expect(q)
        rows = slice(None) if rows is None else rows
        off = (out.double() - ref).abs()[rows]
        bound = (2.0 ** -8 * ref.abs() + tol[..., None] * size)[rows]
        assert bool((off <= bound).all()), float((off - bound).max())
        if lse is not None:
            empty = (ref_lse == -math.inf)[rows]
            assert torch.equal(lse[rows] == -math.inf, empty)
            off = (lse.double() - ref_lse)[rows].masked_fill(empty, 0.0).abs()
            assert bool((off <= slack[rows] + 2.0 ** -23 * ref_lse[rows].abs()).all()), float(off.max())


def mixed(n, seed=0):
    some = [0, 1, 15, 16, 17, 40, 100]
    return [some[(i * 5 + seed) % len(some)] for i in range(n)]


@pytest.mark.parametrize("batch", [1, 2, 31, 32, 33, 64, 65, 97, 130])
@pytest.mark.parametrize("prefix", [1, 127, 128, 129, 257, 1023, 1024, 2500])
def test_one_group(batch, prefix):
    c = Case([batch], [prefix], mixed(batch, prefix), seed=batch + prefix)
    out, lse = c.run()
    assert c.status == 0
    c.check(out, lse)


@pytest.mark.parametrize("num_ctas", [1, 2, 7, 37, 148, 300])
def test_any_number_of_ctas(num_ctas):
    """From one CTA that works on every job to more CTAs than units."""
    c = Case([5, 0, 40, 70], [700, 300, 1500, 129], mixed(115), banks=3, remote=0.2, seed=num_ctas)
    out, lse = c.run(num_ctas)
    assert c.status == 0
    c.check(out, lse)


@pytest.mark.parametrize("own", [-1, 0, 5, 4000, 10 ** 7])
def test_plans_for_other_own_lengths(own):
    """The plan's idea of the own entries decides how many CTAs they get, not the result."""
    c = Case([20, 60], [1100, 300], mixed(80), seed=17)
    out, lse = c.run(own=own)
    assert c.status == 0
    c.check(out, lse)


@pytest.mark.parametrize("sizes,prefixes,suffixes", [
    ([3], [0], [5, 0, 1]),                           # a prefix of no entries
    ([2, 2], [0, 10], [0, 3, 0, 0]),                 # a request with nothing at all
    ([4], [300], [0, 0, 0, 0]),                      # no entries behind the prefix
    ([3, 2], [0, 0], [0, 0, 0, 0, 0]),               # nothing anywhere
    ([0, 3, 0], [50, 20, 30], [1, 0, 2]),            # groups without requests
    ([1, 1, 1, 1, 1], [1, 2, 3, 4, 5], [1, 1, 1, 1, 1]),
    ([6], [40], [3000, 0, 1, 0, 17, 900]),           # own entries that are split over CTAs
    ([300], [64], [1] * 300),                        # many requests per CTA
    ([1, 200], [20000, 10], [3] * 201),              # one request with most of the states, more than the join's room
    ([2], [9], [30000, 0]),                          # the same with own entries
])
def test_empty_and_uneven_lists(sizes, prefixes, suffixes):
    c = Case(sizes, prefixes, suffixes, seed=len(suffixes))
    out, lse = c.run()
    assert c.status == 0
    c.check(out, lse)


@pytest.mark.parametrize("banks", [1, 3, 8])
def test_rows_on_supplier_banks(banks):
    c = Case([20, 45], [1100, 700], mixed(65, banks), banks=banks, remote=0.3, seed=banks)
    out, lse = c.run()
    assert c.status == 0
    c.check(out, lse)


@pytest.mark.parametrize("batch", [8, 40])
def test_growing_maximum_and_peaked_weights(batch):
    """Scores that rise along the prefix by far more than 2^8 (the running output is rescaled many times), and
    queries whose weights sit on a few entries."""
    c = Case([batch], [3000], [30] * batch, seed=2, q_std=4.0)
    ramp = torch.linspace(0.05, 3.0, 3000, device=DEV)[:, None, None]
    c.rows_k[:3000] = (c.rows_k[:3000].float().abs() * ramp).bfloat16()
    c.q.abs_()
    c.put()
    out, lse = c.run()
    assert c.status == 0
    c.check(out, lse)


def test_same_as_decode_over_the_joined_lists():
    c = Case([9, 30], [800, 1200], mixed(39), banks=2, remote=0.1, seed=5)
    out, lse = c.run()
    lists = []
    for grp in range(2):
        for b in range(int(c.gi[grp]), int(c.gi[grp + 1])):
            lists += [c.prefix_pages[int(c.pi[grp]):int(c.pi[grp + 1])], c.own_pages[int(c.ii[b]):int(c.ii[b + 1])]]
    lengths = [len(lists[2 * i]) + len(lists[2 * i + 1]) for i in range(39)]
    ref, ref_lse = torch.empty_like(out), torch.empty_like(lse)
    ws = torch.zeros(ops.decode_workspace_size(39, ops.default_ctas(0)), dtype=torch.uint8, device=DEV)
    ops.tiered_decode(c.q, c.k, c.v, c.C, c.bk, c.bv, indptr(lengths).to(DEV), torch.cat(lists), SCALE, ref, ref_lse, ws)
    torch.testing.assert_close(out.float(), ref.float(), atol=2e-3, rtol=1e-2)
    torch.testing.assert_close(lse, ref_lse, atol=2e-3, rtol=1e-2)


def test_same_answer_every_time():
    c = Case([50, 7], [900, 2000], mixed(57), seed=8)
    first, again = c.run(), c.run()
    assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


def test_strided_queries_outputs_and_pools():
    c = Case([11], [400], mixed(11), seed=9)
    qkv = torch.empty((11, 6144), dtype=torch.bfloat16, device=DEV).normal_(generator=c.g)
    q = qkv[:, :4096].view(11, 32, 128)
    out = torch.zeros((11, 32, 256), dtype=torch.bfloat16, device=DEV)
    both = torch.stack([c.k, c.v], 1)
    c.k, c.v = both[:, 0], both[:, 1]
    _, lse = c.run(q=q, out=out[:, :, :128])
    assert c.status == 0
    c.check(out[:, :, :128], lse, q=q)
    assert not bool(out[:, :, 128:].any())


def test_not_a_number_stays_with_its_request():
    """A NaN among one request's own values, an infinity among another's: their neighbours, whose tiles come
    after theirs in the same buffers, keep their results."""
    c = Case([6], [200], [5, 40, 3, 21, 2, 1], seed=12)
    own = 200
    c.rows_v[own + 5 + 33, 2, 7] = float("nan")
    c.rows_v[own + 5 + 40 + 3 + 20, 4, 9] = float("inf")
    c.put()
    out, lse = c.run(num_ctas=1)
    assert c.status == 0
    bad = torch.zeros((6, 32, 128), dtype=torch.bool, device=DEV)
    bad[1, 8:12, 7] = bad[3, 16:20, 9] = True
    assert torch.equal(~out.isfinite(), bad)
    c.check(out, lse, rows=[0, 2, 4, 5])


def test_queries_that_are_not_numbers_stay_in_their_row():
    c = Case([40], [300], [7] * 40, seed=13)
    c.q[3, 5, 0] = float("nan")
    out, lse = c.run()
    bad = torch.zeros((40, 32), dtype=torch.bool, device=DEV)
    bad[3, 5] = True
    assert torch.equal(out.isnan().any(-1), bad) and torch.equal(lse.isnan(), bad)
    c.q[3, 5, 0] = 0.0
    rows = [i for i in range(40) if i != 3]
    c.check(out, lse, rows=rows)


def test_bad_remote_pages_are_recorded():
    c = Case([3], [100], [4, 4, 4], banks=1, remote=0.2, seed=3)
    c.prefix_pages[50] = c.C + 1 + 10 * c.bk[0].shape[0]
    out, _ = c.run()
    assert c.status == 0x2 and bool(out.isfinite().all())
    c.prefix_pages[50], c.own_pages[5] = 1, -4
    c.run()
    assert c.status == 0x2


def test_a_plan_of_another_batch_is_recorded():
    c = Case([4], [100], [3, 3, 3, 3], seed=4)
    other = ops.shared_prefix_plan([0, 5], [0, 100])
    ws = torch.zeros(ops.shared_prefix_workspace_size(other), dtype=torch.uint8, device=DEV)
    out = torch.empty((4, 32, 128), dtype=torch.bfloat16, device=DEV)
    args = (c.q, c.k, c.v, c.C, [], [], c.prefix_pages, c.ii.to(DEV), c.own_pages, SCALE)
    ops.shared_prefix_decode(*args, other.to(DEV), out, None, ws)
    assert int(ws.view(torch.int32)[0]) == 0x10
    longer = ops.shared_prefix_plan([0, 4], [0, 300])  # entries past the end of the index list
    ops.status_clear(ws)
    big = torch.zeros(ops.shared_prefix_workspace_size(longer), dtype=torch.uint8, device=DEV)
    ops.shared_prefix_decode(*args, longer.to(DEV), out, None, big)
    assert int(big.view(torch.int32)[0]) == 0x10
    # words that are no plan: only the requests' own entries are seen
    ops.status_clear(ws)
    ops.shared_prefix_decode(*args, torch.zeros(1 << 12, dtype=torch.int32, device=DEV), out, None, ws)
    assert int(ws.view(torch.int32)[0]) == 0x10
    own = Case.__new__(Case)
    own.__dict__.update(c.__dict__)
    own.prefixes, own.rows_k, own.rows_v = [0], c.rows_k[100:], c.rows_v[100:]
    own.pi = indptr([0])
    own.check(out, None)
    # a workspace without room for the prefix's states
    plan = c.plan()
    with pytest.raises(_lib.DualError, match="plan for 148 CTAs"):  # fewer words than the CTAs' records
        ops.shared_prefix_decode(*args, plan.to(DEV)[:1000], out, None, ws, 148)
    small = torch.zeros(ops.decode_workspace_size(4, ops.default_ctas(0)) + 1024, dtype=torch.uint8, device=DEV)
    ops.shared_prefix_decode(*args, plan.to(DEV), out, None, small)
    assert int(small.view(torch.int32)[0]) == 0x10


def test_slots_past_four_gigabytes():
    c = Case([5], [300], [9] * 5, seed=6, capacity=(1 << 32) // 2048 + 4000)
    high = torch.arange(c.C - 344, c.C + 1, device=DEV)  # every page at the far end
    c.pages = high[torch.randperm(345, device=DEV)].int()
    c.put()
    c.prefix_pages, c.own_pages = c.pages[:300].clone(), c.pages[300:].clone()
    out, lse = c.run()
    assert c.status == 0
    c.check(out, lse)


def wrapper_for(c, graph=False, workspace=None, room=4096):
    buf = lambda n: torch.zeros(n, dtype=torch.int32, device=DEV)  # noqa: E731
    ws = torch.full((64 << 20,), 255, dtype=torch.uint8, device=DEV) if workspace is None else workspace
    if not graph:
        return SharedPrefixDecodeWrapper(ws)
    return SharedPrefixDecodeWrapper(ws, use_cuda_graph=True, paged_kv_indptr_buffer=buf(65),
                                     paged_kv_indices_buffer=buf(room), prefix_indices_buffer=buf(room),
                                     plan_buffer=buf(1 << 14))


def test_wrapper_tiered_and_local():
    c = Case([7, 35], [500, 1300], mixed(42), banks=2, remote=0.15, seed=21)
    w = wrapper_for(c)
    with pytest.raises(RuntimeError, match="plan"):
        w.run(c.q, (c.k, c.v))
    w.plan(c.gi, c.pi, c.prefix_pages, c.ii, c.own_pages, 32, 8, 128, 1)
    out, lse = w.run_return_lse(c.q, (c.k.unsqueeze(1), c.v.unsqueeze(1)), *c.peers(), c.prefix_pages, c.own_pages,
                                c.C, SCALE)
    c.check(out, lse)
    assert w.status() == 0
    c = Case([7, 35], [500, 1300], mixed(42), seed=22)
    w.plan(c.gi, c.pi, c.prefix_pages, c.ii, c.own_pages, 32, 8, 128, 1)
    c.check(w.run(c.q, torch.stack([c.k, c.v], 1).unsqueeze(2)), None)
    with pytest.raises(ValueError, match="42"):
        w.run(c.q[:3], (c.k, c.v))


def test_captured_run_follows_new_plans_and_shares_its_workspace():
    """Two captured graphs of one workspace, replayed in turn; between replays plan() brings other lists,
    other prefixes and other groups of the same batch."""
    torch.cuda.synchronize()
    workspace = torch.full((64 << 20,), 255, dtype=torch.uint8, device=DEV)
    sets = []
    for seed in (31, 32):
        c = Case([30, 10], [600, 900], mixed(40, seed), seed=seed)
        w = wrapper_for(c, True, workspace)
        w.plan(c.gi, c.pi, c.prefix_pages, c.ii, c.own_pages, 32, 8, 128, 1)
        pool = (torch.zeros((4096, 8, 128), dtype=torch.bfloat16, device=DEV),
                torch.zeros((4096, 8, 128), dtype=torch.bfloat16, device=DEV))
        q = torch.empty_like(c.q)
        out, lse = torch.empty_like(c.q), torch.empty((40, 32), device=DEV)
        w.run(q.copy_(c.q), pool, out=out, lse=lse, return_lse=True)  # first use outside the capture
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            w.run(q, pool, out=out, lse=lse, return_lse=True)
        sets.append((w, pool, q, out, lse, graph))
    for step in range(3):
        for i, (w, pool, q, out, lse, graph) in enumerate(sets):
            sizes, prefixes = [([30, 10], [600, 900]), ([1, 39], [0, 1025]), ([40, 0], [1700, 3])][step]
            c = Case(sizes, prefixes, mixed(40, step + i), seed=40 + 2 * step + i)
            w.plan(c.gi, c.pi, c.prefix_pages, c.ii, c.own_pages, 32, 8, 128, 1)
            pool[0][:c.C + 1], pool[1][:c.C + 1] = c.k, c.v
            q.copy_(c.q)
            for _ in range(2):
                out.fill_(7.0)
                graph.replay()
                c.check(out, lse)
            assert w.status() == 0


def test_on_a_side_stream_between_other_work():
    c = Case([33], [1500], mixed(33), seed=41)
    w = wrapper_for(c)
    stream = torch.cuda.Stream(DEV)
    stream.wait_stream(torch.cuda.current_stream(DEV))
    with torch.cuda.stream(stream):
        w.plan(c.gi, c.pi, c.prefix_pages, c.ii, c.own_pages, 32, 8, 128, 1)
        outs = []
        for _ in range(20):  # each run's queries are made right before it, each output changed right after
            q = c.q * 1
            out, lse = w.run_return_lse(q, (c.k, c.v), c.prefix_pages, c.own_pages, c.C, SCALE)
            outs.append((out * 1, lse * 1))
            q.zero_()
            out.zero_()
    stream.synchronize()
    for out, lse in outs:
        assert torch.equal(out, outs[0][0]) and torch.equal(lse, outs[0][1])
    c.check(*outs[0])


def test_two_calls_at_once():
    """Two batches on two streams, each with a workspace of its own, beside each other."""
    cases = [Case([40], [2000], mixed(40), seed=51), Case([10, 20], [900, 3000], mixed(30), banks=1, remote=0.2, seed=52)]
    wrappers = [wrapper_for(c) for c in cases]
    streams = [torch.cuda.Stream(DEV) for _ in cases]
    for c, w in zip(cases, wrappers):
        w.plan(c.gi, c.pi, c.prefix_pages, c.ii, c.own_pages, 32, 8, 128, 1)
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(15):
        for i, (c, w, stream) in enumerate(zip(cases, wrappers, streams)):
            with torch.cuda.stream(stream):
                outs[i].append(w.run_return_lse(c.q, (c.k, c.v), *c.peers(), c.prefix_pages, c.own_pages, c.C, SCALE))
    torch.cuda.synchronize()
    for c, w, many in zip(cases, wrappers, outs):
        assert w.status() == 0
        for out, lse in many:
            assert torch.equal(out, many[0][0]) and torch.equal(lse, many[0][1])
        c.check(*many[0])


def test_an_empty_batch():
    w = wrapper_for(Case([1], [5], [1], seed=1))
    none = torch.zeros(0, dtype=torch.int32, device=DEV)
    w.plan([0], [0], none, torch.zeros(1, dtype=torch.int32), none, 32, 8, 128, 1)
    pool = torch.zeros((4, 8, 128), dtype=torch.bfloat16, device=DEV)
    out, lse = w.run_return_lse(torch.empty((0, 32, 128), dtype=torch.bfloat16, device=DEV), (pool, pool))
    assert out.shape == (0, 32, 128) and lse.shape == (0, 32)
