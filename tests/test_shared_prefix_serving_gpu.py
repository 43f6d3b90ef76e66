"""The three operators together, as a serving loop uses them: prompts rotated and stored, two groups of requests
that share prefixes decoded step by step (new tokens rotated and stored, then the shared-prefix decode), part of
the prefixes moved to supplier banks in between; history and chunk of an append joined; one step captured and
replayed.  Every attention output is checked against attention in 64 bits over the rows that the pools hold, and
those rows against the rotation in 64 bits."""
import math

import pytest
import torch

from dual_b200 import BatchPrefillWithPagedKVCacheWrapper, SharedPrefixDecodeWrapper, ops
from test_rope_kv_gpu import close as rope_close, rotate64, table

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
SCALE = 128 ** -0.5
CAP, BANKS, BANK_SLOTS = 6000, 2, 700


def attend64(q, k, v, seen=None):
    """q [n, 32, 128] over k / v [L, 8, 128]: (output, sum of share |v|, base-2 LSE); `seen` [n, L] masks."""
    n = q.shape[0]
    score = torch.einsum("nhgd,lhd->nhgl", q.double().view(n, 8, 4, 128), k.double()) * SCALE
    if seen is not None:
        score = score.masked_fill(~seen[:, None, None, :], -math.inf)
    share = score.softmax(-1)
    mix = lambda x: torch.einsum("nhgl,lhd->nhgd", share, x).reshape(n, 32, 128)  # noqa: E731
    return mix(v.double()), mix(v.double().abs()), score.logsumexp(-1).reshape(n, 32) / math.log(2)


class Server:
    def __init__(self, seed):
        self.g = torch.Generator(device=DEV).manual_seed(seed)
        zeros = lambda *s: torch.zeros(s, dtype=torch.bfloat16, device=DEV)  # noqa: E731
        self.k, self.v = zeros(CAP + 1, 8, 128), zeros(CAP + 1, 8, 128)
        self.bk, self.bv = [zeros(BANK_SLOTS, 8, 128) for _ in range(BANKS)], [zeros(BANK_SLOTS, 8, 128) for _ in range(BANKS)]
        self.table = table(128)
        self.qw, self.kw = (1 + 0.2 * self.normal(128) for _ in range(2))
        self.status = torch.zeros(1, dtype=torch.int32, device=DEV)
        self.free = (torch.randperm(CAP, generator=self.g, device=DEV) + 1).tolist()

    def normal(self, *shape):
        return torch.empty(shape, dtype=torch.bfloat16, device=DEV).normal_(generator=self.g)

    def forward(self, positions):
        """New tokens of a layer: slots taken, q / k rotated, k / v stored.  Returns (rotated q, slots)."""
        n = len(positions)
        slots = torch.tensor([self.free.pop() for _ in range(n)], device=DEV)
        pos = torch.tensor(positions, device=DEV)
        qkv = self.normal(n, 6144)
        q, k, v = qkv[:, :4096].view(n, 32, 128), qkv[:, 4096:5120].view(n, 8, 128), qkv[:, 5120:].view(n, 8, 128)
        q0, k0 = q.clone(), k.clone()
        ops.rope_set_kv_buffer(self.k, self.v, slots, pos, self.table, q, k, v, q, self.status, q_norm_weight=self.qw,
                               k_norm_weight=self.kw)
        rope_close(q, rotate64(q0, self.qw, self.table, pos, False, 1e-6), "q")
        rope_close(self.k[slots], rotate64(k0, self.kw, self.table, pos, False, 1e-6), "k")
        assert torch.equal(self.v[slots], v)
        return q, slots.int()

    def rows(self, pages):
        pages, k, v = pages.long(), [], []
        for p in pages.tolist():
            far = p - CAP - 1
            k.append(self.k[p] if far < 0 else self.bk[far % BANKS][far // BANKS])
            v.append(self.v[p] if far < 0 else self.bv[far % BANKS][far // BANKS])
        return torch.stack(k), torch.stack(v)

    def move(self, pages, ids):
        """Local rows to supplier banks; returns the new page ids."""
        local = torch.tensor([self.k.data_ptr(), self.v.data_ptr()], dtype=torch.int64, device=DEV)
        remote = torch.tensor([t.data_ptr() for pair in zip(self.bk, self.bv) for t in pair], dtype=torch.int64, device=DEV)
        ops.migrate_copy(local, remote, 2, BANKS, pages.long(), ids.long(), False, CAP + 1, BANK_SLOTS, self.status)
        return ids.int() + CAP + 1

    def peers(self):
        return [t for pair in zip(self.bk, self.bv) for t in pair]


def check(out, lse, q, k, v, residual):
    ref, size, ref_lse = attend64(q, k, v)
    L = k.shape[0]
    S = max(1.0, float(torch.einsum("nhgd,lhd->nhgl", q.double().abs().view(-1, 8, 4, 128), k.double().abs()).max())
            * SCALE / math.log(2))
    tol = 2.0 ** -15 * S + (2.0 ** -16 if residual else 2.0 ** -8) + L / 16 * 2.0 ** -23  # as in test_shared_prefix_gpu
    off = (out.double() - ref).abs()
    assert bool((off <= 2.0 ** -8 * ref.abs() + tol * size).all()), float(off.max())
    off = (lse.double() - ref_lse).abs()
    assert bool((off <= 2.0 ** -15 * S + 2.0 ** -23 * ref_lse.abs()).all()), float(off.max())


def test_decode_loop_over_two_groups():
    s = Server(1)
    sizes, prompt = [5, 37], [1300, 200]
    prefix = []
    for n in prompt:
        prefix.append(s.forward(range(n))[1])
    own = [torch.empty(0, dtype=torch.int32, device=DEV) for _ in range(sum(sizes))]
    group = [0] * sizes[0] + [1] * sizes[1]
    w = SharedPrefixDecodeWrapper(torch.empty(32 << 20, dtype=torch.uint8, device=DEV))
    gi, pi = [0, 5, 42], [0, 1300, 1500]
    for step in range(4):
        if step == 2:  # the oldest positions of the long prefix move to the suppliers
            ids = torch.randperm(BANKS * BANK_SLOTS, generator=s.g, device=DEV)[:500]
            prefix[0] = torch.cat([s.move(prefix[0][:500], ids), prefix[0][500:]])
        q, slots = s.forward([prompt[group[b]] + step for b in range(42)])
        own = [torch.cat([o, slots[b:b + 1]]) for b, o in enumerate(own)]
        ii = torch.tensor([0] + [o.numel() for o in own]).cumsum(0).int()
        w.plan(gi, pi, torch.cat(prefix), ii, torch.cat(own), 32, 8, 128, 1)
        out, lse = w.run_return_lse(q, (s.k, s.v), *s.peers(), torch.cat(prefix), torch.cat(own), CAP, SCALE)
        assert w.status() == 0 and int(s.status.item()) == 0
        for g in range(2):
            pk, pv = s.rows(prefix[g])
            for b in range(gi[g], gi[g + 1], 3):
                ok, ov = s.rows(own[b])
                check(out[b:b + 1], lse[b:b + 1], q[b:b + 1], torch.cat([pk, ok]), torch.cat([pv, ov]),
                      prompt[g] < 1024)


def test_history_and_chunk_of_an_append_joined():
    """A chunk of 70 new tokens behind 900 stored ones: the history without a mask, the chunk causal, joined."""
    s = Server(2)
    _, history = s.forward(range(900))
    q, chunk = s.forward(range(900, 970))
    ws = torch.empty(1 << 20, dtype=torch.uint8, device=DEV)
    parts = []
    for pages, causal in ((history, False), (chunk, True)):
        w = BatchPrefillWithPagedKVCacheWrapper(ws)
        w.plan([0, 70], [0, pages.numel()], pages, None, 32, 8, 128, 1, causal=causal)
        parts.append(w.run_return_lse(q, (s.k, s.v)))
        assert w.status() == 0
    out, lse = torch.empty_like(q.contiguous()), torch.empty((70, 32), device=DEV)
    ops.merge_attention_states([p[0] for p in parts], [p[1] for p in parts], out, lse)
    k, v = s.rows(torch.cat([history, chunk]))
    seen = torch.arange(970, device=DEV)[None, :] <= 900 + torch.arange(70, device=DEV)[:, None]
    ref, size, ref_lse = attend64(q, k, v, seen)
    # two partial outputs rounded to bf16, and the joined one: 2^-8 each, relative to sum share |v| at most
    off = (out.double() - ref).abs()
    assert bool((off <= 2.0 ** -8 * ref.abs() + (2.0 ** -8 + 2.0 ** -10) * size).all()), float(off.max())
    torch.testing.assert_close(lse.double(), ref_lse, atol=2e-3, rtol=0)


def test_a_whole_step_captured_and_replayed():
    """Rotation, store, shared-prefix decode and a join with a state from elsewhere in one CUDA graph; the buffers
    get other contents between replays."""
    s = Server(3)
    _, prefix = s.forward(range(700))
    B = 20
    own = torch.tensor([s.free.pop() for _ in range(2 * B)], dtype=torch.int32, device=DEV)
    s.k[own.long()], s.v[own.long()] = s.normal(2 * B, 8, 128), s.normal(2 * B, 8, 128)
    qkv, pos = s.normal(B, 6144), torch.full((B,), 701, dtype=torch.int64, device=DEV)
    q, k, v = (qkv[:, a:b].view(B, -1, 128) for a, b in ((0, 4096), (4096, 5120), (5120, 6144)))
    rotated, out, lse = torch.empty((B, 32, 128), dtype=torch.bfloat16, device=DEV), s.normal(B, 32, 128), torch.empty((B, 32), device=DEV)
    far, far_lse, joined = s.normal(B, 32, 128), torch.zeros((B, 32), device=DEV), s.normal(B, 32, 128)
    buf = lambda n: torch.zeros(n, dtype=torch.int32, device=DEV)  # noqa: E731
    w = SharedPrefixDecodeWrapper(torch.empty(32 << 20, dtype=torch.uint8, device=DEV), use_cuda_graph=True,
                                  paged_kv_indptr_buffer=buf(B + 1), paged_kv_indices_buffer=buf(4 * B),
                                  prefix_indices_buffer=buf(1000), plan_buffer=buf(1 << 13))
    w.plan([0, B], [0, 700], prefix, 2 * torch.arange(B + 1), own, 32, 8, 128, 1)
    newest = own.view(B, 2)[:, 1].long()

    def step():
        ops.rope_set_kv_buffer(s.k, s.v, newest, pos, s.table, q, k, v, rotated, s.status)
        w.run(rotated, (s.k, s.v), out=out, lse=lse, return_lse=True)
        ops.merge_attention_states([out, far], [lse, far_lse], joined)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for replay in range(3):
        qkv.normal_(generator=s.g)
        pos.fill_(702 + replay)
        far_lse.normal_(10, 2, generator=s.g)
        graph.replay()
        assert w.status() == 0 and int(s.status.item()) == 0
        pk, pv = s.rows(prefix)
        for b in range(0, B, 4):
            ok, ov = s.rows(own[2 * b:2 * b + 2])
            check(out[b:b + 1], lse[b:b + 1], rotated[b:b + 1], torch.cat([pk, ok]), torch.cat([pv, ov]), True)
        share = torch.softmax(torch.stack([lse, far_lse]).double() * math.log(2), 0)
        want = share[0, :, :, None] * out.double() + share[1, :, :, None] * far.double()
        size = share[0, :, :, None] * out.double().abs() + share[1, :, :, None] * far.double().abs()
        assert bool(((joined.double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -18 * size).all())
