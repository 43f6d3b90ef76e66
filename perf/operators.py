"""What the serving operators are measured on: rotating and storing new tokens' q/k/v, decoding a batch whose
requests share prefixes, and merging partial attention states.

`listed()` and `draw(rng)` give cases (dicts of plain values), `prepare(case, seed)` the inputs on the GPU,
`run(state)` one pass -- in elementary torch operations in 32 bits, or with `own` set through the framework --
`work(case)` the bytes and operations a pass cannot do without, and `exact(case, seed)` the outputs from the
definition in 64 bits.
"""
import math
import random

import torch

own = False

HQ, HKV, D = 32, 8, 128  # the framework's head layout: 32 query heads, 8 kv heads, 128 dims
SCALE = 1.0 / math.sqrt(D)
LOG2E = 1.0 / math.log(2.0)
EPS = 1e-6
DEV = "cuda"


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one request's next token in one layer: the whole cost is latency
        dict(name="rope_one", op="rope", n=1, rotary=128, interleaved=False, norm=True, index64=True),
        # a decode step of a batch of 64
        dict(name="rope_step64", op="rope", n=64, rotary=128, interleaved=False, norm=True, index64=True),
        # a ragged prompt chunk, half of the dims rotated in adjacent pairs, 32-bit indices
        dict(name="rope_chunk", op="rope", n=2049, rotary=64, interleaved=True, norm=False, index64=False),
        # the prompts of a large append forward
        dict(name="rope_prompts", op="rope", n=32768, rotary=128, interleaved=False, norm=True, index64=True),
        # a few requests behind a short common instruction
        dict(name="shared_few", op="shared", batch=3, groups=1, prefix=517, suffix=40, banks=0, remote=0, lens=1),
        # samples of one prompt: the batch is small against the prefix, bytes decide
        dict(name="shared_16", op="shared", batch=16, groups=1, prefix=32768, suffix=256, banks=0, remote=0, lens=2),
        # a batch of 64 over one long document
        dict(name="shared_64", op="shared", batch=64, groups=1, prefix=32768, suffix=512, banks=0, remote=0, lens=3),
        # several system prompts of different lengths, part of the rows on three supplier banks
        dict(name="shared_groups", op="shared", batch=77, groups=5, prefix=9001, suffix=300, banks=3, remote=12, lens=4),
        # a full serving batch behind one system prompt with tools: operations decide
        dict(name="shared_256", op="shared", batch=256, groups=1, prefix=16384, suffix=600, banks=0, remote=0, lens=5),
        # the states of a decode step
        dict(name="merge_step", op="merge", tokens=5, states=2, wide=False),
        # history and chunk of an append forward, joined
        dict(name="merge_append", op="merge", tokens=8192, states=2, wide=False),
        # states of one sequence held in eight places, in 32 bits
        dict(name="merge_eight", op="merge", tokens=1001, states=8, wide=True),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rope", "shared", "shared", "merge"])
    if op == "rope":
        return dict(op=op, n=_log_uniform(rng, 1, 32768), rotary=rng.choice([32, 64, 96, 128, 128]),
                    interleaved=rng.random() < 0.4, norm=rng.random() < 0.6, index64=rng.random() < 0.6)
    if op == "merge":
        states = rng.randint(2, 8)
        wide = rng.random() < 0.4
        return dict(op=op, tokens=_log_uniform(rng, 1, 16384 // (states * (2 if wide else 1))), states=states, wide=wide)
    batch = _log_uniform(rng, 1, 256)
    groups = min(batch, rng.choice([1, 1, 1, 2, 3, 6]))
    prefix = _log_uniform(rng, 48, min(32768, 256 * 16384 // batch))
    banks = rng.choice([0, 0, 1, 3])
    return dict(op=op, batch=batch, groups=groups, prefix=prefix, suffix=_log_uniform(rng, 1, 600), banks=banks,
                remote=rng.randint(3, 18) if banks else 0, lens=rng.randint(0, 1 << 20))


def _lengths(case):
    """Requests per group, prefix length per group, own length per request (some are 0)."""
    rng = random.Random(case["lens"])
    g, b = case["groups"], case["batch"]
    sizes = [b // g + (i < b % g) for i in range(g)]
    for i in range(g - 1):  # uneven groups of the same total
        move = rng.randint(0, sizes[i] // 2)
        sizes[i] -= move
        sizes[i + 1] += move
    prefixes = [case["prefix"]] if g == 1 else [rng.randint(max(1, case["prefix"] // 4), case["prefix"]) for _ in range(g)]
    suffixes = [rng.randint(0, case["suffix"]) for _ in range(b)]
    return sizes, prefixes, suffixes


def work(case):
    if case["op"] == "rope":
        n = case["n"]
        rows = n * (HQ + 2 * HKV) * D * 2
        index = n * (16 if case["index64"] else 8)
        flops = n * (HQ + HKV) * (3 * case["rotary"] + (4 * D if case["norm"] else 0))
        return {"bytes": 2 * rows + n * case["rotary"] * 4 + index, "flops": flops}
    if case["op"] == "merge":
        rows = case["tokens"] * HQ
        e = 4 if case["wide"] else 2
        return {"bytes": case["states"] * rows * (D * e + 4) + rows * (D * 2 + 4), "flops": case["states"] * rows * 2 * D}
    sizes, prefixes, suffixes = _lengths(case)
    entries = sum(prefixes) + sum(suffixes)
    seen = sum(s * p for s, p in zip(sizes, prefixes)) + sum(suffixes)
    return {"bytes": entries * (2 * HKV * D * 2 + 4) + case["batch"] * HQ * (2 * D * 2 + 4), "flops": seen * HQ * D * 4}


# ----------------------------------------------------------------------------------------------- inputs
def _normal(g, *shape, std=1.0, dtype=torch.bfloat16):
    return torch.empty(shape, dtype=torch.float32, device=DEV).normal_(0.0, std, generator=g).to(dtype)


def _indptr(lengths, dtype=torch.int32):
    return torch.tensor([0] + lengths, device=DEV).cumsum(0).to(dtype)


def _prepare_rope(case, g):
    n, rotary = case["n"], case["rotary"]
    capacity, max_pos = n + n // 4 + 64, 40960
    index = torch.int64 if case["index64"] else torch.int32
    freq = 1e6 ** (-torch.arange(0, rotary, 2, dtype=torch.float64, device=DEV) / rotary)
    angle = torch.arange(max_pos, dtype=torch.float64, device=DEV)[:, None] * freq[None, :]
    qkv = _normal(g, n, (HQ + 2 * HKV) * D)  # the fused projection's output: q | k | v of each token
    s = dict(q=qkv[:, :HQ * D].view(n, HQ, D), k=qkv[:, HQ * D:(HQ + HKV) * D].view(n, HKV, D),
             v=qkv[:, (HQ + HKV) * D:].view(n, HKV, D),
             table=torch.cat([angle.cos(), angle.sin()], 1).float(),
             positions=torch.randint(0, max_pos, (n,), generator=g, device=DEV).to(index),
             locations=(torch.randperm(capacity, generator=g, device=DEV)[:n] + 1).to(index),
             k_pool=_normal(g, capacity + 1, HKV, D), v_pool=_normal(g, capacity + 1, HKV, D),
             q_norm=None, k_norm=None, out=torch.empty((n, HQ, D), dtype=torch.bfloat16, device=DEV),
             status=torch.zeros(1, dtype=torch.int32, device=DEV), interleaved=case["interleaved"])
    if case["norm"]:
        s["q_norm"] = (1.0 + 0.2 * _normal(g, D, dtype=torch.float32)).bfloat16()
        s["k_norm"] = (1.0 + 0.2 * _normal(g, D, dtype=torch.float32)).bfloat16()
    return s


def _prepare_shared(case, g):
    sizes, prefixes, suffixes = _lengths(case)
    batch, banks = case["batch"], case["banks"]
    total = sum(prefixes) + sum(suffixes)
    far = torch.rand(total, generator=g, device=DEV) * 100 < case["remote"]  # every entry local without banks
    n_far = int(far.sum())
    n_near = total - n_far
    capacity = n_near + n_near // 8 + 64
    slots = n_far // max(banks, 1) + 1
    pages = torch.empty(total, dtype=torch.int32, device=DEV)
    pages[~far] = (torch.randperm(capacity, generator=g, device=DEV)[:n_near] + 1).int()
    pages[far] = (torch.randperm(max(banks, 1) * slots, generator=g, device=DEV)[:n_far] + capacity + 1).int()
    s = dict(q=_normal(g, batch, HQ, D, std=1.5), k_pool=_normal(g, capacity + 1, HKV, D),
             v_pool=_normal(g, capacity + 1, HKV, D), capacity=capacity,
             k_bank=_normal(g, banks, slots, HKV, D), v_bank=_normal(g, banks, slots, HKV, D),
             prefix_pages=pages[:sum(prefixes)].clone(), pages=pages[sum(prefixes):].clone(),
             group_indptr=_indptr(sizes), prefix_indptr=_indptr(prefixes), indptr=_indptr(suffixes),
             most=(max(sizes), max(prefixes), max(1, max(suffixes))), handle=None)
    if own:  # the plan a serving loop makes once for a step and uses in every layer
        from dual_b200 import SharedPrefixDecodeWrapper
        s["handle"] = SharedPrefixDecodeWrapper(torch.empty(128 << 20, dtype=torch.uint8, device=DEV))
        s["handle"].plan(s["group_indptr"], s["prefix_indptr"], s["prefix_pages"], s["indptr"], s["pages"],
                         HQ, HKV, D, 1)
        s["peers"] = [t for pair in zip(s["k_bank"].unbind(0), s["v_bank"].unbind(0)) for t in pair]
    return s


def _prepare_merge(case, g):
    tokens, n = case["tokens"], case["states"]
    dtype = torch.float32 if case["wide"] else torch.bfloat16
    outs = [_normal(g, tokens, HQ, D, std=0.3, dtype=dtype) for _ in range(n)]
    lses = [_normal(g, tokens, HQ, std=2.0, dtype=torch.float32) + 12.0 for _ in range(n)]
    for o, l in zip(outs, lses):  # a request that a state has no entry of: output 0, LSE -inf
        empty = torch.rand(tokens, generator=g, device=DEV) < 0.06
        o[empty] = 0
        l[empty] = -math.inf
    return dict(outs=outs, lses=lses, out=torch.empty((tokens, HQ, D), dtype=torch.bfloat16, device=DEV),
                lse=torch.empty((tokens, HQ), dtype=torch.float32, device=DEV))


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed) * 7919 + 17)
    state = {"rope": _prepare_rope, "shared": _prepare_shared, "merge": _prepare_merge}[case["op"]](case, g)
    state["op"] = case["op"]
    return state


# ----------------------------------------------------------------------------------------- one pass
def _rotated(x, weight, table, positions, interleaved):
    """RMS norm over the head's dims (where a weight is given) and rotation, in 32 bits; rounded once."""
    x = x.float()
    if weight is not None:
        x = x / (x * x).mean(-1, keepdim=True).add(EPS).sqrt() * weight.float()
    rotary = table.shape[1]
    row = table[positions.long()][:, None, :]
    c, s = row[..., :rotary // 2], row[..., rotary // 2:]
    part, rest = x[..., :rotary], x[..., rotary:]
    if interleaved:
        a, b = part[..., 0::2], part[..., 1::2]
        part = torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2)
    else:
        a, b = part[..., :rotary // 2], part[..., rotary // 2:]
        part = torch.cat([a * c - b * s, b * c + a * s], -1)
    return torch.cat([part, rest], -1).to(torch.bfloat16)


def _run_rope(s):
    if own:
        from dual_b200 import ops
        ops.rope_set_kv_buffer(s["k_pool"], s["v_pool"], s["locations"], s["positions"], s["table"], s["q"], s["k"],
                               s["v"], s["out"], s["status"], interleaved=s["interleaved"],
                               q_norm_weight=s["q_norm"], k_norm_weight=s["k_norm"], norm_eps=EPS)
    else:
        where = s["locations"].long()
        s["out"].copy_(_rotated(s["q"], s["q_norm"], s["table"], s["positions"], s["interleaved"]))
        s["k_pool"][where] = _rotated(s["k"], s["k_norm"], s["table"], s["positions"], s["interleaved"])
        s["v_pool"][where] = s["v"]
    return {"q": s["out"], "k_pool": s["k_pool"], "v_pool": s["v_pool"]}


def _rows(pages, pool, bank, capacity):
    """Rows that page ids name: local slot p up to the capacity, then banks in turn; in 32 bits."""
    pages = pages.long()
    rows = pool[pages.clamp(max=capacity)]
    if bank.shape[0]:
        far = (pages - capacity - 1).clamp(min=0)
        far_rows = bank[far % bank.shape[0], far // bank.shape[0]]
        rows = torch.where((pages > capacity)[..., None, None], far_rows, rows)
    return rows.float()


def _padded(pages, indptr, most):
    """Lists of page ids as a matrix, and which of its places are entries."""
    first, last = indptr[:-1].long()[:, None], indptr[1:].long()[:, None]
    at = first + torch.arange(most, device=DEV)[None, :]
    valid = at < last
    if pages.numel() == 0:
        return torch.zeros_like(at), valid
    return pages[torch.where(valid, at, 0)], valid


def _run_shared(s):
    if own:
        out, lse = s["handle"].run_return_lse(s["q"], (s["k_pool"], s["v_pool"]), *s["peers"], s["prefix_pages"],
                                              s["pages"], s["capacity"], SCALE)
        return {"out": out, "lse": lse}
    most_b, most_p, most_s = s["most"]
    batch = s["q"].shape[0]
    # a group's prefix, seen by all of its requests: [groups, kv heads, requests x 4, entries]
    first = s["group_indptr"][:-1].long()[:, None]
    member = first + torch.arange(most_b, device=DEV)[None, :]
    inside = member < s["group_indptr"][1:].long()[:, None]
    q = s["q"].float().view(batch, HKV, HQ // HKV, D)
    qg = q[torch.where(inside, member, 0)].permute(0, 2, 1, 3, 4).flatten(2, 3)
    pages, valid = _padded(s["prefix_pages"], s["prefix_indptr"], most_p)
    k = _rows(pages, s["k_pool"], s["k_bank"], s["capacity"]).permute(0, 2, 1, 3)
    v = _rows(pages, s["v_pool"], s["v_bank"], s["capacity"]).permute(0, 2, 1, 3)
    score_p = (qg @ k.transpose(-1, -2) * SCALE).masked_fill(~valid[:, None, None, :], -math.inf)
    # each request's own entries: [requests, kv heads, 4, entries]
    pages, valid = _padded(s["pages"], s["indptr"], most_s)
    ks = _rows(pages, s["k_pool"], s["k_bank"], s["capacity"]).permute(0, 2, 1, 3)
    vs = _rows(pages, s["v_pool"], s["v_bank"], s["capacity"]).permute(0, 2, 1, 3)
    score_s = (q @ ks.transpose(-1, -2) * SCALE).masked_fill(~valid[:, None, None, :], -math.inf)

    def by_request(x):  # [groups, kv heads, requests x 4, ...] -> [requests, kv heads, 4, ...]
        x = x.unflatten(2, (most_b, HQ // HKV)).transpose(1, 2)
        return x[inside]

    top_p = score_p.amax(-1, keepdim=True)
    top_p = torch.where(top_p == -math.inf, 0.0, top_p)
    p = torch.exp(score_p - top_p)
    sum_p, out_p, top_p = by_request(p.sum(-1, keepdim=True)), by_request(p @ v), by_request(top_p)
    top_s = score_s.amax(-1, keepdim=True)
    top_s = torch.where(top_s == -math.inf, 0.0, top_s)
    p = torch.exp(score_s - top_s)
    sum_s, out_s = p.sum(-1, keepdim=True), p @ vs
    top = torch.maximum(torch.where(sum_p > 0, top_p, -math.inf), torch.where(sum_s > 0, top_s, -math.inf))
    top = torch.where(top == -math.inf, 0.0, top)
    a, b = torch.where(sum_p > 0, torch.exp(top_p - top), 0.0), torch.where(sum_s > 0, torch.exp(top_s - top), 0.0)
    total = a * sum_p + b * sum_s
    out = torch.where(total > 0, (a * out_p + b * out_s) / total, 0.0)
    lse = (top + torch.log(total)) * LOG2E
    return {"out": out.reshape(batch, HQ, D).to(torch.bfloat16), "lse": lse.reshape(batch, HQ)}


def _run_merge(s):
    if own:
        from dual_b200 import ops
        ops.merge_attention_states(s["outs"], s["lses"], s["out"], s["lse"])
        return {"out": s["out"], "lse": s["lse"]}
    o, l = torch.stack(s["outs"]).float(), torch.stack(s["lses"])
    top = l.amax(0)
    top = torch.where(top == -math.inf, 0.0, top)
    w = torch.exp2(l - top)
    total = w.sum(0)
    out = torch.where(w[..., None] > 0, w[..., None] * o, 0.0).sum(0) / torch.where(total > 0, total, 1.0)[..., None]
    return {"out": out.to(torch.bfloat16), "lse": top + torch.log2(total)}


def run(state):
    if state["op"] == "rope":
        return _run_rope(state)
    return _run_shared(state) if state["op"] == "shared" else _run_merge(state)


# -------------------------------------------------------------------- the definition in 64 bits
def _exact_rope(s):
    n, rotary = s["q"].shape[0], s["table"].shape[1]
    t = s["table"].double()[s["positions"].long()]
    turn = torch.complex(t[:, :rotary // 2], t[:, rotary // 2:])[:, None, :]  # c + i s of each pair

    def turned(x, weight):
        x = x.double().clone()
        if weight is not None:
            x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * weight.double()
        if s["interleaved"]:
            z = torch.view_as_complex(x[..., :rotary].unflatten(-1, (-1, 2)).contiguous()) * turn
            x[..., :rotary] = torch.view_as_real(z).flatten(-2)
        else:
            z = torch.complex(x[..., :rotary // 2].contiguous(), x[..., rotary // 2:rotary].contiguous()) * turn
            x[..., :rotary // 2], x[..., rotary // 2:rotary] = z.real, z.imag
        return x

    k_pool, v_pool = s["k_pool"].double(), s["v_pool"].double()
    k_pool[s["locations"].long()] = turned(s["k"], s["k_norm"])
    v_pool[s["locations"].long()] = s["v"].double()
    assert n == s["positions"].numel()
    return {"q": turned(s["q"], s["q_norm"]), "k_pool": k_pool, "v_pool": v_pool}


def _exact_shared(s):
    batch = s["q"].shape[0]
    capacity, banks = s["capacity"], s["k_bank"].shape[0]
    out = torch.zeros((batch, HQ, D), dtype=torch.float64, device=DEV)
    lse = torch.full((batch, HQ), -math.inf, dtype=torch.float64, device=DEV)
    ends = [t.tolist() for t in (s["group_indptr"], s["prefix_indptr"], s["indptr"])]

    def rows(pages, pool, bank):
        pages = pages.long()
        got = torch.empty((pages.numel(), HKV, D), dtype=torch.float64, device=DEV)
        near = pages <= capacity
        got[near] = pool[pages[near]].double()
        for i in range(banks):
            here = ~near & ((pages - capacity - 1) % banks == i)
            got[here] = bank[i][(pages[here] - capacity - 1) // banks].double()
        return got

    for g in range(len(ends[0]) - 1):
        shared = s["prefix_pages"][ends[1][g]:ends[1][g + 1]]
        kp, vp = rows(shared, s["k_pool"], s["k_bank"]), rows(shared, s["v_pool"], s["v_bank"])
        for b in range(ends[0][g], ends[0][g + 1]):
            mine = s["pages"][ends[2][b]:ends[2][b + 1]]
            k = torch.cat([kp, rows(mine, s["k_pool"], s["k_bank"])])
            v = torch.cat([vp, rows(mine, s["v_pool"], s["v_bank"])])
            if k.shape[0] == 0:
                continue
            score = torch.einsum("hgd,lhd->hgl", s["q"][b].double().view(HKV, HQ // HKV, D), k) * SCALE
            out[b] = torch.einsum("hgl,lhd->hgd", score.softmax(-1), v).reshape(HQ, D)
            lse[b] = (score.logsumexp(-1) * LOG2E).reshape(HQ)
    return {"out": out, "lse": lse}


def _exact_merge(s):
    o, l = torch.stack(s["outs"]).double(), torch.stack(s["lses"]).double() * math.log(2.0)
    both = l.logsumexp(0)  # -inf where no state saw anything
    share = torch.exp(l - torch.where(both == -math.inf, 0.0, both))
    return {"out": (share[..., None] * o).sum(0), "lse": both * LOG2E}


def exact(case, seed):
    global own
    kept, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = kept
    return {"rope": _exact_rope, "shared": _exact_shared, "merge": _exact_merge}[case["op"]](s)
