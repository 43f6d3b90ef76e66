"""The KV writer with the position rotation on the way, against the rotation written in 64 bits.

Tolerance, element by element: a bf16 rounding is off by at most 2^-8 of the value.  In front of it
stand fp32 operations on terms a c and b s: two products and a sum (2^-24 each), and with the norm a
sum of 128 squares (at most 128 roundings, halved by the root), an inverse root and the weights --
together less than 2^-17 of |a c| + |b s|.  v rows are copied bit by bit.
"""
import pytest
import torch

from dual_b200 import ops

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
MAX_POS = 5000


def table(rotary, device=DEV):
    freq = 1e4 ** (-torch.arange(0, rotary, 2, dtype=torch.float64, device=device) / rotary)
    angle = torch.arange(MAX_POS, dtype=torch.float64, device=device)[:, None] * freq
    return torch.cat([angle.cos(), angle.sin()], 1).float().contiguous()


def rotate64(x, weight, cs, positions, interleaved, eps):
    """(R_p(norm(x)), |a c| + |b s|) in 64 bits."""
    x = x.double()
    if weight is not None:
        x = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * weight.double()
    rotary = cs.shape[1]
    t = cs.double()[positions.long()][:, None, :]
    c, s = t[..., :rotary // 2], t[..., rotary // 2:]
    out, size = x.clone(), x.abs()
    first = slice(0, rotary, 2) if interleaved else slice(0, rotary // 2)
    second = slice(1, rotary, 2) if interleaved else slice(rotary // 2, rotary)
    a, b = x[..., first], x[..., second]
    out[..., first], out[..., second] = a * c - b * s, b * c + a * s
    size[..., first], size[..., second] = (a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs()
    return out, size


def close(got, want, what):
    ref, size = want
    off = (got.double() - ref).abs()
    assert bool((off <= 2.0 ** -8 * ref.abs() + 2.0 ** -17 * size).all()), (what, float(off.max()))


def inputs(n, rotary, norm, index, seed, capacity=None, scale=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    capacity = capacity or n + 50
    mk = lambda *s: torch.empty(s, dtype=torch.bfloat16, device=DEV).normal_(0, scale, generator=g)  # noqa: E731
    qkv = mk(n, 6144)
    return dict(k_local=mk(capacity + 1, 8, 128), v_local=mk(capacity + 1, 8, 128),
                locations=(torch.randperm(capacity, generator=g, device=DEV)[:n] + 1).to(index),
                positions=torch.randint(0, MAX_POS, (n,), generator=g, device=DEV).to(index), cos_sin=table(rotary),
                q=qkv[:, :4096].view(n, 32, 128), k=qkv[:, 4096:5120].view(n, 8, 128),
                v=qkv[:, 5120:].view(n, 8, 128), q_out=torch.empty((n, 32, 128), dtype=torch.bfloat16, device=DEV),
                status=torch.zeros(1, dtype=torch.int32, device=DEV),
                q_norm_weight=1 + 0.3 * mk(128) if norm else None, k_norm_weight=1 + 0.3 * mk(128) if norm else None)


def check(a, before, interleaved, eps, keep=None):
    """Every row of the pools and of q_out, given the state before; `keep`: tokens that are stored."""
    n = a["q"].shape[0]
    keep = torch.ones(n, dtype=torch.bool, device=DEV) if keep is None else keep
    where = a["locations"].long()[keep]
    pos = a["positions"].long().clamp(0, MAX_POS - 1)
    close(a["k_local"][where], [t[keep] for t in rotate64(before["k"], a["k_norm_weight"], a["cos_sin"], pos,
                                                          interleaved, eps)], "k")
    assert torch.equal(a["v_local"][where].view(torch.int16), before["v"][keep].view(torch.int16))
    rest = torch.ones(a["k_local"].shape[0], dtype=torch.bool, device=DEV)
    rest[where] = False
    for name in ("k_local", "v_local"):
        assert torch.equal(a[name][rest].view(torch.int16), before[name][rest].view(torch.int16)), name
    return rotate64(before["q"], a["q_norm_weight"], a["cos_sin"], pos, interleaved, eps)


def snapshot(a):
    return {k: a[k].clone() for k in ("k_local", "v_local", "q", "k", "v", "q_out")}


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("n,rotary,index", [(1, 128, torch.int64), (2, 16, torch.int32), (7, 48, torch.int64),
                                            (64, 128, torch.int32), (333, 96, torch.int64), (2500, 64, torch.int32)])
def test_rotation_and_store_match_64_bits(n, rotary, index, norm, interleaved):
    a = inputs(n, rotary, norm, index, seed=n + rotary)
    before = snapshot(a)
    ops.rope_set_kv_buffer(**a, interleaved=interleaved, norm_eps=1e-5)
    assert int(a["status"].item()) == 0
    close(a["q_out"], check(a, before, interleaved, 1e-5), "q")


def test_first_and_last_positions_and_only_one_norm():
    a = inputs(4, 128, True, torch.int64, seed=5)
    a["positions"] = torch.tensor([0, MAX_POS - 1, 1, MAX_POS - 1], device=DEV)
    a["q_norm_weight"] = None
    before = snapshot(a)
    ops.rope_set_kv_buffer(**a)
    close(a["q_out"], check(a, before, False, 1e-6), "q")
    assert torch.equal(a["q_out"][0], before["q"][0])  # position 0: the angle is 0


def test_in_place_q_strided_pools_and_slot_zero():
    """q rotated in place inside the fused buffer (k and v next to it stay), pools with a slot stride of
    their own, and the dummy slot as a target."""
    a = inputs(130, 128, False, torch.int64, seed=9, capacity=200)
    wide = torch.empty((201, 2, 8, 128), dtype=torch.bfloat16, device=DEV).normal_()
    a["k_local"], a["v_local"] = wide[:, 0], wide[:, 1]
    a["locations"][17] = 0
    a["q_out"] = a["q"]
    before = snapshot(a)
    ops.rope_set_kv_buffer(**a)
    close(a["q"], check(a, before, False, 1e-6), "q")
    for name in ("k", "v"):
        assert torch.equal(a[name], before[name])


@pytest.mark.parametrize("index", [torch.int64, torch.int32])
def test_bad_positions_and_slots_are_skipped_and_recorded(index):
    a = inputs(9, 64, False, index, seed=3, capacity=40)
    a["positions"][2], a["positions"][5] = -1, MAX_POS
    a["locations"][4], a["locations"][7] = 41, -3
    a["q_out"].fill_(7.0)
    before = snapshot(a)
    ops.rope_set_kv_buffer(**a)
    assert int(a["status"].item()) == 0x40 | 0x1
    keep = torch.ones(9, dtype=torch.bool, device=DEV)
    keep[[2, 4, 5, 7]] = False
    ref, size = check(a, before, False, 1e-6, keep)
    turned = torch.ones(9, dtype=torch.bool, device=DEV)
    turned[[2, 5]] = False
    close(a["q_out"][turned], (ref[turned], size[turned]), "q")
    assert bool((a["q_out"][~turned] == 7.0).all())


def test_not_a_number_stays_in_its_head_row():
    """A NaN spoils its pair (with the norm: its head row), nothing else."""
    a = inputs(3, 128, False, torch.int64, seed=4)
    a["q"][1, 5, 3] = float("nan")
    before = snapshot(a)
    before["q"] = before["q"].nan_to_num(0.0)
    ops.rope_set_kv_buffer(**a)
    bad = torch.zeros((3, 32, 128), dtype=torch.bool, device=DEV)
    bad[1, 5, 3] = bad[1, 5, 67] = True
    assert torch.equal(a["q_out"].isnan(), bad)
    ref, size = check(a, before, False, 1e-6)
    close(torch.where(bad, 0, a["q_out"]), (ref.masked_fill(bad, 0), size), "q")


def test_padded_entries_may_share_the_dummy_slot():
    a = inputs(40, 128, False, torch.int64, seed=6)
    a["locations"][20:] = 0
    before = snapshot(a)
    ops.rope_set_kv_buffer(**a)
    assert int(a["status"].item()) == 0
    where = a["locations"][:20]
    ref = rotate64(before["k"][:20], None, a["cos_sin"], a["positions"][:20], False, 0)
    close(a["k_local"][where], ref, "k")
    assert torch.equal(a["v_local"][where], before["v"][:20])
    rest = torch.ones(a["k_local"].shape[0], dtype=torch.bool, device=DEV)
    rest[where] = False
    rest[0] = False
    assert torch.equal(a["k_local"][rest], before["k_local"][rest])


def test_captured_and_replayed_on_another_stream():
    a = inputs(5, 128, True, torch.int64, seed=8)
    stream = torch.cuda.Stream(DEV)
    stream.wait_stream(torch.cuda.current_stream(DEV))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        ops.rope_set_kv_buffer(**a)
    for step in range(3):  # new contents of the same buffers
        a["positions"].copy_(torch.randint(0, MAX_POS, (5,), device=DEV))
        a["q"].normal_()
        a["k"].normal_()
        before = snapshot(a)
        graph.replay()
        close(a["q_out"], check(a, before, False, 1e-6), "q")


def test_rows_past_four_gigabytes():
    """Slots whose byte offset needs more than 32 bits."""
    slots = (1 << 32) // 2048 + 300
    k_local = torch.zeros((slots, 8, 128), dtype=torch.bfloat16, device=DEV)
    v_local = torch.zeros_like(k_local)
    a = inputs(6, 128, False, torch.int64, seed=11)
    a["k_local"], a["v_local"] = k_local, v_local
    a["locations"] = torch.arange(slots - 6, slots, device=DEV)
    ops.rope_set_kv_buffer(**a)
    close(k_local[-6:], rotate64(a["k"], None, a["cos_sin"], a["positions"], False, 0), "k")
    assert torch.equal(v_local[-6:], a["v"])
    assert not bool(k_local[:400].any()) and not bool(v_local[:400].any())


def test_no_tokens():
    a = inputs(4, 128, False, torch.int64, seed=1)
    before = snapshot(a)
    empty = {k: a[k][:0] for k in ("locations", "positions", "q", "k", "v", "q_out")}
    ops.rope_set_kv_buffer(**{**a, **empty})
    assert torch.equal(a["k_local"], before["k_local"]) and torch.equal(a["v_local"], before["v_local"])


def test_pools_with_a_page_axis_and_one_token_of_a_wide_buffer():
    """Pools [slots, 1, 8, 128], and a single token whose tensors have strides of a larger buffer."""
    a = inputs(3, 128, True, torch.int32, seed=12)
    before = snapshot(a)
    paged = {k: a[k].unsqueeze(1) for k in ("k_local", "v_local")}
    one = {k: a[k][1:2] for k in ("locations", "positions", "q", "k", "v", "q_out")}
    ops.rope_set_kv_buffer(**{**a, **paged, **one})
    only = torch.tensor([False, True, False], device=DEV)
    ref, size = check(a, before, False, 1e-6, only)
    close(a["q_out"][1:2], (ref[1:2], size[1:2]), "q")
    assert torch.equal(a["q_out"][0].view(torch.int16), before["q_out"][0].view(torch.int16))
