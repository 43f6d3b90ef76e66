"""What the rotating KV writer and the merge of attention states refuse, on the host and before any launch."""
import ctypes as C

import pytest
import torch

from dual_b200 import _lib, ops

BF = torch.bfloat16


def rope_args(n=3, capacity=10, rotary=64):
    qkv = torch.zeros((n, 6144), dtype=BF)
    return dict(k_local=torch.zeros((capacity + 1, 8, 128), dtype=BF), v_local=torch.zeros((capacity + 1, 8, 128), dtype=BF),
                locations=torch.arange(n), positions=torch.arange(n), cos_sin=torch.zeros((20, rotary)),
                q=qkv[:, :4096].view(n, 32, 128), k=qkv[:, 4096:5120].view(n, 8, 128), v=qkv[:, 5120:].view(n, 8, 128),
                q_out=torch.zeros((n, 32, 128), dtype=BF), status=torch.zeros(1, dtype=torch.int32))


@pytest.mark.parametrize("change,said", [
    (dict(q=torch.zeros((3, 16, 128), dtype=BF)), "q must be"),
    (dict(q=torch.zeros((3, 32, 128))), "q must be"),
    (dict(q_out=torch.zeros((3, 32, 64), dtype=BF)), "q_out must be"),
    (dict(k=torch.zeros((2, 8, 128), dtype=BF)), "k must be"),
    (dict(v=torch.zeros((3, 8, 256), dtype=BF)[:, :, ::2]), "v must be"),
    (dict(locations=torch.arange(3, dtype=torch.int16)), "locations must be"),
    (dict(positions=torch.arange(4)), "positions must be"),
    (dict(positions=torch.arange(6)[::2]), "positions must be"),
    (dict(cos_sin=torch.zeros((20, 64), dtype=BF)), "cos_sin must be"),
    (dict(cos_sin=torch.zeros((20, 128))[:, :64]), "cos_sin must be"),
    (dict(q_norm_weight=torch.zeros(128)), "q_norm_weight must be"),
    (dict(k_norm_weight=torch.zeros(64, dtype=BF)), "k_norm_weight must be"),
    (dict(status=torch.zeros(1, dtype=torch.int64)), "status must be"),
    (dict(v_local=torch.zeros((9, 8, 128), dtype=BF)), "pools must share"),
    (dict(k_local=torch.zeros((11, 4, 128), dtype=BF)), "k_local"),
])
def test_rope_refusals(change, said):
    with pytest.raises(ValueError, match=said):
        ops.rope_set_kv_buffer(**{**rope_args(), **change})


def test_rope_overlaps():
    a = rope_args()
    buf = torch.zeros((4, 32, 128), dtype=BF)
    with pytest.raises(ValueError, match="q itself"):
        ops.rope_set_kv_buffer(**{**a, "q": buf[:3], "q_out": buf[1:]})
    fused = torch.zeros((3, 6144), dtype=BF)
    part = lambda i, j, h: fused[:, i:j].view(3, h, 128)  # noqa: E731
    with pytest.raises(ValueError, match="k or v"):
        ops.rope_set_kv_buffer(**{**a, "k": part(3000, 4024, 8), "q_out": part(0, 4096, 32)})
    # side by side in one fused buffer is no overlap, nor is q in its own place: refused only for the device
    with pytest.raises(ValueError, match="CUDA tensor"):
        ops.rope_set_kv_buffer(**{**a, "q": part(0, 4096, 32), "k": part(4096, 5120, 8), "v": part(5120, 6144, 8),
                                  "q_out": part(0, 4096, 32)})


def merge_args(n=2, T=3, dtype=BF):
    return dict(states=[torch.zeros((T, 32, 128), dtype=dtype) for _ in range(n)],
                lses=[torch.zeros((T, 32)) for _ in range(n)], out=torch.zeros((T, 32, 128), dtype=BF),
                lse=torch.zeros((T, 32)))


def test_merge_refusals():
    for change, said in [
            (dict(states=[], lses=[]), "1 to 8"), (dict(merge_args(9)), "1 to 8"),
            (dict(lses=merge_args()["lses"][:1]), "1 to 8"),
            (dict(states=[torch.zeros((3, 32, 128)), torch.zeros((3, 32, 128), dtype=BF)]), "share a type"),
            (dict(states=[torch.zeros((3, 32, 128), dtype=torch.float16)] * 2), r"states\[0\] must be"),
            (dict(states=[torch.zeros((4, 32, 128), dtype=BF)] * 2), r"states\[0\] must be"),
            (dict(lses=[torch.zeros((3, 32)), torch.zeros((3, 32), dtype=BF)]), r"lses\[1\] must be"),
            (dict(lse=torch.zeros((3, 64))[:, ::2]), "lse must be"),
            (dict(out=torch.zeros((3, 32, 256), dtype=BF)[:, :, ::2]), "out must be")]:
        with pytest.raises(ValueError, match=said):
            ops.merge_attention_states(**{**merge_args(), **change})
    a = merge_args()
    buf = torch.zeros((4, 32, 128), dtype=BF)
    with pytest.raises(ValueError, match="one of the states"):
        ops.merge_attention_states([buf[:3], a["states"][1]], a["lses"], buf[1:], None)
    with pytest.raises(ValueError, match="one of the states"):  # in place needs the same type
        wide = torch.zeros((3, 32, 128))
        ops.merge_attention_states([wide], a["lses"][:1], wide.view(BF)[..., :128], None)
    with pytest.raises(ValueError, match="CUDA tensor"):
        ops.merge_attention_states(**{**a, "out": a["states"][0], "lse": a["lses"][1]})


def test_c_abi_refusals_come_before_any_launch():
    lib = _lib.load()

    def rope(n=2, stride=2048, loc=16, pos=16, cs=16, mp=4, rd=64, q=16, qs=4096, k=16, ks=1024, v=16, vs=1024,
             qo=16, qos=4096, qn=None, eps=1e-6, status=16, capacity=9):
        rc = lib.dual_rope_set_kv_buffer(16, 16, stride, capacity, loc, 1, pos, 1, cs, mp, rd, 0, q, qs, k, ks, v, vs,
                                         qo, qos, qn, None, eps, n, status, -1, None)
        return rc, lib.dual_last_error().decode()

    assert rope(n=0, q=None) == (0, "")
    for change, said in [(dict(n=-1), "n must"), (dict(q=None), "null"), (dict(status=None), "null"),
                         (dict(stride=1024), "slot stride"), (dict(capacity=-1), "local_capacity"),
                         (dict(rd=0), "rotary_dim"), (dict(rd=72), "rotary_dim"), (dict(rd=144), "rotary_dim"),
                         (dict(mp=0), "cos_sin"), (dict(cs=20), "cos_sin"), (dict(q=18), "aligned"),
                         (dict(qs=4000), "token strides"), (dict(ks=1028), "token strides"), (dict(qos=8), "token strides"),
                         (dict(qn=8), "norm weights"), (dict(eps=-1.0), "norm_eps"), (dict(eps=float("nan")), "norm_eps")]:
        rc, msg = rope(**change)
        assert rc == 1 and said in msg, (change, msg)

    def merge(n=2, T=4, states=(16, 16), st=(4096, 4096), sh=(128, 128), lses=(16, 16), wide=0, out=16, ost=4096, osh=128):
        arr = lambda v: (C.c_void_p * 2)(*v)  # noqa: E731
        i64 = lambda v: (C.c_int64 * 2)(*v)  # noqa: E731
        rc = lib.dual_merge_attention_states(arr(states), i64(st), i64(sh), arr(lses), n, wide, T, out, ost, osh, 0,
                                             None, -1, None)
        return rc, lib.dual_last_error().decode()

    assert merge(T=0)[0] == 0
    for change, said in [(dict(T=-1), "tokens"), (dict(n=0), "num_states"), (dict(n=9), "num_states"),
                         (dict(T=1 << 40), "too many"), (dict(out=None), "null"), (dict(states=(16, 0)), "state 1"),
                         (dict(lses=(0, 16)), "state 0"), (dict(states=(24, 16)), "state 0"), (dict(st=(4096, 4100)), "state 1"),
                         (dict(sh=(130, 128)), "state 0"), (dict(out=20), "out must"), (dict(osh=129), "out must")]:
        rc, msg = merge(**change)
        assert rc == 1 and said in msg, (change, msg)
