"""Outputs and states of a merge that lie in one buffer: side by side they are taken, overlapping they are refused
(no GPU: what is taken is refused for its device only)."""
import pytest
import torch

from dual_b200 import ops

BF, FP = torch.bfloat16, torch.float32
T = 5


def merge(states, out):
    ops.merge_attention_states(states, [torch.zeros((T, 32)) for _ in states], out)


def halves(dtype=BF):
    wide = torch.zeros((T, 32, 256), dtype=dtype)
    return wide[..., :128], wide[..., 128:]


def by_head(n, dtype=BF):
    return torch.zeros((T, 32, n, 128), dtype=dtype).unbind(2)


def heads_first():
    return torch.zeros((32, T, 2, 128), dtype=BF).permute(2, 1, 0, 3).unbind(0)


def shifted(by):
    """A state and an output of the same strides whose rows are `by` values apart."""
    flat = torch.zeros(T * 32 * 256 + 1024, dtype=BF)
    view = lambda at: flat[at:].as_strided((T, 32, 128), (32 * 256, 256, 1), flat[at:].storage_offset())  # noqa: E731
    return view(512), view(512 + by)


@pytest.mark.parametrize("states,out", [
    ((lambda h: ([h[0]], h[1]))(halves())),
    ((lambda h: ([h[1]], h[0]))(halves(FP))),
    ((lambda h: ([h[0], h[2]], h[1]))(by_head(3))),
    ((lambda h: ([h[0], h[1]], h[0]))(by_head(2, FP))),
    ((lambda h: ([h[0]], h[1]))(heads_first())),
    ((lambda h: ([h[0]], h[1]))(shifted(128))),
    ((lambda h: ([h[0]], h[1]))(shifted(-128))),
    ((lambda h: ([h[0]], h[1]))(shifted(128 + 256))),
])
def test_side_by_side(states, out):
    with pytest.raises(ValueError, match="CUDA tensor"):
        merge(list(states), out)


@pytest.mark.parametrize("by", [8, 64, 120, 136, 248, 256, -8, -120, -136, -256, 512])
def test_rows_that_overlap(by):
    state, out = shifted(by)
    with pytest.raises(ValueError, match="one of the states"):
        merge([state], out)


def test_other_strides_in_one_buffer():
    flat = torch.zeros(T * 32 * 256, dtype=BF)
    wide, narrow = flat.view(T, 32, 256)[..., 128:], flat[:T * 4096].view(T, 32, 128)
    with pytest.raises(ValueError, match="one of the states"):
        merge([wide], narrow)
    odd = torch.zeros(20000, dtype=BF)  # token strides that are no multiple of the head stride
    a, b = (odd[at:].as_strided((2, 32, 128), (32 * 256 + 128, 256, 1), at) for at in (0, 128))
    with pytest.raises(ValueError, match="one of the states"):
        ops.merge_attention_states([a], [torch.zeros((2, 32))], b)
