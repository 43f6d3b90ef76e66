"""Sizes past what the plan's 32-bit words and the launches hold are refused (no GPU)."""
import ctypes as C

import pytest
import torch

from dual_b200 import SharedPrefixDecodeWrapper, _lib, ops


@pytest.mark.parametrize("gi,pi", [([0, 2], [0, (1 << 32) + 5]), ([0, (1 << 32) + 2], [0, 5]), ([0, 2], [0, 1 << 31]),
                                   ([0, 2, -(1 << 32) + 3], [0, 1, 2])])
def test_indptrs_that_do_not_fit_32_bits(gi, pi):
    """Cut to 32 bits, 2^32 + 5 shared entries would be 5."""
    for make in (list, torch.tensor):
        with pytest.raises(ValueError, match="32 bits"):
            ops.shared_prefix_plan(make(gi), make(pi), 8)


def test_own_entries_out_of_range():
    for own in (1 << 31, 1 << 62):
        with pytest.raises(_lib.DualError, match="own_entries"):
            ops.shared_prefix_plan([0, 2], [0, 5], 8, own)
    ops.shared_prefix_plan([0, 2], [0, 5], 8, (1 << 31) - 1)
    assert torch.equal(ops.shared_prefix_plan([0, 2], [0, 5], 8, -1), ops.shared_prefix_plan([0, 2], [0, 5], 8, -7))


def test_more_requests_than_the_join_has_blocks():
    lib, n = _lib.load(), C.c_int64(0)
    gi, pi = torch.tensor([0, (1 << 28)], dtype=torch.int32), torch.tensor([0, 0], dtype=torch.int32)
    assert lib.dual_shared_prefix_plan(gi.data_ptr(), pi.data_ptr(), 1, 8, -1, None, 0, C.byref(n)) == 1
    assert "requests" in lib.dual_last_error().decode()
    size, words = C.c_size_t(0), C.c_int64(0)
    assert lib.dual_shared_prefix_limits(1 << 28, 1, 8, C.byref(size), C.byref(words)) == 1
    rc = lib.dual_shared_prefix_decode(256, 4096, 128, 256, 256, 2048, 9, None, None, 0, 0, 0, None, 0, 16, None, 0, 1 << 28,
                                       0.1, 256, 1 << 30, 256, 4096, 128, None, 256, 1 << 62, 8, -1, None)
    assert rc == 1 and "batch" in lib.dual_last_error().decode()


def test_states_past_the_plans_offsets():
    """A plan's offsets are 32 bits of 16-byte units: 64 GiB of partial states."""
    with pytest.raises(_lib.DualError, match="states"):
        ops.shared_prefix_plan([0, 4100000], [0, 100], 148)
    plan = ops.shared_prefix_plan([0, 4000000], [0, 100], 148)
    assert ops.shared_prefix_workspace_size(plan) > 130 * 10 ** 9


def test_empty_and_odd_indptrs_of_the_wrapper():
    w = SharedPrefixDecodeWrapper(torch.zeros(1 << 20, dtype=torch.uint8), num_ctas=8)
    none, ends = torch.zeros(0, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    for gi in ([], [[0, 2]], [0.0, 2.0]):
        with pytest.raises(ValueError, match="group_indptr must be a list of integers"):
            w.plan(gi, [0, 0], none, ends, none, 32, 8, 128, 1)


@pytest.mark.parametrize("out", [torch.zeros((1, 32, 128), dtype=torch.bfloat16).expand(3, 32, 128),
                                 torch.zeros((3, 1, 128), dtype=torch.bfloat16).expand(3, 32, 128),
                                 torch.zeros(16384, dtype=torch.bfloat16).as_strided((3, 32, 128), (4096, 64, 1)),
                                 torch.zeros(16384, dtype=torch.bfloat16).as_strided((3, 32, 128), (64, 128, 1))])
def test_output_rows_that_share_memory(out):
    from test_shared_prefix_plan import decode_args
    with pytest.raises(ValueError, match="out must not repeat rows"):
        ops.shared_prefix_decode(**{**decode_args(), "out": out})


def test_one_request_has_no_token_stride():
    from test_shared_prefix_plan import decode_args
    out = torch.zeros((1, 32, 128), dtype=torch.bfloat16).as_strided((1, 32, 128), (0, 128, 1))
    with pytest.raises(ValueError, match="CUDA tensors"):
        ops.shared_prefix_decode(**{**decode_args(B=1), "out": out})
