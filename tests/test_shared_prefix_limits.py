"""ops.shared_prefix_limits: the workspace and plan words that serve every plan of a batch (no GPU)."""
import ctypes as C
import random

import pytest
import torch

from dual_b200 import SharedPrefixDecodeWrapper, _lib, ops

OWN = [-1, 0, 1, 16, 100, 500, 1091, 3000, 5120, 20000, 77000, 300000, 10 ** 6, 10 ** 8]


def indptr(lengths):
    return torch.tensor([0] + list(lengths)).cumsum(0).tolist()


def check(sizes, prefixes, ctas):
    most, words = ops.shared_prefix_limits(sum(sizes), len(sizes), ctas)
    need = [ops.shared_prefix_plan(indptr(sizes), indptr(prefixes), ctas, own) for own in OWN]
    assert max(p.numel() for p in need) <= words
    sizes_of = [ops.shared_prefix_workspace_size(p) for p in need]
    assert max(sizes_of) <= most
    return sizes_of, most


@pytest.mark.parametrize("sizes,prefixes", [
    ([256], [4096]), ([256], [16384]), ([23, 94, 84], [18625, 13607, 1650]), ([64], [32768]), ([3], [517]),
    ([1] * 200, [700] * 200), ([4] * 64, [300] * 64), ([65, 0, 129, 1], [5000, 10, 0, 40000]), ([7], [0]), ([0], [50])])
@pytest.mark.parametrize("ctas", [1, 2, 37, 148, 300])
def test_limits_cover_every_number_of_own_entries(sizes, prefixes, ctas):
    check(sizes, prefixes, ctas)


@pytest.mark.parametrize("seed", range(25))
def test_limits_cover_drawn_groups(seed):
    rng = random.Random(seed)
    groups = rng.choice([1, 2, 3, 9, 40])
    sizes = [rng.choice([0, 1, 2, 5, 31, 32, 33, 63, 64, 65, 100, 200]) for _ in range(groups)]
    check(sizes, [rng.choice([0, 1, 100, 128, 1000, 5000, 40000]) for _ in sizes], rng.choice([1, 3, 20, 148]))


def test_the_need_moves_with_the_own_entries_and_the_limit_does_not():
    """Why a workspace is sized by the limits: a plan made without the own entries can need less than the next step's."""
    needs, most = check([256], [4096], 148)
    assert max(needs) > needs[0]
    assert most <= 1.3 * max(needs)  # and it is no waste


def test_a_wrapper_of_the_limits_plans_every_step():
    sizes, prefixes = [23, 94, 84], [18625, 13607, 1650]
    most, words = ops.shared_prefix_limits(201, 3, 148)
    n, entries = sum(prefixes), 30000
    buf = lambda k: torch.zeros(k, dtype=torch.int32)  # noqa: E731
    wrapper = SharedPrefixDecodeWrapper(torch.zeros(most, dtype=torch.uint8), num_ctas=148, use_cuda_graph=True,
                                        paged_kv_indptr_buffer=buf(202), paged_kv_indices_buffer=buf(entries),
                                        prefix_indices_buffer=buf(n), plan_buffer=buf(words))
    for own in (0, 1091, 201 * 20, entries):
        lengths = [own // 201 + (i < own % 201) for i in range(201)]
        try:
            wrapper.plan(indptr(sizes), indptr(prefixes), buf(n), torch.tensor(indptr(lengths)), buf(own), 32, 8, 128, 1)
        except ValueError as e:  # the lists are in place; without a GPU the status word is not cleared
            assert str(e).startswith("expected a CUDA tensor")


def test_limits_grow_with_the_batch_and_its_groups():
    last = (0, 0)
    for batch, groups in [(0, 0), (1, 1), (3, 1), (3, 2), (64, 2), (65, 2), (65, 65), (300, 65), (300, 300)]:
        now = ops.shared_prefix_limits(batch, groups, 148)
        assert now[0] >= last[0] and now[1] >= last[1]
        last = now
    assert ops.shared_prefix_limits(5, 9, 148) == ops.shared_prefix_limits(5, 5, 148)  # five groups hold a request


def test_limits_refusals():
    for args in [(-1, 1, 8), (1, -1, 8), (1, 1, -1), (1, 1, 1 << 16)]:
        with pytest.raises(_lib.DualError, match="limits"):
            ops.shared_prefix_limits(*args)
    lib, words = _lib.load(), C.c_int64(0)
    assert lib.dual_shared_prefix_limits(1, 1, 8, None, C.byref(words)) == 1
