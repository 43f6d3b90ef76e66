"""A kv_indptr that is no list of prefix sums from 0 on is recorded (every access stays inside the lists whatever it
holds), and padded batches, whose last requests have no entries, are none."""
import pytest
import torch

from dual_b200 import ops
from test_shared_prefix_gpu import Case, DEV, SCALE

pytestmark = pytest.mark.gpu


def status(c, ends, plan=None):
    plan = c.plan() if plan is None else plan
    ws = torch.zeros(ops.shared_prefix_workspace_size(plan), dtype=torch.uint8, device=DEV)
    out, lse = torch.empty_like(c.q), torch.empty((c.q.shape[0], 32), device=DEV)
    ops.shared_prefix_decode(c.q, c.k, c.v, c.C, [], [], c.prefix_pages, torch.tensor(ends, dtype=torch.int32, device=DEV),
                             c.own_pages, SCALE, plan.to(DEV), out, lse, ws)
    return ops.status_read(ws), out, lse


@pytest.mark.parametrize("prefix", [0, 200])
def test_no_prefix_sums(prefix):
    c = Case([4], [prefix], [10, 20, 5, 30], seed=prefix + 1)
    assert status(c, [0, 10, 30, 35, 65])[0] == 0
    for ends in ([3, 10, 30, 35, 65],    # entries in front of the first request's
                 [0, 30, 10, 35, 65],    # a list of negative length
                 [0, 10, 30, 70, 65],
                 [-4, 10, 30, 35, 65],
                 [0, 10, 30, 35, -1],
                 [0, 10, 30, 35, 66]):   # past the end of the list
        assert status(c, ends)[0] == 0x10, ends
    assert status(c, [0, 0, 0, 0, 0])[0] == 0


def test_padded_batch():
    c = Case([4, 3], [200, 50], [10, 0, 5, 30, 0, 0, 0], seed=3)
    word, out, lse = status(c, c.ii.tolist())
    assert word == 0
    c.check(out, lse)
