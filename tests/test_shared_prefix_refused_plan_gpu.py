"""A plan() that is refused leaves a captured run as it was."""
import pytest
import torch

from dual_b200 import SharedPrefixDecodeWrapper
from test_shared_prefix_gpu import Case, DEV, mixed

pytestmark = pytest.mark.gpu


def test_replay_after_refused_plans():
    c = Case([30, 10], [600, 900], mixed(40), seed=71)
    buf = lambda n: torch.zeros(n, dtype=torch.int32, device=DEV)  # noqa: E731
    w = SharedPrefixDecodeWrapper(torch.full((64 << 20,), 255, dtype=torch.uint8, device=DEV), use_cuda_graph=True,
                                  paged_kv_indptr_buffer=buf(41), paged_kv_indices_buffer=buf(c.own_pages.numel() + 5),
                                  prefix_indices_buffer=buf(1500), plan_buffer=buf(1 << 14))
    w.plan(c.gi, c.pi, c.prefix_pages, c.ii, c.own_pages, 32, 8, 128, 1)
    out, lse = torch.empty_like(c.q), torch.empty((40, 32), device=DEV)
    w.run(c.q, (c.k, c.v), out=out, lse=lse, return_lse=True)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        w.run(c.q, (c.k, c.v), out=out, lse=lse, return_lse=True)
    for other, said in [(Case([5, 35], [1400, 101], [1] * 40, seed=72), "prefix buffer"),
                        (Case([5, 35], [1400, 50], mixed(40), seed=73), None),
                        (Case([40, 0], [500, 5], [40] * 40, seed=74), "indices buffer")]:
        if said is None:  # fewer own entries listed than indptr says
            with pytest.raises(ValueError, match="shorter"):
                w.plan(other.gi, other.pi, other.prefix_pages, other.ii, other.own_pages[:-1], 32, 8, 128, 1)
        else:
            with pytest.raises(ValueError, match=said):
                w.plan(other.gi, other.pi, other.prefix_pages, other.ii, other.own_pages, 32, 8, 128, 1)
        out.fill_(7.0)
        graph.replay()
        c.check(out, lse)
        assert w.status() == 0
