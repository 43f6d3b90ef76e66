"""The buffers and lists that SharedPrefixDecodeWrapper takes over (no GPU): what it refuses before it writes any."""
import pytest
import torch

from dual_b200 import SharedPrefixDecodeWrapper


def buf(n=4096, **kw):
    return torch.zeros(n, dtype=torch.int32, **kw)


NAMES = {"paged_kv_indptr_buffer": "indptr", "paged_kv_indices_buffer": "indices", "prefix_indices_buffer": "prefix",
         "plan_buffer": "plan"}
BAD = {"int64": lambda: buf().long(), "int32 in float": lambda: buf().view(torch.float32), "strided": lambda: buf()[::2],
       "two dimensions": lambda: buf().view(64, 64), "another device": lambda: buf(device="meta")}


@pytest.mark.parametrize("graph", [False, True])
@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("kind", BAD)
def test_buffers_that_are_no_words_of_the_device(name, kind, graph):
    """The kernel reads a buffer as that many int32 words at its address, with or without graphs."""
    buffers = {n: buf() for n in NAMES}
    buffers[name] = BAD[kind]()
    with pytest.raises(ValueError, match=NAMES[name] + " buffer must"):
        SharedPrefixDecodeWrapper(torch.zeros(1 << 20, dtype=torch.uint8), use_cuda_graph=graph, num_ctas=8, **buffers)


@pytest.mark.parametrize("graph", [False, True])
def test_plan_buffer_off_its_alignment(graph):
    buffers = {n: buf() for n in NAMES}
    buffers["plan_buffer"] = buf()[1:]
    with pytest.raises(ValueError, match="plan buffer"):
        SharedPrefixDecodeWrapper(torch.zeros(1 << 20, dtype=torch.uint8), use_cuda_graph=graph, num_ctas=8, **buffers)
    buffers["plan_buffer"] = buf()[4:]
    SharedPrefixDecodeWrapper(torch.zeros(1 << 20, dtype=torch.uint8), use_cuda_graph=graph, num_ctas=8, **buffers)


def wrapper(graph, indptr=4, indices=64, prefix=64, plan=4096, fill=-9):
    buf = lambda n: torch.full((n,), fill, dtype=torch.int32)  # noqa: E731
    buffers = dict(paged_kv_indptr_buffer=buf(indptr), paged_kv_indices_buffer=buf(indices),
                   prefix_indices_buffer=buf(prefix), plan_buffer=buf(plan))
    w = SharedPrefixDecodeWrapper(torch.zeros(1 << 22, dtype=torch.uint8), use_cuda_graph=graph, num_ctas=8,
                                  **(buffers if graph else {}))
    return w, buffers


def plan(w, prefix=20, listed=None, own=(5, 0, 7), own_listed=None):
    """A plan of three requests of one group, up to the GPU call at its end; lists may be shorter than they should be."""
    ids = lambda n: torch.arange(n, dtype=torch.int32)  # noqa: E731
    ends = torch.tensor([0] + list(own)).cumsum(0)
    try:
        w.plan([0, 3], [0, prefix], ids(prefix if listed is None else listed), ends,
               ids(sum(own) if own_listed is None else own_listed), 32, 8, 128, 1)
    except ValueError as e:
        if not str(e).startswith("expected a CUDA tensor"):
            raise


@pytest.mark.parametrize("graph", [False, True])
@pytest.mark.parametrize("own_listed", [0, 1, 11])
def test_lists_shorter_than_their_indptr(graph, own_listed):
    """With graphs the kernel is given the whole buffer, so it would read what an earlier plan left there."""
    w, _ = wrapper(graph)
    plan(w)
    with pytest.raises(ValueError, match="indices is shorter than the requests' own entries"):
        plan(w, own_listed=own_listed)
    with pytest.raises(ValueError, match="prefix_indices is shorter"):
        plan(w, listed=19)
    plan(w, own_listed=12)
    plan(w, own_listed=30)  # longer ones are taken


@pytest.mark.parametrize("short", [dict(indptr=3), dict(indices=11), dict(prefix=19), dict(plan=100)])
def test_a_refused_plan_writes_nothing(short):
    """A captured run is replayed on these buffers: a new work plan beside old lists would be a mixture of both."""
    w, buffers = wrapper(True, **short)
    with pytest.raises(ValueError, match="exceed the CUDA-graph"):
        plan(w)
    for name, t in buffers.items():
        assert bool((t == -9).all()), name


def test_a_plan_writes_each_buffer():
    w, buffers = wrapper(True, indptr=4, indices=12, prefix=20)
    plan(w)
    assert buffers["paged_kv_indptr_buffer"].tolist() == [0, 5, 5, 12]
    assert buffers["paged_kv_indices_buffer"].tolist() == list(range(12))
    assert buffers["prefix_indices_buffer"].tolist() == list(range(20))


@pytest.mark.parametrize("change", [
    dict(prefix_indices=torch.zeros((1, 20), dtype=torch.int32)), dict(indices=torch.zeros((2, 6), dtype=torch.int32)),
    dict(indptr=torch.tensor([[0, 5, 5, 12]])), dict(indices=torch.zeros(12)), dict(prefix_indices=torch.zeros(20))])
def test_lists_of_another_shape_write_nothing(change):
    w, buffers = wrapper(True)
    lists = dict(prefix_indices=torch.zeros(20, dtype=torch.int32), indptr=torch.tensor([0, 5, 5, 12]),
                 indices=torch.zeros(12, dtype=torch.int32))
    with pytest.raises(ValueError, match="list of integers"):
        w.plan([0, 3], [0, 20], **{**lists, **change}, num_qo_heads=32, num_kv_heads=8, head_dim=128, page_size=1)
    for name, t in buffers.items():
        assert bool((t == -9).all()), name
