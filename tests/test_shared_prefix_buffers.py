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
