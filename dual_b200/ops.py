"""Torch-tensor front end of the C-ABI kernels (device pointers + current stream).

PyTorch only supplies device memory and streams here; every computation is a
kernel from libdual_b200.so.  Functions validate shapes/dtypes on the host and
launch asynchronously on ``torch.cuda.current_stream()``; all of them are safe
inside CUDA-graph capture (no host synchronisation, no allocation) except
``status`` which reads the device status word back.
"""
from __future__ import annotations

import ctypes as C
import math
from typing import Optional, Sequence, Tuple

import torch

from . import _lib

NUM_QO_HEADS = 32
NUM_KV_HEADS = 8
HEAD_DIM = 128
SLOT_BYTES = NUM_KV_HEADS * HEAD_DIM * 2  # one token slot of one plane (K or V) of one layer


def _ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def _stream(device: torch.device) -> int:
    return torch.cuda.current_stream(device).cuda_stream


def _raw_stream(device: int) -> int:
    """The current stream's handle without a Stream object around it (1-2 us of a call's host time)."""
    return torch._C._cuda_getCurrentRawStream(device)


def _dev(t: torch.Tensor) -> int:
    if t.device.type != "cuda":
        raise ValueError(f"expected a CUDA tensor, got {t.device}")
    return t.device.index


def _check(cond: bool, msg: str) -> None:
    if not cond:
        raise ValueError(msg)


def decode_workspace_size(batch: int, num_ctas: int = 0) -> int:
    return int(_lib.load().dual_decode_workspace_size(int(batch), int(num_ctas)))


def decode_workspace_reset(workspace: torch.Tensor, batch: int) -> None:
    """Zero a decode workspace's status word and arrival counters (once before first use; again after
    a launch that reported a timeout or a bad length)."""
    lib = _lib.load()
    _lib.check(lib.dual_decode_workspace_reset(workspace.data_ptr(), workspace.numel() * workspace.element_size(),
                                               int(batch), _dev(workspace), _stream(workspace.device)))


def default_ctas(device: int = 0) -> int:
    return int(_lib.load().dual_decode_default_ctas(int(device)))


def _pool_stride(pool: torch.Tensor, name: str) -> int:
    """Byte stride between consecutive token slots of an NHD page_size-1 plane."""
    if pool.dtype is not torch.bfloat16:
        raise ValueError(f"{name} must be bf16")
    shape, st = pool.shape, pool.stride()
    if len(shape) == 4:  # [pages, page_size=1, heads, dim]
        if shape[1] != 1:
            raise ValueError(f"{name}: page_size must be 1")
        if st[2:] != (HEAD_DIM, 1):
            raise ValueError(f"{name}: heads x dim must be contiguous")
        if shape[2:] != (NUM_KV_HEADS, HEAD_DIM):
            raise ValueError(f"{name}: expected 8 kv heads x 128")
    else:
        if len(shape) != 3 or shape[1:] != (NUM_KV_HEADS, HEAD_DIM):
            raise ValueError(f"{name}: expected [slots, 8, 128] or [slots, 1, 8, 128]")
        if st[1:] != (HEAD_DIM, 1):
            raise ValueError(f"{name}: heads x dim must be contiguous")
    return st[0] * 2


def tiered_decode(q: torch.Tensor, k_local: torch.Tensor, v_local: torch.Tensor, local_capacity: int,
                  peer_k: Sequence[torch.Tensor], peer_v: Sequence[torch.Tensor],
                  kv_indptr: torch.Tensor, unified_indices: torch.Tensor, sm_scale: float,
                  out: torch.Tensor, lse: Optional[torch.Tensor], workspace: torch.Tensor,
                  num_ctas: int = 0, batch: Optional[int] = None) -> None:
    """One decode layer over the tiered pool (local HBM + supplier banks)."""
    dev = _dev(q)
    B = q.shape[0] if batch is None else int(batch)
    _check(q.dtype == torch.bfloat16 and q.dim() == 3 and tuple(q.shape[1:]) == (NUM_QO_HEADS, HEAD_DIM)
           and q.stride(2) == 1, "q must be bf16 [B, 32, 128] with contiguous head_dim")
    _check(out.dtype == torch.bfloat16 and out.dim() == 3 and out.stride(2) == 1, "out must be bf16 [B, 32, 128]")
    _check(kv_indptr.dtype == torch.int32 and unified_indices.dtype == torch.int32, "indptr/indices must be int32")
    _check(kv_indptr.numel() >= B + 1, "kv_indptr too short")
    if lse is not None:
        _check(lse.dtype == torch.float32 and lse.is_contiguous() and lse.numel() >= B * NUM_QO_HEADS,
               "lse must be contiguous fp32 [B, 32]")
    ls = _pool_stride(k_local, "k_local")
    _check(_pool_stride(v_local, "v_local") == ls, "k/v local pools must share a slot stride")
    n = len(peer_k)
    _check(len(peer_v) == n, "peer_k / peer_v count mismatch")
    pk = (C.c_void_p * max(n, 1))(*[p.data_ptr() for p in peer_k])
    pv = (C.c_void_p * max(n, 1))(*[p.data_ptr() for p in peer_v])
    ps, slots = 0, 0
    if n:
        ps = _pool_stride(peer_k[0], "peer_k0")
        slots = peer_k[0].shape[0]
        for i in range(n):
            _check(_pool_stride(peer_k[i], f"peer_k{i}") == ps and _pool_stride(peer_v[i], f"peer_v{i}") == ps,
                   "all supplier banks must share a slot stride")
            _check(peer_k[i].shape[0] == slots and peer_v[i].shape[0] == slots, "supplier banks differ in size")
    lib = _lib.load()
    _lib.check(lib.dual_tiered_decode(
        q.data_ptr(), q.stride(0), q.stride(1),
        k_local.data_ptr(), v_local.data_ptr(), ls, int(local_capacity),
        pk, pv, n, ps, slots,
        kv_indptr.data_ptr(), unified_indices.data_ptr(), unified_indices.numel(), B,
        float(sm_scale),
        out.data_ptr(), out.stride(0), out.stride(1), _ptr(lse),
        workspace.data_ptr(), workspace.numel() * workspace.element_size(), int(num_ctas),
        dev, _stream(q.device)))


def _host_indptr(t, name: str) -> torch.Tensor:
    t = torch.as_tensor(t)
    if t.dim() != 1 or t.numel() < 1 or t.is_floating_point():
        raise ValueError(f"{name} must be a list of integers [groups + 1]")
    t = t.to("cpu")
    if t.dtype is not torch.int32 and not torch.equal(t.to(torch.int32), t):
        raise ValueError(f"{name} must fit 32 bits")
    return t.to(torch.int32).contiguous()


def shared_prefix_plan(group_indptr, prefix_indptr, num_ctas: int = 0, own_entries: int = -1) -> torch.Tensor:
    """Host-side work plan of a decode with shared prefixes, an int32 CPU tensor: requests
    ``group_indptr[g] .. group_indptr[g + 1]`` share the prefix of ``prefix_indptr[g + 1] - prefix_indptr[g]``
    entries.  It stays valid while both do.  ``own_entries``: how many entries of their own the requests have in all,
    if known; it only decides how many CTAs work on them.  ``group_indptr`` / ``prefix_indptr``: host sequences or
    tensors."""
    gi, pi = _host_indptr(group_indptr, "group_indptr"), _host_indptr(prefix_indptr, "prefix_indptr")
    if gi.numel() != pi.numel():
        raise ValueError("group_indptr and prefix_indptr need one entry per group and one more")
    groups, ctas = gi.numel() - 1, int(num_ctas) or default_ctas(0)
    lib = _lib.load()
    n = C.c_int64(0)
    _lib.check(lib.dual_shared_prefix_plan(gi.data_ptr(), pi.data_ptr(), groups, ctas, own_entries, None, 0, C.byref(n)))
    plan = torch.empty(n.value, dtype=torch.int32)
    _lib.check(lib.dual_shared_prefix_plan(gi.data_ptr(), pi.data_ptr(), groups, ctas, own_entries, plan.data_ptr(),
                                           n.value, C.byref(n)))
    return plan


def shared_prefix_limits(batch: int, groups: int, num_ctas: int = 0) -> Tuple[int, int]:
    """(Workspace bytes, plan words) that are enough for every plan of up to ``batch`` requests in up to ``groups``
    groups, whatever the lengths of the prefixes and of the own lists: what a serving program allocates once."""
    nbytes, words = C.c_size_t(0), C.c_int64(0)
    _lib.check(_lib.load().dual_shared_prefix_limits(int(batch), int(groups), int(num_ctas) or default_ctas(0),
                                                     C.byref(nbytes), C.byref(words)))
    return int(nbytes.value), int(words.value)


def shared_prefix_workspace_size(plan: torch.Tensor) -> int:
    """Workspace bytes of a call with this (host) plan.  A plan for another number of own entries can need more:
    ``shared_prefix_limits`` covers them all."""
    if plan.device.type != "cpu" or plan.dtype is not torch.int32 or not plan.is_contiguous():
        raise ValueError("plan must be a host plan of shared_prefix_plan")
    n = C.c_size_t(0)
    _lib.check(_lib.load().dual_shared_prefix_workspace_size(plan.data_ptr(), plan.numel(), C.byref(n)))
    return int(n.value)


def shared_prefix_decode(q: torch.Tensor, k_local: torch.Tensor, v_local: torch.Tensor, local_capacity: int,
                         peer_k: Sequence[torch.Tensor], peer_v: Sequence[torch.Tensor],
                         prefix_indices: torch.Tensor, kv_indptr: torch.Tensor, unified_indices: torch.Tensor,
                         sm_scale: float, plan: torch.Tensor, out: torch.Tensor, lse: Optional[torch.Tensor],
                         workspace: torch.Tensor, num_ctas: int = 0) -> None:
    """One decode layer of a batch in groups that share prefixes: request b sees its group's part of
    ``prefix_indices`` and its own entries ``unified_indices[kv_indptr[b] .. kv_indptr[b + 1]]``.  ``plan``: that of
    ``shared_prefix_plan`` on the device.  ``workspace``: ``shared_prefix_workspace_size`` bytes; its first word is the
    status word (``status_clear`` it before the first call), the rest may hold anything."""
    dev = q.get_device()
    for t, name in ((kv_indptr, "kv_indptr"), (plan, "plan")):
        if t.dtype is not torch.int32 or t.dim() != 1 or not t.is_contiguous() or t.get_device() != dev:
            raise ValueError(f"{name} must be contiguous int32 [n] on q's device")
    if kv_indptr.numel() < q.shape[0] + 1:
        raise ValueError("kv_indptr too short")
    if not workspace.is_contiguous() or workspace.get_device() != dev:
        raise ValueError("workspace must be contiguous and on q's device")
    _shared_prefix_launch(q, k_local, v_local, local_capacity, peer_k, peer_v, prefix_indices, kv_indptr.data_ptr(),
                          unified_indices, sm_scale, plan.data_ptr(), plan.numel(), out, lse, workspace.data_ptr(),
                          workspace.numel() * workspace.element_size(), num_ctas or default_ctas(dev))


def _shared_prefix_launch(q, k_local, v_local, local_capacity, peer_k, peer_v, prefix_indices, kv_indptr: int,
                          unified_indices, sm_scale, plan: int, plan_words: int, out, lse, workspace: int,
                          workspace_bytes: int, num_ctas: int) -> None:
    """``shared_prefix_decode`` where the index pointer array, the plan and the workspace are the caller's own."""
    dev = q.get_device()
    shape, qt, ot = q.shape, q.stride(), out.stride()
    B = shape[0]
    if q.dtype is not torch.bfloat16 or shape != (B, NUM_QO_HEADS, HEAD_DIM) or qt[2] != 1:
        raise ValueError("q must be bf16 [B, 32, 128] with contiguous head_dim")
    if out.dtype is not torch.bfloat16 or out.shape != shape or ot[2] != 1:
        raise ValueError("out must be bf16 [B, 32, 128] with contiguous head_dim")
    if ot[1] < HEAD_DIM or (B > 1 and ot[0] < HEAD_DIM):
        raise ValueError("out must not repeat rows")
    if (prefix_indices.dtype is not torch.int32 or prefix_indices.dim() != 1 or not prefix_indices.is_contiguous()
            or prefix_indices.get_device() != dev):
        raise ValueError("prefix_indices must be contiguous int32 [n] on q's device")
    if (unified_indices.dtype is not torch.int32 or unified_indices.dim() != 1 or not unified_indices.is_contiguous()
            or unified_indices.get_device() != dev):
        raise ValueError("unified_indices must be contiguous int32 [n] on q's device")
    if lse is not None and (lse.dtype is not torch.float32 or lse.shape != (B, NUM_QO_HEADS) or not lse.is_contiguous()
                            or lse.get_device() != dev):
        raise ValueError("lse must be contiguous fp32 [B, 32] on q's device")
    ls = _pool_stride(k_local, "k_local")
    if v_local.shape != k_local.shape or v_local.dtype is not torch.bfloat16 or v_local.stride() != k_local.stride():
        raise ValueError("k/v local pools must share a slot stride and a size")
    if not 0 <= local_capacity < k_local.shape[0]:
        raise ValueError("local_capacity must be a slot of the local pools")
    if not out.get_device() == k_local.get_device() == v_local.get_device() == dev:
        raise ValueError("out and the pools must be on q's device")
    n = len(peer_k)
    if len(peer_v) != n:
        raise ValueError("peer_k / peer_v count mismatch")
    if n > 8:
        raise ValueError("at most 8 supplier banks")
    pk = pv = None
    ps = slots = 0
    if n:
        bank = peer_k[0]
        ps, slots, bshape, bstride = _pool_stride(bank, "peer_k0"), bank.shape[0], bank.shape, bank.stride()
        for banks, name in ((peer_k, "peer_k"), (peer_v, "peer_v")):
            for i, t in enumerate(banks):
                if (t.dtype is not torch.bfloat16 or t.shape != bshape or t.stride() != bstride
                        or (t.get_device() < 0) != (dev < 0)):
                    raise ValueError(f"{name}{i}: all supplier banks must share a size and a slot stride, on GPUs")
        pk, pv = (C.c_void_p * n)(*[t.data_ptr() for t in peer_k]), (C.c_void_p * n)(*[t.data_ptr() for t in peer_v])
    if dev < 0:
        raise ValueError(f"expected CUDA tensors, got {q.device}")
    row = NUM_QO_HEADS * HEAD_DIM  # one request has no stride of its own
    _lib.check(_lib.load().dual_shared_prefix_decode(
        q.data_ptr(), qt[0] if B > 1 else row, qt[1], k_local.data_ptr(), v_local.data_ptr(), ls, local_capacity, pk,
        pv, n, ps, slots, prefix_indices.data_ptr(), prefix_indices.numel(), kv_indptr, unified_indices.data_ptr(),
        unified_indices.numel(), B, sm_scale, plan, plan_words, out.data_ptr(), ot[0] if B > 1 else row, ot[1],
        None if lse is None else lse.data_ptr(), workspace, workspace_bytes, num_ctas, dev, _raw_stream(dev)))


def append_plan(qo_indptr, kv_indptr, causal: bool, remote_counts=None) -> torch.Tensor:
    """Host-side work list (request, kv head, 64-token query pair, kv tiles it sees), grouped by
    (request, kv head), longest groups first and pairs longest first, as an int32 CPU tensor [n, 4].
    ``qo_indptr`` / ``kv_indptr``: host sequences or CPU tensors.  ``remote_counts`` (optional, per
    request: list entries on suppliers) spreads the items of mostly-remote requests over the launch."""
    qo = torch.as_tensor(qo_indptr, dtype=torch.int32).cpu().contiguous()
    kv = torch.as_tensor(kv_indptr, dtype=torch.int32).cpu().contiguous()
    B = qo.numel() - 1
    rc = None
    if remote_counts is not None:
        rc = torch.as_tensor(remote_counts, dtype=torch.int32).cpu().contiguous()
        _check(rc.numel() == B, "remote_counts needs one count per request")
    lib = _lib.load()
    n = C.c_int64(0)
    _lib.check(lib.dual_append_plan(qo.data_ptr(), kv.data_ptr(), _ptr(rc), B, int(bool(causal)), None, 0,
                                    C.byref(n)))
    work = torch.empty((max(n.value, 1), 4), dtype=torch.int32)
    _lib.check(lib.dual_append_plan(qo.data_ptr(), kv.data_ptr(), _ptr(rc), B, int(bool(causal)), work.data_ptr(),
                                    n.value, C.byref(n)))
    return work[: n.value]


def tiered_append(q: torch.Tensor, k_local: torch.Tensor, v_local: torch.Tensor, local_capacity: int,
                  peer_k: Sequence[torch.Tensor], peer_v: Sequence[torch.Tensor], qo_indptr: torch.Tensor,
                  kv_indptr: torch.Tensor, unified_indices: torch.Tensor, causal: bool, sm_scale: float,
                  work: torch.Tensor, out: torch.Tensor, lse: Optional[torch.Tensor], status: torch.Tensor) -> None:
    """Causal (or non-causal) append attention over the tiered pool; ``work`` from ``append_plan`` on the device."""
    dev = _dev(q)
    _check(q.dtype == torch.bfloat16 and q.dim() == 3 and tuple(q.shape[1:]) == (NUM_QO_HEADS, HEAD_DIM)
           and q.stride(2) == 1, "q must be bf16 [sum q, 32, 128]")
    _check(out.dtype == torch.bfloat16 and out.shape == q.shape and out.stride(2) == 1, "out must match q")
    _check(qo_indptr.dtype == torch.int32 and kv_indptr.dtype == torch.int32 and unified_indices.dtype == torch.int32,
           "indptrs / indices must be int32")
    _check(work.dtype == torch.int32 and work.is_contiguous() and work.device == q.device, "work must be int32 on the device")
    if lse is not None:
        _check(lse.dtype == torch.float32 and lse.is_contiguous(), "lse must be contiguous fp32 [sum q, 32]")
    ls = _pool_stride(k_local, "k_local")
    _check(_pool_stride(v_local, "v_local") == ls, "k/v local pools must share a slot stride")
    n = len(peer_k)
    pk = (C.c_void_p * max(n, 1))(*[t.data_ptr() for t in peer_k])
    pv = (C.c_void_p * max(n, 1))(*[t.data_ptr() for t in peer_v])
    ps = _pool_stride(peer_k[0], "peer_k0") if n else 0
    slots = peer_k[0].shape[0] if n else 0
    lib = _lib.load()
    _lib.check(lib.dual_tiered_append(
        q.data_ptr(), q.stride(0), q.stride(1), k_local.data_ptr(), v_local.data_ptr(), ls, int(local_capacity),
        pk, pv, n, ps, slots, qo_indptr.data_ptr(), kv_indptr.data_ptr(), unified_indices.data_ptr(),
        unified_indices.numel(), qo_indptr.numel() - 1, int(bool(causal)), float(sm_scale), work.data_ptr(),
        work.shape[0], out.data_ptr(), out.stride(0), out.stride(1), _ptr(lse), status.data_ptr(), dev,
        _stream(q.device)))


def pack_read_order(tier: torch.Tensor, slot: torch.Tensor, req_pool_indices: torch.Tensor,
                    seq_lens: torch.Tensor, local_capacity: int, remote_rows: int, tile_rows: int,
                    full_out: torch.Tensor, prefix_lens: Optional[torch.Tensor] = None,
                    history_out: Optional[torch.Tensor] = None, new_loc: Optional[torch.Tensor] = None,
                    status: Optional[torch.Tensor] = None) -> None:
    """Unified index list in the interleaved read order (decode: prefix_lens=None)."""
    dev = _dev(tier)
    for name, t in (("tier", tier), ("slot", slot), ("req_pool_indices", req_pool_indices),
                    ("seq_lens", seq_lens), ("full_out", full_out)):
        _check(t.dtype == torch.int32, f"{name} must be int32")
    _check(tier.shape == slot.shape and tier.stride() == slot.stride() and tier.stride(1) == 1,
           "tier/slot must be row-major tables of one shape")
    if prefix_lens is not None:
        _check(prefix_lens.dtype == torch.int32, "prefix_lens must be int32")
    if new_loc is not None:
        _check(new_loc.dtype == torch.int64, "new_loc must be int64 (out_cache_loc)")
    B = req_pool_indices.numel()
    lib = _lib.load()
    _lib.check(lib.dual_pack_read_order(
        tier.data_ptr(), slot.data_ptr(), tier.shape[0], tier.stride(0), req_pool_indices.data_ptr(), seq_lens.data_ptr(),
        _ptr(prefix_lens), _ptr(new_loc), B, int(local_capacity), int(remote_rows), int(tile_rows),
        full_out.data_ptr(), _ptr(history_out), _ptr(status), dev, _stream(tier.device)))


def write_prefill_layout(tier: torch.Tensor, slot: torch.Tensor, req_pool_indices: torch.Tensor,
                         start: torch.Tensor, length: torch.Tensor, prefix: torch.Tensor,
                         locations: torch.Tensor, max_length: int, status: Optional[torch.Tensor] = None) -> None:
    """tier=0, slot=locations for the newly appended positions of every request."""
    dev = _dev(tier)
    _check(locations.dtype in (torch.int64, torch.int32), "locations must be int32 or int64")
    for name, t in (("req", req_pool_indices), ("start", start), ("length", length), ("prefix", prefix)):
        _check(t.dtype == torch.int32, f"{name} must be int32")
    lib = _lib.load()
    _lib.check(lib.dual_write_prefill_layout(
        tier.data_ptr(), slot.data_ptr(), tier.shape[0], tier.stride(0), req_pool_indices.data_ptr(),
        start.data_ptr(), length.data_ptr(), prefix.data_ptr(), locations.data_ptr(),
        int(locations.dtype == torch.int64), req_pool_indices.numel(), int(max_length), _ptr(status), dev,
        _stream(tier.device)))


def set_kv_buffer(k_local: torch.Tensor, v_local: torch.Tensor, locations: torch.Tensor, k: torch.Tensor,
                  v: torch.Tensor, status: torch.Tensor) -> None:
    """New tokens' K / V rows ``[n, 8, 128]`` (token stride free) into local slots ``locations``
    (SGLang ``out_cache_loc``, int64 or int32) of one layer's pools; bad slots are skipped and recorded."""
    ls = _pool_stride(k_local, "k_local")
    _check(_pool_stride(v_local, "v_local") == ls, "k/v local pools must share a slot stride")
    n = locations.numel()
    for t, name in ((k, "k"), (v, "v")):
        _check(t.dtype == torch.bfloat16 and t.dim() == 3 and tuple(t.shape[1:]) == (NUM_KV_HEADS, HEAD_DIM)
               and t.stride(2) == 1 and t.stride(1) == HEAD_DIM and t.shape[0] == n,
               f"{name} must be bf16 [n, 8, 128] with heads x dims contiguous")
    _check(locations.dtype in (torch.int64, torch.int32) and locations.is_contiguous(), "locations must be int64/int32")
    _check(status.dtype in (torch.int32, torch.uint32) and status.numel() >= 1, "status must be a 32-bit word")
    lib = _lib.load()
    _lib.check(lib.dual_set_kv_buffer(
        k_local.data_ptr(), v_local.data_ptr(), ls, k_local.shape[0] - 1, k.data_ptr(), k.stride(0), v.data_ptr(),
        v.stride(0), locations.data_ptr(), int(locations.dtype == torch.int64), n, status.data_ptr(), _dev(k_local),
        _stream(k_local.device)))


def _rows(t: torch.Tensor, n: int, heads: int, name: str, device: int) -> Tuple[int, int]:
    """(pointer, token stride) of ``t``, checked to be bf16 [n, heads, 128], heads x dims contiguous, on ``device``."""
    st = t.stride()
    if not (t.dtype is torch.bfloat16 and t.shape == (n, heads, HEAD_DIM) and (n == 0 or st[1:] == (HEAD_DIM, 1))):
        raise ValueError(f"{name} must be bf16 [n, {heads}, 128] with heads x dims contiguous")
    if t.get_device() != device:
        raise ValueError(f"{name} must be on the pools' device")
    return t.data_ptr(), st[0] if n > 1 else heads * HEAD_DIM  # one token has no stride of its own


def _index(t: torch.Tensor, n: int, name: str, device: int) -> int:
    """Whether ``t``, checked to be contiguous [n] integers on ``device``, has 64 bits."""
    if not ((t.dtype is torch.int64 or t.dtype is torch.int32) and t.shape == (n,) and t.is_contiguous()):
        raise ValueError(f"{name} must be contiguous int64/int32 [n]")
    if t.get_device() != device:
        raise ValueError(f"{name} must be on the pools' device")
    return int(t.dtype is torch.int64)


def _weight(t: Optional[torch.Tensor], name: str, device: int) -> Optional[int]:
    if t is None:
        return None
    if not (t.dtype is torch.bfloat16 and t.shape == (HEAD_DIM,) and t.is_contiguous()):
        raise ValueError(f"{name} must be contiguous bf16 [128]")
    if t.get_device() != device:
        raise ValueError(f"{name} must be on the pools' device")
    return t.data_ptr()


def _overlap(a: int, a_step: int, a_size: int, b: int, b_step: int, b_size: int, n: int) -> bool:
    """Whether n rows of ``a_size`` bytes every ``a_step`` from ``a`` on meet those of ``b``.  Rows at one step
    that lie side by side (a fused projection's q | k | v) do not."""
    if a + (n - 1) * a_step + a_size <= b or b + (n - 1) * b_step + b_size <= a:
        return False
    if a_step == b_step and a_step > 0:
        at = (b - a) % a_step
        return at < a_size or at + b_size > a_step
    return True


def rope_set_kv_buffer(k_local: torch.Tensor, v_local: torch.Tensor, locations: torch.Tensor,
                       positions: torch.Tensor, cos_sin: torch.Tensor, q: torch.Tensor, k: torch.Tensor,
                       v: torch.Tensor, q_out: torch.Tensor, status: torch.Tensor, *, interleaved: bool = False,
                       q_norm_weight: Optional[torch.Tensor] = None, k_norm_weight: Optional[torch.Tensor] = None,
                       norm_eps: float = 1e-6) -> None:
    """``set_kv_buffer`` with the position rotation on the way: ``q`` [n, 32, 128] rotated into ``q_out``
    (which may be ``q``), ``k`` [n, 8, 128] rotated and ``v`` as it is into local slots ``locations`` of one
    layer's pools.  ``positions`` [n] name rows of ``cos_sin`` (fp32 [positions, rotary dims]: cosines, then
    sines); the first ``rotary dims`` of each head are turned, in pairs (j, j + half) or, ``interleaved``,
    (2j, 2j + 1).  With norm weights [128] bf16 each q / k head row is RMS-normalised first.  Token strides
    are free (views of a fused qkv buffer); otherwise q, k, v, ``q_out`` and the pools do not overlap.  Tokens with a bad position are skipped, rows with a bad slot are
    not stored; both are recorded in ``status``."""
    ls = _pool_stride(k_local, "k_local")
    if not (v_local.shape == k_local.shape and v_local.dtype is k_local.dtype
            and v_local.stride() == k_local.stride()):
        raise ValueError("k/v local pools must share a slot stride and a size")
    dev = k_local.get_device()
    n = locations.numel()
    loc64, pos64 = _index(locations, n, "locations", dev), _index(positions, n, "positions", dev)
    qp, qs = _rows(q, n, NUM_QO_HEADS, "q", dev)
    kp, ks = _rows(k, n, NUM_KV_HEADS, "k", dev)
    vp, vs = _rows(v, n, NUM_KV_HEADS, "v", dev)
    op, os_ = _rows(q_out, n, NUM_QO_HEADS, "q_out", dev)
    if not (cos_sin.dtype is torch.float32 and cos_sin.dim() == 2 and cos_sin.is_contiguous()):
        raise ValueError("cos_sin must be contiguous fp32 [positions, rotary dims]")
    qw, kw = _weight(q_norm_weight, "q_norm_weight", dev), _weight(k_norm_weight, "k_norm_weight", dev)
    if not (status.dtype in (torch.int32, torch.uint32) and status.numel() >= 1):
        raise ValueError("status must be a 32-bit word")
    if not (v_local.get_device() == cos_sin.get_device() == status.get_device() == dev):
        raise ValueError("v_local, cos_sin and status must be on the pools' device")
    q_row, kv_row = NUM_QO_HEADS * HEAD_DIM * 2, NUM_KV_HEADS * HEAD_DIM * 2
    if (op, os_) != (qp, qs) and _overlap(op, 2 * os_, q_row, qp, 2 * qs, q_row, n):
        raise ValueError("q_out must be q itself or not overlap it")
    if (_overlap(op, 2 * os_, q_row, kp, 2 * ks, kv_row, n)
            or _overlap(op, 2 * os_, q_row, vp, 2 * vs, kv_row, n)):
        raise ValueError("q_out must not overlap k or v")
    if dev < 0:
        raise ValueError(f"expected CUDA tensors, got {k_local.device}")
    max_pos, rotary = cos_sin.shape
    _lib.check(_lib.load().dual_rope_set_kv_buffer(
        k_local.data_ptr(), v_local.data_ptr(), ls, k_local.shape[0] - 1, locations.data_ptr(), loc64,
        positions.data_ptr(), pos64, cos_sin.data_ptr(), max_pos, rotary, bool(interleaved), qp, qs, kp, ks, vp, vs,
        op, os_, qw, kw, norm_eps, n, status.data_ptr(), dev, _raw_stream(dev)))


def merge_attention_states(states: Sequence[torch.Tensor], lses: Sequence[torch.Tensor], out: torch.Tensor,
                           lse: Optional[torch.Tensor] = None) -> None:
    """Join 1 to 8 partial attention states of the same queries over disjoint keys (what
    ``run_return_lse`` returns): ``states[i]`` [T, 32, 128], all bf16 or all fp32, ``lses[i]`` fp32 [T, 32]
    (base 2).  ``out`` [T, 32, 128] bf16 or fp32 and ``lse`` [T, 32] (optional) may be one of them."""
    n = len(states)
    if not (1 <= n <= 8 and len(lses) == n):
        raise ValueError("need 1 to 8 states, each with its lse")
    dev = out.get_device()
    T = out.shape[0]
    shape, lse_shape, row = (T, NUM_QO_HEADS, HEAD_DIM), (T, NUM_QO_HEADS), NUM_QO_HEADS * HEAD_DIM
    st = out.stride()
    if not ((out.dtype is torch.bfloat16 or out.dtype is torch.float32) and out.shape == shape
            and (T == 0 or st[2] == 1)):
        raise ValueError("out must be bf16 or fp32 [T, 32, 128] with contiguous head_dim")
    op, ot, oh, oe = out.data_ptr(), st[0] if T > 1 else row, st[1], out.element_size()
    if oh < HEAD_DIM or ot < HEAD_DIM:
        raise ValueError("out must not repeat rows")
    osize = oe * (oh * (NUM_QO_HEADS - 1) + HEAD_DIM)  # bytes from a token's first value to its last
    oend = op + oe * (T - 1) * ot + osize
    lp = None
    if lse is not None:
        if not (lse.dtype is torch.float32 and lse.shape == lse_shape and lse.is_contiguous()
                and lse.get_device() == dev):
            raise ValueError("lse must be contiguous fp32 [T, 32] on out's device")
        lp = lse.data_ptr()
    dtype = states[0].dtype
    e = 2 if dtype is torch.bfloat16 else 4
    ptrs, toks, heads, lptrs = (C.c_void_p * n)(), (C.c_int64 * n)(), (C.c_int64 * n)(), (C.c_void_p * n)()
    for i in range(n):
        s, l = states[i], lses[i]
        st = s.stride()
        if not ((dtype is torch.bfloat16 or dtype is torch.float32) and s.shape == shape and (T == 0 or st[2] == 1)
                and s.get_device() == dev):
            raise ValueError(f"states[{i}] must be bf16 or fp32 [T, 32, 128] with contiguous head_dim on out's device")
        if s.dtype is not dtype:
            raise ValueError("states must share a type")
        sp, tok, head = s.data_ptr(), st[0] if T > 1 else row, st[1]
        if sp < oend and (sp, tok, head, e) != (op, ot, oh, oe) and _overlap(
                op, oe * ot, osize, sp, e * tok, e * (head * (NUM_QO_HEADS - 1) + HEAD_DIM), T):
            # of the same strides, their rows may still lie side by side: both start at multiples of one distance
            step = math.gcd(oe * ot, oe * oh)
            at = (sp - op) % step
            if (e * tok, e * head) != (oe * ot, oe * oh) or at < oe * HEAD_DIM or at + e * HEAD_DIM > step:
                raise ValueError("out must be one of the states or not overlap them")
        if not (l.dtype is torch.float32 and l.shape == lse_shape and l.is_contiguous() and l.get_device() == dev):
            raise ValueError(f"lses[{i}] must be contiguous fp32 [T, 32] on out's device")
        a = l.data_ptr()
        if lp is not None and a != lp and abs(a - lp) < T * NUM_QO_HEADS * 4:
            raise ValueError("lse must be one of the lses or not overlap them")
        ptrs[i], toks[i], heads[i], lptrs[i] = sp, tok, head, a
    if dev < 0:
        raise ValueError(f"expected CUDA tensors, got {out.device}")
    _lib.check(_lib.load().dual_merge_attention_states(ptrs, toks, heads, lptrs, n, e == 4, T, op, ot, oh, oe == 4, lp,
                                                       dev, _raw_stream(dev)))


def migrate_copy(local_planes: torch.Tensor, remote_planes: torch.Tensor, num_planes: int, num_banks: int,
                 source: torch.Tensor, target: torch.Tensor, reverse: bool, local_slots: int,
                 remote_slots: int, status: torch.Tensor, row_bytes: int = SLOT_BYTES, max_ctas: int = 0) -> None:
    """Byte-exact copy of token slots across all planes between the local pool and supplier banks."""
    dev = _dev(source)
    _check(local_planes.dtype == torch.int64 and remote_planes.dtype == torch.int64, "pointer tables must be int64")
    _check(local_planes.numel() >= num_planes and remote_planes.numel() >= num_banks * num_planes,
           "pointer tables too short")
    _check(source.dtype == torch.int64 and target.dtype == torch.int64 and source.numel() == target.numel(),
           "source/target must be int64 of equal length")
    _check(status.dtype in (torch.int32, torch.uint32) and status.numel() >= 1, "status must be a 32-bit word")
    lib = _lib.load()
    _lib.check(lib.dual_migrate_copy(
        local_planes.data_ptr(), remote_planes.data_ptr(), int(num_planes), int(num_banks), source.data_ptr(),
        target.data_ptr(), source.numel(), int(bool(reverse)), int(row_bytes), int(local_slots), int(remote_slots),
        status.data_ptr(), int(max_ctas), dev, _stream(source.device)))


def stage_remote_rows(peer_k: Sequence[torch.Tensor], peer_v: Sequence[torch.Tensor],
                      stage_k: Sequence[torch.Tensor], stage_v: Sequence[torch.Tensor],
                      unified_indices: torch.Tensor, local_capacity: int, status: torch.Tensor,
                      num_indices: Optional[int] = None, max_ctas: int = 0) -> None:
    """Copy the supplier rows the index list names (both planes) into the same rows of local stage
    buffers, which then replace the banks in ``tiered_append`` with the index list unchanged."""
    _check(unified_indices.dtype == torch.int32 and unified_indices.is_contiguous(), "indices must be contiguous int32")
    _check(status.dtype in (torch.int32, torch.uint32) and status.numel() >= 1, "status must be a 32-bit word")
    n, slots, ps, ss = _stage_shapes(peer_k, peer_v, stage_k, stage_v, unified_indices.device)
    count = unified_indices.numel() if num_indices is None else int(num_indices)
    _check(0 <= count <= unified_indices.numel(), "num_indices out of range")
    lib = _lib.load()
    _lib.check(lib.dual_stage_remote_rows(
        _ptrs(peer_k), _ptrs(peer_v), _ptrs(stage_k), _ptrs(stage_v), n, ps, ss, slots, SLOT_BYTES,
        unified_indices.data_ptr(), count, int(local_capacity), status.data_ptr(), int(max_ctas),
        _dev(unified_indices), _stream(unified_indices.device)))


def stage_bank_range(peer_k: Sequence[torch.Tensor], peer_v: Sequence[torch.Tensor],
                     stage_k: Sequence[torch.Tensor], stage_v: Sequence[torch.Tensor],
                     row_ranges: Sequence[Sequence[int]], streams: Sequence[torch.cuda.Stream]) -> None:
    """Copy rows [begin, end) of both planes of every bank into the same rows of its stage buffers
    on the copy engines, bank b on ``streams[b]`` (no SM work)."""
    n, slots, ps, ss = _stage_shapes(peer_k, peer_v, stage_k, stage_v, stage_k[0].device)
    _check(len(row_ranges) == n and len(streams) == n, "need one row range and one stream per bank")
    begin = (C.c_int64 * n)(*[int(r[0]) for r in row_ranges])
    end = (C.c_int64 * n)(*[int(r[1]) for r in row_ranges])
    handles = (C.c_void_p * n)(*[s.cuda_stream for s in streams])
    lib = _lib.load()
    _lib.check(lib.dual_stage_bank_range(
        _ptrs(peer_k), _ptrs(peer_v), _ptrs(stage_k), _ptrs(stage_v), n, ps, ss, slots, SLOT_BYTES, begin, end,
        handles, _dev(stage_k[0])))


def _ptrs(ts: Sequence[torch.Tensor]):
    return (C.c_void_p * len(ts))(*[t.data_ptr() for t in ts])


def _stage_shapes(peer_k, peer_v, stage_k, stage_v, device):
    """(banks, rows, bank stride, stage stride) after checking every bank / stage plane."""
    n = len(peer_k)
    _check(n >= 1 and len(peer_v) == n and len(stage_k) == n and len(stage_v) == n,
           "need one (k, v) bank and one (k, v) stage buffer per supplier")
    slots = peer_k[0].shape[0]
    ps = _pool_stride(peer_k[0], "peer_k0")
    ss = _pool_stride(stage_k[0], "stage_k0")
    for i in range(n):
        for t, name, stride in ((peer_k[i], "peer_k", ps), (peer_v[i], "peer_v", ps), (stage_k[i], "stage_k", ss),
                                (stage_v[i], "stage_v", ss)):
            _check(t.shape[0] == slots and _pool_stride(t, f"{name}{i}") == stride,
                   f"{name}{i}: every bank and stage buffer needs the same rows and stride")
        _check(stage_k[i].device == device and stage_v[i].device == device,
               "stage buffers must be on the index list's device")
    return n, slots, ps, ss


def debug_inject(mask: int) -> None:
    """Test hook: DUAL_INJECT_* bits for the following launches (0 disables; see dual_b200.h)."""
    _lib.check(_lib.load().dual_debug_inject(int(mask)))


INJECT_APPEND_WITHHOLD_K0 = 0x1
STATUS_WAIT_TIMEOUT = 0x4


def status_clear(status: torch.Tensor) -> None:
    lib = _lib.load()
    _lib.check(lib.dual_status_clear(status.data_ptr(), _dev(status), _stream(status.device)))


def status_read(status: torch.Tensor) -> int:
    lib = _lib.load()
    v = C.c_uint32(0)
    _lib.check(lib.dual_status_read(status.data_ptr(), C.byref(v), _dev(status), _stream(status.device)))
    return int(v.value)
