"""PyTorch-facing operator surface of the B200 decode engine.

The four functions below keep the names, argument order, argument meaning and
error behaviour (``RuntimeError`` with the same messages) of the reference's
extension module, ``tests/persistentkv_torch_extension.cu:319-336``, so the
reference's serving harness can load this module in place of its own:

    paged_attention(q, k_pages, v_pages, block_table, output, workspace,
                    context, page_size, num_splits)
    paged_attention_masked(q, k_pages, v_pages, block_table, seq_lens, output,
                           workspace, bucket_context, page_size, num_splits)
    paged_attention_indexed(q_source, k_pages, v_pages, block_table, seq_lens,
                            q_indices, out_indices, output, workspace,
                            bucket_context, page_size, num_splits)
    paged_attention_workqueue(q_source, k_pages, v_pages, block_table, seq_lens,
                              work_items, split_offsets, merge_counters,
                              q_indices, out_indices, output, workspace,
                              bucket_context, page_size, total_partial_slots,
                              fused_merge)

Each call only validates tensors and forwards raw pointers to the C ABI of
``libpkv_b200.so`` on the current CUDA stream; PyTorch supplies device memory
and streams, never the computation.  Beyond the reference, q/K/V/output may be
bfloat16 (all of them), and two calls serve sequence sharding across GPUs
(``paged_attention_workqueue_state`` and ``combine_states``).
"""

from __future__ import annotations

import torch

from . import _native

HEAD_DIM = 128
STATE_STRIDE = HEAD_DIM + 2

_DTYPES = {torch.float16: _native.PKV_DTYPE_F16, torch.bfloat16: _native.PKV_DTYPE_BF16}
_SUPPORTED_G = (1, 2, 4, 8)


def _check_tensor(tensor: torch.Tensor, name: str, dtype, dims: int) -> None:
    # reference check_tensor (tests/persistentkv_torch_extension.cu:9-19)
    if not tensor.is_cuda:
        raise RuntimeError(f"{name} must be a CUDA tensor")
    if (tensor.dtype not in dtype) if isinstance(dtype, tuple) else tensor.dtype != dtype:
        raise RuntimeError(f"{name} has wrong dtype")
    if tensor.dim() != dims:
        raise RuntimeError(f"{name} has wrong rank")
    if not tensor.is_contiguous():
        raise RuntimeError(f"{name} must be contiguous")


def _check_supported_gqa(hq: int, hkv: int) -> None:
    # reference check_supported_gqa (tests/persistentkv_torch_extension.cu:21-31)
    if hkv <= 0:
        raise RuntimeError("Hkv must be positive")
    if hq % hkv != 0:
        raise RuntimeError("Hq must be divisible by Hkv")
    g = hq // hkv
    if g not in (1, 2, 4, 8):
        raise RuntimeError(
            f"PersistentKV supports G=Hq/Hkv in {{1,2,4,8}}; got G={g} from Hq={hq} Hkv={hkv}"
        )


def _check_kv(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, page_size: int):
    dt = q.dtype
    _check_tensor(k_pages, "k_pages", dt, 4)
    _check_tensor(v_pages, "v_pages", dt, 4)
    d = q.size(2)
    hkv = k_pages.size(1)
    physical_pages = k_pages.size(0)
    if d != HEAD_DIM:
        raise RuntimeError("PersistentKV extension currently requires d=128")
    if not (v_pages.size(0) == physical_pages and v_pages.size(1) == hkv
            and v_pages.size(2) == page_size and v_pages.size(3) == d):
        raise RuntimeError("v_pages shape mismatch")
    if not (k_pages.size(2) == page_size and k_pages.size(3) == d):
        raise RuntimeError("k_pages shape mismatch")
    return hkv, physical_pages


def _workspace(workspace: torch.Tensor):
    if not workspace.is_cuda:
        raise RuntimeError("workspace must be a CUDA tensor")
    if not workspace.is_contiguous():
        raise RuntimeError("workspace must be contiguous")
    if workspace.numel() == 0:
        return None, 0
    return workspace.data_ptr(), workspace.numel() * workspace.element_size()


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _stream() -> int:
    """Raw ``cudaStream_t`` of the current stream on the current device (the
    raw getter avoids building a ``torch.cuda.Stream`` object per call)."""
    if _raw_stream is not None:
        return _raw_stream(torch.cuda.current_device())
    return torch.cuda.current_stream().cuda_stream


def _positive(value: int, name: str) -> None:
    if value <= 0:
        raise RuntimeError(f"{name} must be positive")


def paged_attention(q, k_pages, v_pages, block_table, output, workspace, context: int,
                    page_size: int, num_splits: int) -> None:
    """Reference ``persistentkv_paged_attention`` (extension :35-93)."""
    _check_tensor(q, "q", tuple(_DTYPES), 3)
    hkv, physical_pages = _check_kv(q, k_pages, v_pages, page_size)
    _check_tensor(block_table, "block_table", torch.int32, 2)
    _check_tensor(output, "output", q.dtype, 3)
    ws_ptr, ws_bytes = _workspace(workspace)
    b, hq, d = q.shape
    if not (output.size(0) == b and output.size(1) == hq and output.size(2) == d):
        raise RuntimeError("output shape must match q")
    if block_table.size(0) != b:
        raise RuntimeError("block_table batch mismatch")
    _check_supported_gqa(hq, hkv)
    _positive(context, "context")
    _positive(page_size, "page_size")
    _positive(num_splits, "num_splits")
    lib = _native.load()
    _native.check(lib.pkv_paged_attention(
        q.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), block_table.data_ptr(),
        output.data_ptr(), ws_ptr, ws_bytes, b, hq, hkv, d, physical_pages, page_size,
        block_table.size(1), int(context), int(num_splits), _DTYPES[q.dtype], _stream()))


def paged_attention_masked(q, k_pages, v_pages, block_table, seq_lens, output, workspace,
                           bucket_context: int, page_size: int, num_splits: int) -> None:
    """Reference ``persistentkv_paged_attention_masked`` (extension :95-157)."""
    _check_tensor(q, "q", tuple(_DTYPES), 3)
    hkv, physical_pages = _check_kv(q, k_pages, v_pages, page_size)
    _check_tensor(block_table, "block_table", torch.int32, 2)
    _check_tensor(seq_lens, "seq_lens", torch.int32, 1)
    _check_tensor(output, "output", q.dtype, 3)
    ws_ptr, ws_bytes = _workspace(workspace)
    b, hq, d = q.shape
    if not (output.size(0) == b and output.size(1) == hq and output.size(2) == d):
        raise RuntimeError("output shape must match q")
    if seq_lens.size(0) != b:
        raise RuntimeError("seq_lens batch mismatch")
    if block_table.size(0) != b:
        raise RuntimeError("block_table batch mismatch")
    _check_supported_gqa(hq, hkv)
    _positive(bucket_context, "bucket_context")
    _positive(page_size, "page_size")
    _positive(num_splits, "num_splits")
    lib = _native.load()
    _native.check(lib.pkv_paged_attention_masked(
        q.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), block_table.data_ptr(),
        seq_lens.data_ptr(), output.data_ptr(), ws_ptr, ws_bytes, b, hq, hkv, d,
        physical_pages, page_size, block_table.size(1), int(bucket_context), int(num_splits),
        _DTYPES[q.dtype], _stream()))


def paged_attention_indexed(q_source, k_pages, v_pages, block_table, seq_lens, q_indices,
                            out_indices, output, workspace, bucket_context: int,
                            page_size: int, num_splits: int) -> None:
    """Reference ``persistentkv_paged_attention_indexed`` (extension :159-228)."""
    _check_tensor(q_source, "q_source", tuple(_DTYPES), 3)
    hkv, physical_pages = _check_kv(q_source, k_pages, v_pages, page_size)
    _check_tensor(block_table, "block_table", torch.int32, 2)
    _check_tensor(seq_lens, "seq_lens", torch.int32, 1)
    _check_tensor(q_indices, "q_indices", torch.int32, 1)
    _check_tensor(out_indices, "out_indices", torch.int32, 1)
    _check_tensor(output, "output", q_source.dtype, 3)
    ws_ptr, ws_bytes = _workspace(workspace)
    b = block_table.size(0)
    hq, d = q_source.size(1), q_source.size(2)
    if not (output.size(1) == hq and output.size(2) == d):
        raise RuntimeError("output shape must match q head dimensions")
    if seq_lens.size(0) != b:
        raise RuntimeError("seq_lens batch mismatch")
    if q_indices.size(0) != b:
        raise RuntimeError("q_indices batch mismatch")
    if out_indices.size(0) != b:
        raise RuntimeError("out_indices batch mismatch")
    _check_supported_gqa(hq, hkv)
    _positive(bucket_context, "bucket_context")
    _positive(page_size, "page_size")
    _positive(num_splits, "num_splits")
    lib = _native.load()
    _native.check(lib.pkv_paged_attention_indexed(
        q_source.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), block_table.data_ptr(),
        seq_lens.data_ptr(), q_indices.data_ptr(), out_indices.data_ptr(), output.data_ptr(),
        ws_ptr, ws_bytes, b, q_source.size(0), output.size(0), hq, hkv, d, physical_pages,
        page_size, block_table.size(1), int(bucket_context), int(num_splits),
        _DTYPES[q_source.dtype], _stream()))


def _check_workqueue(q_source, k_pages, v_pages, block_table, seq_lens, work_items,
                     split_offsets, merge_counters, q_indices, page_size):
    _check_tensor(q_source, "q_source", tuple(_DTYPES), 3)
    hkv, physical_pages = _check_kv(q_source, k_pages, v_pages, page_size)
    _check_tensor(block_table, "block_table", torch.int32, 2)
    _check_tensor(seq_lens, "seq_lens", torch.int32, 1)
    _check_tensor(work_items, "work_items", torch.int32, 2)
    _check_tensor(split_offsets, "split_offsets", torch.int32, 1)
    _check_tensor(merge_counters, "merge_counters", torch.int32, 2)
    _check_tensor(q_indices, "q_indices", torch.int32, 1)
    b = block_table.size(0)
    if work_items.size(1) != 5:
        raise RuntimeError("work_items must have shape [T, 5]")
    if split_offsets.size(0) != b + 1:
        raise RuntimeError("split_offsets batch mismatch")
    if not (merge_counters.size(0) == b and merge_counters.size(1) == hkv):
        raise RuntimeError("merge_counters shape mismatch")
    if seq_lens.size(0) != b:
        raise RuntimeError("seq_lens batch mismatch")
    if q_indices.size(0) != b:
        raise RuntimeError("q_indices batch mismatch")
    return hkv, physical_pages, b


def paged_attention_workqueue(q_source, k_pages, v_pages, block_table, seq_lens, work_items,
                              split_offsets, merge_counters, q_indices, out_indices, output,
                              workspace, bucket_context: int, page_size: int,
                              total_partial_slots: int, fused_merge: bool) -> None:
    """Reference ``persistentkv_paged_attention_workqueue`` (extension :230-317)."""
    hkv, physical_pages, b = _check_workqueue(q_source, k_pages, v_pages, block_table, seq_lens,
                                              work_items, split_offsets, merge_counters,
                                              q_indices, page_size)
    _check_tensor(out_indices, "out_indices", torch.int32, 1)
    _check_tensor(output, "output", q_source.dtype, 3)
    ws_ptr, ws_bytes = _workspace(workspace)
    hq, d = q_source.size(1), q_source.size(2)
    if not (output.size(1) == hq and output.size(2) == d):
        raise RuntimeError("output shape must match q head dimensions")
    if out_indices.size(0) != b:
        raise RuntimeError("out_indices batch mismatch")
    _check_supported_gqa(hq, hkv)
    _positive(bucket_context, "bucket_context")
    _positive(page_size, "page_size")
    if work_items.size(0) <= 0:
        raise RuntimeError("work_items must not be empty")
    if total_partial_slots <= 0:
        raise RuntimeError("total_partial_slots must be positive")
    lib = _native.load()
    _native.check(lib.pkv_paged_attention_workqueue(
        q_source.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), block_table.data_ptr(),
        seq_lens.data_ptr(), work_items.data_ptr(), split_offsets.data_ptr(),
        merge_counters.data_ptr(), q_indices.data_ptr(), out_indices.data_ptr(),
        output.data_ptr(), ws_ptr, ws_bytes, b, q_source.size(0), output.size(0), hq, hkv, d,
        physical_pages, page_size, block_table.size(1), int(bucket_context),
        work_items.size(0), int(total_partial_slots), 1 if fused_merge else 0,
        _DTYPES[q_source.dtype], _stream()))


def paged_attention_workqueue_state(q_source, k_pages, v_pages, block_table, seq_lens,
                                    work_items, split_offsets, merge_counters, q_indices,
                                    state_out, workspace, page_size: int,
                                    total_partial_slots: int, fused_merge: bool) -> None:
    """Work-queue decode that writes each row's combined (m, l, acc) state.

    ``state_out`` is float32 ``[B, Hq, 130]``; no counterpart in the reference.
    """
    hkv, physical_pages, b = _check_workqueue(q_source, k_pages, v_pages, block_table, seq_lens,
                                              work_items, split_offsets, merge_counters,
                                              q_indices, page_size)
    _check_tensor(state_out, "state_out", torch.float32, 3)
    hq, d = q_source.size(1), q_source.size(2)
    if tuple(state_out.shape) != (b, hq, STATE_STRIDE):
        raise RuntimeError("state_out must have shape [B, Hq, 130]")
    _check_supported_gqa(hq, hkv)
    ws_ptr, ws_bytes = _workspace(workspace)
    lib = _native.load()
    _native.check(lib.pkv_paged_attention_workqueue_state(
        q_source.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), block_table.data_ptr(),
        seq_lens.data_ptr(), work_items.data_ptr(), split_offsets.data_ptr(),
        merge_counters.data_ptr() if fused_merge else None, q_indices.data_ptr(),
        state_out.data_ptr(), ws_ptr, ws_bytes, b, q_source.size(0), hq, hkv, d,
        physical_pages, page_size, block_table.size(1), work_items.size(0),
        int(total_partial_slots), _DTYPES[q_source.dtype], _stream()))


def paged_attention_auto(q_source, k_pages, v_pages, block_table, seq_lens, output, workspace,
                         q_indices=None, out_indices=None, merge_counters=None,
                         plan=None, groups: int = 0) -> None:
    """Paged decode with the device-side schedule (no work queue, no host builder).

    Row b attends to ``seq_lens[b]`` tokens of ``block_table[b]``, reads
    ``q_source[q_indices[b]]`` and writes ``output[out_indices[b]]`` (identity
    when an index tensor is None).  ``merge_counters`` (zeroed int32
    ``[B, Hkv]``) selects the fused merge.  ``workspace`` needs
    ``auto_workspace_bytes(B, Hq, Hkv)`` bytes.  ``plan`` (optional) is a
    device int32 copy of ``scheduler.build_auto_plan`` for exactly this step's
    metadata: the kernel then starts from it instead of deriving the schedule;
    ``groups`` is the group count the plan was built for (0: the maximum).
    No counterpart in the reference.
    """
    _check_tensor(q_source, "q_source", tuple(_DTYPES), 3)
    hkv, physical_pages = _check_kv(q_source, k_pages, v_pages, k_pages.size(2))
    _check_tensor(block_table, "block_table", torch.int32, 2)
    _check_tensor(seq_lens, "seq_lens", torch.int32, 1)
    _check_tensor(output, "output", q_source.dtype, 3)
    b = block_table.size(0)
    hq, d = q_source.size(1), q_source.size(2)
    if seq_lens.size(0) != b:
        raise RuntimeError("seq_lens batch mismatch")
    if not (output.size(1) == hq and output.size(2) == d):
        raise RuntimeError("output shape must match q head dimensions")
    ptrs = []
    for name, t in (("q_indices", q_indices), ("out_indices", out_indices)):
        if t is None:
            ptrs.append(None)
        else:
            _check_tensor(t, name, torch.int32, 1)
            if t.size(0) != b:
                raise RuntimeError(f"{name} batch mismatch")
            ptrs.append(t.data_ptr())
    ctr = None
    if merge_counters is not None:
        _check_tensor(merge_counters, "merge_counters", torch.int32, 2)
        if not (merge_counters.size(0) == b and merge_counters.size(1) == hkv):
            raise RuntimeError("merge_counters shape mismatch")
        ctr = merge_counters.data_ptr()
    _check_supported_gqa(hq, hkv)
    ws_ptr, ws_bytes = _workspace(workspace)
    lib = _native.load()
    if plan is not None:
        _check_tensor(plan, "plan", torch.int32, 1)
        _native.check(lib.pkv_paged_attention_auto_planned(
            q_source.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), block_table.data_ptr(),
            seq_lens.data_ptr(), ptrs[0], ptrs[1], output.data_ptr(), ws_ptr, ws_bytes, ctr,
            plan.data_ptr(), plan.numel() * 4, int(groups), b, q_source.size(0), output.size(0),
            hq, hkv, d,
            physical_pages,
            k_pages.size(2), block_table.size(1), _DTYPES[q_source.dtype], _stream()))
        return
    _native.check(lib.pkv_paged_attention_auto(
        q_source.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), block_table.data_ptr(),
        seq_lens.data_ptr(), ptrs[0], ptrs[1], output.data_ptr(), ws_ptr, ws_bytes, ctr, b,
        q_source.size(0), output.size(0), hq, hkv, d, physical_pages, k_pages.size(2),
        block_table.size(1), _DTYPES[q_source.dtype], _stream()))


def paged_attention_auto_state(q_source, k_pages, v_pages, block_table, seq_lens, state_out,
                               workspace, q_indices=None, merge_counters=None) -> None:
    """``paged_attention_auto`` writing each row's (m, l, acc) state to the float32
    ``state_out[B, Hq, 130]`` (one GPU's part of a sequence-sharded decode)."""
    _check_tensor(q_source, "q_source", tuple(_DTYPES), 3)
    hkv, physical_pages = _check_kv(q_source, k_pages, v_pages, k_pages.size(2))
    _check_tensor(block_table, "block_table", torch.int32, 2)
    _check_tensor(seq_lens, "seq_lens", torch.int32, 1)
    _check_tensor(state_out, "state_out", torch.float32, 3)
    b = block_table.size(0)
    hq, d = q_source.size(1), q_source.size(2)
    if tuple(state_out.shape) != (b, hq, STATE_STRIDE):
        raise RuntimeError("state_out must have shape [B, Hq, 130]")
    qi = None
    if q_indices is not None:
        _check_tensor(q_indices, "q_indices", torch.int32, 1)
        qi = q_indices.data_ptr()
    ctr = None
    if merge_counters is not None:
        _check_tensor(merge_counters, "merge_counters", torch.int32, 2)
        ctr = merge_counters.data_ptr()
    _check_supported_gqa(hq, hkv)
    ws_ptr, ws_bytes = _workspace(workspace)
    _native.check(_native.load().pkv_paged_attention_auto_state(
        q_source.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), block_table.data_ptr(),
        seq_lens.data_ptr(), qi, state_out.data_ptr(), ws_ptr, ws_bytes, ctr, b,
        q_source.size(0), hq, hkv, d, physical_pages, k_pages.size(2), block_table.size(1),
        _DTYPES[q_source.dtype], _stream()))


class Exchange:
    """This rank's end of the fused sharded-decode exchange (``pkv_exchange``).

    Create one per rank on its own device, gather every rank's ``handle`` (in
    rank order) and pass them to :meth:`connect`; ``world == 1`` needs no
    connect.  ``close`` synchronises the device and frees the buffer: call it
    only after every rank has synchronised its device (a barrier), since a
    peer's kernel stores into this rank's buffer.
    """

    def __init__(self, world: int, rank: int, max_batch: int, hq: int, hkv: int):
        import ctypes

        lib = _native.load()
        self._ptr = ctypes.c_void_p()
        buf = ctypes.create_string_buffer(_native.EXCHANGE_HANDLE_BYTES)
        _native.check(lib.pkv_exchange_create(world, rank, max_batch, hq, hkv,
                                              ctypes.byref(self._ptr), buf))
        self.handle = bytes(buf.raw)
        self.world, self.rank, self.max_batch, self.hq, self.hkv = world, rank, max_batch, hq, hkv
        self.device = torch.cuda.current_device()

    def connect(self, handles) -> None:
        """``handles``: every rank's ``handle`` bytes, in rank order."""
        if len(handles) != self.world:
            raise RuntimeError("one handle per rank is required")
        blob = b"".join(bytes(h) for h in handles)
        _native.check(_native.load().pkv_exchange_connect(self._ptr, blob))

    @property
    def ptr(self):
        if not self._ptr:
            raise RuntimeError("exchange is closed")
        return self._ptr

    def close(self) -> None:
        if self._ptr:
            _native.check(_native.load().pkv_exchange_destroy(self._ptr))
            self._ptr = type(self._ptr)()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


def exchange_bytes(world: int, max_batch: int, hq: int, hkv: int) -> int:
    return int(_native.load().pkv_exchange_bytes(world, max_batch, hq, hkv))


def paged_attention_sharded(q_source, k_pages, v_pages, block_table, seq_lens, output, workspace,
                            merge_counters, exchange: Exchange, q_indices=None,
                            out_indices=None, plan=None, groups: int = 0) -> None:
    """One step of sequence-sharded decode with the state exchange fused into
    the kernel: ``block_table`` / ``seq_lens`` hold this rank's page range of
    every row; every rank gets the merged ``output``.  All ranks must call it
    with the same batch, in the same order.  ``plan``: a device int32 copy of
    this rank's host plan (``scheduler.build_auto_plan`` over the same rows,
    indices and ``groups``).  No counterpart in the reference."""
    _check_tensor(q_source, "q_source", tuple(_DTYPES), 3)
    hkv, physical_pages = _check_kv(q_source, k_pages, v_pages, k_pages.size(2))
    _check_tensor(block_table, "block_table", torch.int32, 2)
    _check_tensor(seq_lens, "seq_lens", torch.int32, 1)
    _check_tensor(output, "output", q_source.dtype, 3)
    _check_tensor(merge_counters, "merge_counters", torch.int32, 2)
    b = block_table.size(0)
    hq, d = q_source.size(1), q_source.size(2)
    if seq_lens.size(0) != b:
        raise RuntimeError("seq_lens batch mismatch")
    if not (output.size(1) == hq and output.size(2) == d):
        raise RuntimeError("output shape must match q head dimensions")
    if not (merge_counters.size(0) == b and merge_counters.size(1) == hkv):
        raise RuntimeError("merge_counters shape mismatch")
    ptrs = []
    for name, t in (("q_indices", q_indices), ("out_indices", out_indices)):
        if t is None:
            ptrs.append(None)
        else:
            _check_tensor(t, name, torch.int32, 1)
            if t.size(0) != b:
                raise RuntimeError(f"{name} batch mismatch")
            ptrs.append(t.data_ptr())
    _check_supported_gqa(hq, hkv)
    ws_ptr, ws_bytes = _workspace(workspace)
    if plan is not None:
        _check_tensor(plan, "plan", torch.int32, 1)
        _native.check(_native.load().pkv_paged_attention_sharded_planned(
            q_source.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), block_table.data_ptr(),
            seq_lens.data_ptr(), ptrs[0], ptrs[1], output.data_ptr(), ws_ptr, ws_bytes,
            merge_counters.data_ptr(), exchange.ptr, plan.data_ptr(), plan.numel() * 4,
            int(groups), b, q_source.size(0), output.size(0), hq, hkv, d, physical_pages,
            k_pages.size(2), block_table.size(1), _DTYPES[q_source.dtype], _stream()))
        return
    _native.check(_native.load().pkv_paged_attention_sharded(
        q_source.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), block_table.data_ptr(),
        seq_lens.data_ptr(), ptrs[0], ptrs[1], output.data_ptr(), ws_ptr, ws_bytes,
        merge_counters.data_ptr(), exchange.ptr, b, q_source.size(0), output.size(0), hq, hkv, d,
        physical_pages, k_pages.size(2), block_table.size(1), _DTYPES[q_source.dtype],
        _stream()))


def paged_attention_auto_fp8(q_source, k_pages, v_pages, k_scale: float, v_scale: float,
                             block_table, seq_lens, output, workspace, q_indices=None,
                             out_indices=None, merge_counters=None) -> None:
    """``paged_attention_auto`` over an e4m3 (``torch.float8_e4m3fn``) K/V cache
    with per-tensor scales (K = k_scale * k_pages, V = v_scale * v_pages); q and
    output are fp16.  No counterpart in the reference."""
    _check_tensor(q_source, "q_source", torch.float16, 3)
    _check_tensor(k_pages, "k_pages", torch.float8_e4m3fn, 4)
    _check_tensor(v_pages, "v_pages", torch.float8_e4m3fn, 4)
    _check_tensor(block_table, "block_table", torch.int32, 2)
    _check_tensor(seq_lens, "seq_lens", torch.int32, 1)
    _check_tensor(output, "output", torch.float16, 3)
    if tuple(v_pages.shape) != tuple(k_pages.shape) or k_pages.size(3) != HEAD_DIM:
        raise RuntimeError("k_pages / v_pages shape mismatch")
    hkv, physical_pages, page_size = k_pages.size(1), k_pages.size(0), k_pages.size(2)
    b = block_table.size(0)
    hq, d = q_source.size(1), q_source.size(2)
    if d != HEAD_DIM:
        raise RuntimeError("PersistentKV extension currently requires d=128")
    if seq_lens.size(0) != b:
        raise RuntimeError("seq_lens batch mismatch")
    if not (output.size(1) == hq and output.size(2) == d):
        raise RuntimeError("output shape must match q head dimensions")
    ptrs = []
    for name, t in (("q_indices", q_indices), ("out_indices", out_indices)):
        if t is None:
            ptrs.append(None)
        else:
            _check_tensor(t, name, torch.int32, 1)
            if t.size(0) != b:
                raise RuntimeError(f"{name} batch mismatch")
            ptrs.append(t.data_ptr())
    ctr = None
    if merge_counters is not None:
        _check_tensor(merge_counters, "merge_counters", torch.int32, 2)
        if not (merge_counters.size(0) == b and merge_counters.size(1) == hkv):
            raise RuntimeError("merge_counters shape mismatch")
        ctr = merge_counters.data_ptr()
    _check_supported_gqa(hq, hkv)
    ws_ptr, ws_bytes = _workspace(workspace)
    _native.check(_native.load().pkv_paged_attention_auto_fp8(
        q_source.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), float(k_scale),
        float(v_scale), block_table.data_ptr(), seq_lens.data_ptr(), ptrs[0], ptrs[1],
        output.data_ptr(), ws_ptr, ws_bytes, ctr, b, q_source.size(0), output.size(0), hq, hkv,
        d, physical_pages, page_size, block_table.size(1), _stream()))


def kv_append(k_new, v_new, k_pages, v_pages, block_table, positions, free_pages=None,
              free_count=None, counters=None) -> None:
    """Writes one new token per row into the paged pools (``pkv_kv_append``).

    ``k_new`` / ``v_new`` [B, Hkv, 128] (the pools' dtype) land at token
    ``positions[b]`` of row b.  With ``free_pages`` (int32 stack), ``free_count``
    (int32 [1]) and zeroed ``counters`` (int32 [1]), rows whose token opens a
    page take pages from the top of the stack in row order and record them in
    ``block_table``.  No counterpart in the reference."""
    dt = k_pages.dtype
    _check_tensor(k_new, "k_new", dt, 3)
    _check_tensor(v_new, "v_new", dt, 3)
    _check_tensor(k_pages, "k_pages", tuple(_DTYPES), 4)
    _check_tensor(v_pages, "v_pages", dt, 4)
    _check_tensor(block_table, "block_table", torch.int32, 2)
    _check_tensor(positions, "positions", torch.int32, 1)
    b, hkv, d = k_new.shape
    if tuple(v_new.shape) != (b, hkv, d) or k_pages.size(1) != hkv or d != HEAD_DIM:
        raise RuntimeError("k_new / v_new shape must be [B, Hkv, 128] matching the pools")
    if tuple(v_pages.shape) != tuple(k_pages.shape):
        raise RuntimeError("v_pages shape mismatch")
    if block_table.size(0) != b or positions.size(0) != b:
        raise RuntimeError("block_table / positions batch mismatch")
    fp = fc = ctr = None
    if free_pages is not None:
        _check_tensor(free_pages, "free_pages", torch.int32, 1)
        if free_count is None or counters is None:
            raise RuntimeError("a free-page list needs free_count and counters")
        _check_tensor(free_count, "free_count", torch.int32, 1)
        _check_tensor(counters, "counters", torch.int32, 1)
        if free_pages.numel() == 0:
            # no address, which would mean that there is no stack: one of no pages
            free_pages = free_count = torch.zeros_like(free_count)
        fp, fc, ctr = free_pages.data_ptr(), free_count.data_ptr(), counters.data_ptr()
    _native.check(_native.load().pkv_kv_append(
        k_new.data_ptr(), v_new.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(),
        block_table.data_ptr(), positions.data_ptr(), fp, fc, ctr, b, hkv, d, k_pages.size(0),
        k_pages.size(2), block_table.size(1), _DTYPES[dt], _stream()))


# The calls below are a few microseconds of GPU work at their smallest, so their
# checks are two: one expression over everything a call needs, and, where it
# fails, the checks that say what is wrong.


def _check_current_device(*tensors) -> None:
    """Kernels launch on the current device: every operand must live there."""
    device = torch.cuda.current_device()
    for t in tensors:
        if t is not None and t.get_device() != device:
            raise RuntimeError(f"operands must be on the current device, cuda:{device}")


def _stream_of(device: int) -> int:
    """Raw stream of ``device``, which is the current one."""
    if _raw_stream is not None:
        return _raw_stream(device)
    return torch.cuda.current_stream().cuda_stream


def _check_packed(t, name: str, dtype) -> None:
    """A packed operand [tokens, heads, 128]: contiguous heads of 128, any
    token and head strides (a slice of a fused projection's output is fine)."""
    if not t.is_cuda:
        raise RuntimeError(f"{name} must be a CUDA tensor")
    if (t.dtype not in dtype) if isinstance(dtype, tuple) else t.dtype != dtype:
        raise RuntimeError(f"{name} has wrong dtype")
    if t.dim() != 3:
        raise RuntimeError(f"{name} has wrong rank")
    if t.size(2) != HEAD_DIM:
        raise RuntimeError("PersistentKV extension currently requires d=128")
    if t.stride(2) != 1:
        raise RuntimeError(f"{name} must be contiguous in its last dimension")


def _check_block_scales(k_pages, k_scales, v_scales) -> int:
    """Scales [P, Hkv, page / block] of e4m3 pools; returns the block's tokens."""
    _check_tensor(k_scales, "k_scales", torch.float32, 3)
    _check_tensor(v_scales, "v_scales", torch.float32, 3)
    pages, hkv, page_size, _ = k_pages.shape
    blocks = k_scales.size(2)
    if k_scales.shape != v_scales.shape or k_scales.size(0) != pages or k_scales.size(1) != hkv:
        raise RuntimeError("k_scales / v_scales shape must be [P, Hkv, page_size / block]")
    if blocks == 0 or page_size % blocks != 0 or (page_size // blocks) % 16 != 0:
        raise RuntimeError("a scale block must be a multiple of 16 tokens that divides the page")
    return page_size // blocks


def _check_block_decode(q_source, k_pages, v_pages, k_scales, v_scales, block_table, seq_lens,
                        output, workspace, q_indices, out_indices, merge_counters) -> None:
    _check_tensor(q_source, "q_source", tuple(_DTYPES), 3)
    _check_tensor(k_pages, "k_pages", torch.float8_e4m3fn, 4)
    _check_tensor(v_pages, "v_pages", torch.float8_e4m3fn, 4)
    _check_tensor(block_table, "block_table", torch.int32, 2)
    _check_tensor(seq_lens, "seq_lens", torch.int32, 1)
    _check_tensor(output, "output", q_source.dtype, 3)
    if v_pages.shape != k_pages.shape or k_pages.size(3) != HEAD_DIM:
        raise RuntimeError("k_pages / v_pages shape mismatch")
    hkv = k_pages.size(1)
    _check_block_scales(k_pages, k_scales, v_scales)
    b = block_table.size(0)
    q_rows, hq, d = q_source.shape
    if d != HEAD_DIM:
        raise RuntimeError("PersistentKV extension currently requires d=128")
    if seq_lens.size(0) != b:
        raise RuntimeError("seq_lens batch mismatch")
    if output.size(1) != hq or output.size(2) != d:
        raise RuntimeError("output shape must match q head dimensions")
    for name, t in (("q_indices", q_indices), ("out_indices", out_indices)):
        if t is not None:
            _check_tensor(t, name, torch.int32, 1)
            if t.size(0) != b:
                raise RuntimeError(f"{name} batch mismatch")
    # without an index tensor row b reads q_source[b] and writes output[b]
    if (q_indices is None and q_rows < b) or (out_indices is None and output.size(0) < b):
        raise RuntimeError("q_source and output need a row per block_table row")
    if merge_counters is not None:
        _check_tensor(merge_counters, "merge_counters", torch.int32, 2)
        if merge_counters.size(0) != b or merge_counters.size(1) != hkv:
            raise RuntimeError("merge_counters shape mismatch")
    _check_supported_gqa(hq, hkv)
    _workspace(workspace)
    _check_current_device(q_source, k_pages, v_pages, k_scales, v_scales, block_table, seq_lens,
                          output, workspace, q_indices, out_indices, merge_counters)


def paged_attention_auto_fp8_block(q_source, k_pages, v_pages, k_scales, v_scales, block_table,
                                   seq_lens, output, workspace, q_indices=None, out_indices=None,
                                   merge_counters=None) -> None:
    """``paged_attention_auto`` over an e4m3 (``torch.float8_e4m3fn``) K/V cache
    with one float32 scale per block of tokens and head: ``k_scales`` /
    ``v_scales`` [P, Hkv, page_size / block], block a multiple of 16 tokens.  q
    and output are fp16 or bf16.  Half the cache's bytes, read at the same
    rate.  No counterpart in the reference."""
    dt, pool, scale, table = q_source.dtype, k_pages.shape, k_scales.shape, block_table.shape
    qs, outs, dev = q_source.shape, output.shape, q_source.get_device()
    i32, f8 = torch.int32, torch.float8_e4m3fn
    if not (
        dev >= 0 and dt in _DTYPES and output.dtype is dt and k_pages.dtype is f8
        and v_pages.dtype is f8 and k_scales.dtype is torch.float32
        and v_scales.dtype is torch.float32 and block_table.dtype is i32 and seq_lens.dtype is i32
        and len(qs) == 3 and len(outs) == 3 and len(pool) == 4 and len(scale) == 3
        and len(table) == 2 and seq_lens.shape == table[:1] and qs[1:] == outs[1:]
        and qs[2] == HEAD_DIM and pool[3] == HEAD_DIM and v_pages.shape == pool
        and v_scales.shape == scale and scale[:2] == pool[:2] and scale[2] > 0
        and pool[2] % (16 * scale[2]) == 0 and pool[1] > 0 and qs[1] % pool[1] == 0
        and qs[1] // pool[1] in _SUPPORTED_G
        and q_indices is None and out_indices is None and qs[0] >= table[0] and outs[0] >= table[0]
        and q_source.is_contiguous() and output.is_contiguous() and k_pages.is_contiguous()
        and v_pages.is_contiguous() and k_scales.is_contiguous() and v_scales.is_contiguous()
        and block_table.is_contiguous() and seq_lens.is_contiguous()
        and workspace.is_contiguous() and k_pages.get_device() == dev
        and v_pages.get_device() == dev and k_scales.get_device() == dev
        and v_scales.get_device() == dev and block_table.get_device() == dev
        and seq_lens.get_device() == dev and output.get_device() == dev
        and workspace.get_device() == dev and torch.cuda.current_device() == dev
        and (merge_counters is None or (
            merge_counters.dtype is i32 and merge_counters.shape == (table[0], pool[1])
            and merge_counters.is_contiguous() and merge_counters.get_device() == dev))
    ):
        _check_block_decode(q_source, k_pages, v_pages, k_scales, v_scales, block_table, seq_lens,
                            output, workspace, q_indices, out_indices, merge_counters)
    ws_bytes = workspace.numel() * workspace.element_size()
    _native.check(_native.load().pkv_paged_attention_auto_fp8_block(
        q_source.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), k_scales.data_ptr(),
        v_scales.data_ptr(), block_table.data_ptr(), seq_lens.data_ptr(),
        None if q_indices is None else q_indices.data_ptr(),
        None if out_indices is None else out_indices.data_ptr(), output.data_ptr(),
        workspace.data_ptr() if ws_bytes else None, ws_bytes,
        None if merge_counters is None else merge_counters.data_ptr(), table[0], qs[0], outs[0],
        qs[1], pool[1], HEAD_DIM, pool[0], pool[2], table[1], pool[2] // scale[2], _DTYPES[dt],
        _stream_of(dev)))


def _check_prompt_slots(cached_lens, new_lens, block_table, slots, cu_seqlens, seq_lens,
                        free_pages, free_count, free_left, counters, page_size) -> None:
    _check_tensor(cached_lens, "cached_lens", torch.int32, 1)
    _check_tensor(new_lens, "new_lens", torch.int32, 1)
    _check_tensor(block_table, "block_table", torch.int32, 2)
    _check_tensor(slots, "slots", torch.int32, 1)
    _check_tensor(cu_seqlens, "cu_seqlens", torch.int32, 1)
    _check_tensor(seq_lens, "seq_lens", torch.int32, 1)
    b = block_table.size(0)
    if cached_lens.size(0) != b or new_lens.size(0) != b or seq_lens.size(0) != b:
        raise RuntimeError("cached_lens / new_lens / seq_lens batch mismatch")
    if cu_seqlens.size(0) != b + 1:
        raise RuntimeError("cu_seqlens must hold B + 1 values")
    _positive(page_size, "page_size")
    if free_pages is not None:
        _check_tensor(free_pages, "free_pages", torch.int32, 1)
        if free_count is None or free_left is None or counters is None:
            raise RuntimeError("a free-page list needs free_count, free_left and counters")
        for name, t in (("free_count", free_count), ("free_left", free_left),
                        ("counters", counters)):
            _check_tensor(t, name, torch.int32, 1)
            if t.size(0) < 1:
                raise RuntimeError(f"{name} must hold one value")
    _check_current_device(cached_lens, new_lens, block_table, slots, cu_seqlens, seq_lens,
                          free_pages, free_count, free_left, counters)


def prompt_slots(cached_lens, new_lens, block_table, slots, cu_seqlens, seq_lens, free_pages,
                 free_count, free_left, counters, page_size: int) -> None:
    """Block tables and slot map of a batch, on the GPU, from its lengths.

    Row b holds ``cached_lens[b]`` tokens and gets ``new_lens[b]`` more (int32
    [B]).  The rows, in order, take the pages they open from the top of the
    ``free_pages`` stack (``free_count`` int32 [1] entries) into ``block_table``.
    Written: ``slots`` (page * page_size + offset of every new token, packed; -1
    for rows not served and behind the last token), ``cu_seqlens`` [B + 1],
    ``seq_lens`` [B] (the lengths after the call) and ``free_left`` [1] (may be
    ``free_count``).  ``counters``: one zeroed int32, left zero.  With
    ``free_pages`` None every page is in ``block_table`` already (an empty
    ``free_pages`` is a stack without pages).  See
    ``pkv_prompt_slots`` for the rows that are not served.  No counterpart in
    the reference."""
    i32, dev, table, n = torch.int32, cached_lens.get_device(), block_table.shape, slots.shape
    rows = cached_lens.shape
    if not (
        dev >= 0 and cached_lens.dtype is i32 and new_lens.dtype is i32
        and block_table.dtype is i32 and slots.dtype is i32 and cu_seqlens.dtype is i32
        and seq_lens.dtype is i32 and len(rows) == 1 and len(table) == 2 and len(n) == 1
        and table[0] == rows[0] and new_lens.shape == rows and seq_lens.shape == rows
        and cu_seqlens.shape == (rows[0] + 1,) and page_size > 0
        and cached_lens.is_contiguous() and new_lens.is_contiguous()
        and block_table.is_contiguous() and slots.is_contiguous() and cu_seqlens.is_contiguous()
        and seq_lens.is_contiguous() and new_lens.get_device() == dev
        and block_table.get_device() == dev and slots.get_device() == dev
        and cu_seqlens.get_device() == dev and seq_lens.get_device() == dev
        and torch.cuda.current_device() == dev
        and (free_pages is None or (
            free_count is not None and free_left is not None and counters is not None
            and free_pages.dtype is i32 and free_count.dtype is i32 and free_left.dtype is i32
            and counters.dtype is i32 and free_pages.dim() == 1 and free_count.shape == (1,)
            and free_left.shape == (1,) and counters.shape == (1,) and free_pages.is_contiguous()
            and free_pages.get_device() == dev and free_count.get_device() == dev
            and free_left.get_device() == dev and counters.get_device() == dev))
    ):
        _check_prompt_slots(cached_lens, new_lens, block_table, slots, cu_seqlens, seq_lens,
                            free_pages, free_count, free_left, counters, page_size)
    fp = fc = fl = ctr = None
    capacity = 0
    if free_pages is not None:
        # (an empty tensor has no address, and none would mean that there is no stack)
        fc = free_count.data_ptr()
        fp = free_pages.data_ptr() or fc
        fl, ctr = free_left.data_ptr(), counters.data_ptr()
        capacity = free_pages.numel()
    _native.check(_native.load().pkv_prompt_slots(
        cached_lens.data_ptr(), new_lens.data_ptr(), block_table.data_ptr(), slots.data_ptr(),
        cu_seqlens.data_ptr(), seq_lens.data_ptr(), fp, fc, fl, ctr, table[0], table[1],
        int(page_size), n[0], capacity, _stream_of(dev)))


def _check_write(k, v, k_pages, v_pages, slots, pool_dtype) -> None:
    _check_packed(k, "k", tuple(_DTYPES))
    _check_packed(v, "v", k.dtype)
    _check_tensor(k_pages, "k_pages", pool_dtype, 4)
    _check_tensor(v_pages, "v_pages", pool_dtype, 4)
    _check_tensor(slots, "slots", torch.int32, 1)
    if v.shape != k.shape or k_pages.size(1) != k.size(1) or k_pages.size(3) != HEAD_DIM:
        raise RuntimeError("k / v shape must be [T, Hkv, 128] matching the pools")
    if v_pages.shape != k_pages.shape:
        raise RuntimeError("v_pages shape mismatch")
    if slots.size(0) != k.size(0):
        raise RuntimeError("slots must hold one value per token")


def kv_write(k, v, k_pages, v_pages, slots) -> None:
    """Writes packed tokens ``k`` / ``v`` [T, Hkv, 128] into 16-bit pools of their
    dtype at ``slots`` [T] (page * page_size + offset; negative skips a token).
    No counterpart in the reference."""
    dt, ks, pool, dev = k.dtype, k.shape, k_pages.shape, k.get_device()
    kst, vst = k.stride(), v.stride()
    if not (
        dev >= 0 and dt in _DTYPES and v.dtype is dt and k_pages.dtype is dt
        and v_pages.dtype is dt and slots.dtype is torch.int32 and len(ks) == 3 and len(pool) == 4
        and v.shape == ks and v_pages.shape == pool and slots.shape == ks[:1]
        and pool[1] == ks[1] and ks[2] == HEAD_DIM and pool[3] == HEAD_DIM and kst[2] == 1
        and vst[2] == 1 and k_pages.is_contiguous() and v_pages.is_contiguous()
        and slots.is_contiguous() and v.get_device() == dev and k_pages.get_device() == dev
        and v_pages.get_device() == dev and slots.get_device() == dev
        and torch.cuda.current_device() == dev
    ):
        _check_write(k, v, k_pages, v_pages, slots, dt)
        _check_current_device(k, v, k_pages, v_pages, slots)
    _native.check(_native.load().pkv_kv_write(
        k.data_ptr(), v.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), slots.data_ptr(),
        ks[0], ks[1], HEAD_DIM, kst[0], kst[1], vst[0], vst[1], pool[0], pool[2], _DTYPES[dt],
        _stream_of(dev)))


def kv_write_fp8_block(k, v, k_pages, v_pages, k_scales, v_scales, slots) -> None:
    """``kv_write`` into e4m3 pools with one scale per block of tokens and head
    (``paged_attention_auto_fp8_block``'s cache): each block that the call
    touches gets the least power of two that holds its new tokens, and its
    earlier tokens if the call starts inside it.  The tokens of one block must
    be consecutive and in slot order.  No counterpart in the reference."""
    dt, ks, pool, dev = k.dtype, k.shape, k_pages.shape, k.get_device()
    kst, vst, scale, f8 = k.stride(), v.stride(), k_scales.shape, torch.float8_e4m3fn
    if not (
        dev >= 0 and dt in _DTYPES and v.dtype is dt and k_pages.dtype is f8
        and v_pages.dtype is f8 and slots.dtype is torch.int32 and len(ks) == 3 and len(pool) == 4
        and k_scales.dtype is torch.float32 and v_scales.dtype is torch.float32
        and len(scale) == 3 and v_scales.shape == scale and scale[:2] == pool[:2] and scale[2] > 0
        and pool[2] % (16 * scale[2]) == 0
        and v.shape == ks and v_pages.shape == pool and slots.shape == ks[:1]
        and pool[1] == ks[1] and ks[2] == HEAD_DIM and pool[3] == HEAD_DIM and kst[2] == 1
        and vst[2] == 1 and k_pages.is_contiguous() and v_pages.is_contiguous()
        and k_scales.is_contiguous() and v_scales.is_contiguous() and slots.is_contiguous()
        and v.get_device() == dev and k_pages.get_device() == dev and v_pages.get_device() == dev
        and k_scales.get_device() == dev and v_scales.get_device() == dev
        and slots.get_device() == dev and torch.cuda.current_device() == dev
    ):
        _check_write(k, v, k_pages, v_pages, slots, f8)
        _check_block_scales(k_pages, k_scales, v_scales)
        _check_current_device(k, v, k_pages, v_pages, k_scales, v_scales, slots)
    _native.check(_native.load().pkv_kv_write_fp8_block(
        k.data_ptr(), v.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), k_scales.data_ptr(),
        v_scales.data_ptr(), slots.data_ptr(), ks[0], ks[1], HEAD_DIM, kst[0], kst[1], vst[0],
        vst[1], pool[0], pool[2], pool[2] // scale[2], _DTYPES[dt], _stream_of(dev)))


def _check_prompt(q, k, v, cu_seqlens_q, cu_seqlens_k, output, lse) -> None:
    _check_packed(q, "q", tuple(_DTYPES))
    _check_packed(k, "k", q.dtype)
    _check_packed(v, "v", q.dtype)
    _check_tensor(cu_seqlens_q, "cu_seqlens_q", torch.int32, 1)
    _check_tensor(output, "output", q.dtype, 3)
    if v.shape != k.shape:
        raise RuntimeError("v shape must match k")
    if output.shape != q.shape:
        raise RuntimeError("output shape must match q")
    if cu_seqlens_q.size(0) < 1:
        raise RuntimeError("cu_seqlens_q must hold B + 1 values")
    if cu_seqlens_k is not None:
        _check_tensor(cu_seqlens_k, "cu_seqlens_k", torch.int32, 1)
        if cu_seqlens_k.size(0) != cu_seqlens_q.size(0):
            raise RuntimeError("cu_seqlens_k batch mismatch")
    if lse is not None:
        _check_tensor(lse, "lse", torch.float32, 2)
        if lse.size(0) != q.size(0) or lse.size(1) != q.size(1):
            raise RuntimeError("lse must have shape [Tq, Hq]")
    _check_supported_gqa(q.size(1), k.size(1))
    _check_current_device(q, k, v, cu_seqlens_q, cu_seqlens_k, output, lse)


def prompt_attention(q, k, v, cu_seqlens_q, cu_seqlens_k, output, lse=None) -> None:
    """Causal attention of packed sequences with grouped heads.

    ``q`` [Tq, Hq, 128], ``k`` / ``v`` [Tk, Hkv, 128] (fp16 or bf16, any token
    and head strides that are multiples of 8); sequence b has the rows
    ``cu_seqlens_q[b]`` to ``cu_seqlens_q[b + 1]`` of q and the keys
    ``cu_seqlens_k[b]`` to ``cu_seqlens_k[b + 1]`` (None: the same), and its
    last row sees its last key.  ``output`` [Tq, Hq, 128] contiguous; ``lse``
    (optional, float32 [Tq, Hq]) gets each row's log-sum-exp.  A row that sees
    no key gives zeros and -inf; rows of no sequence are left as they were.  No
    counterpart in the reference."""
    dt, qs, ks, dev, cq = q.dtype, q.shape, k.shape, q.get_device(), cu_seqlens_q.shape
    qst, kst, vst = q.stride(), k.stride(), v.stride()
    if not (
        dev >= 0 and dt in _DTYPES and k.dtype is dt and v.dtype is dt and output.dtype is dt
        and cu_seqlens_q.dtype is torch.int32 and len(qs) == 3 and len(ks) == 3 and len(cq) == 1
        and cq[0] > 0 and v.shape == ks and output.shape == qs and qs[2] == HEAD_DIM
        and ks[2] == HEAD_DIM and ks[1] > 0 and qs[1] % ks[1] == 0
        and qs[1] // ks[1] in _SUPPORTED_G and qst[2] == 1 and kst[2] == 1 and vst[2] == 1
        and output.is_contiguous() and cu_seqlens_q.is_contiguous() and k.get_device() == dev
        and v.get_device() == dev and output.get_device() == dev
        and cu_seqlens_q.get_device() == dev and torch.cuda.current_device() == dev
        and (cu_seqlens_k is None or (
            cu_seqlens_k.dtype is torch.int32 and cu_seqlens_k.shape == cq
            and cu_seqlens_k.is_contiguous() and cu_seqlens_k.get_device() == dev))
        and (lse is None or (lse.dtype is torch.float32 and lse.shape == qs[:2]
                             and lse.is_contiguous() and lse.get_device() == dev))
    ):
        _check_prompt(q, k, v, cu_seqlens_q, cu_seqlens_k, output, lse)
    _native.check(_native.load().pkv_prompt_attention(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), cu_seqlens_q.data_ptr(),
        None if cu_seqlens_k is None else cu_seqlens_k.data_ptr(), output.data_ptr(),
        None if lse is None else lse.data_ptr(), cq[0] - 1, qs[0], ks[0], qs[1], ks[1], HEAD_DIM,
        qst[0], qst[1], kst[0], kst[1], vst[0], vst[1], _DTYPES[dt], _stream_of(dev)))


def _check_prefill(q, k, v, cu_seqlens, slots, output, lse, k_pages, v_pages, scales) -> None:
    """Everything that the write (``kv_write_fp8_block`` with ``scales``, else
    ``kv_write``) and ``prompt_attention`` of one batch of prompts would refuse."""
    _check_prompt(q, k, v, cu_seqlens, None, output, lse)
    _check_write(k, v, k_pages, v_pages, slots, k.dtype if scales is None else torch.float8_e4m3fn)
    if q.size(0) != k.size(0):
        raise RuntimeError("q, k and v must hold the same tokens")
    ks, vs = (None, None) if scales is None else scales
    block = 0 if scales is None else _check_block_scales(k_pages, ks, vs)
    _check_current_device(k_pages, v_pages, slots, ks, vs)
    _native.check(_native.load().pkv_prefill_check(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), output.data_ptr(),
        None if lse is None else lse.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(),
        None if ks is None else ks.data_ptr(), None if vs is None else vs.data_ptr(),
        cu_seqlens.size(0) - 1, q.size(0), q.size(1), k.size(1), HEAD_DIM, q.stride(0), q.stride(1),
        k.stride(0), k.stride(1), v.stride(0), v.stride(1), k_pages.size(0), k_pages.size(2), block,
        _DTYPES[q.dtype]))


def auto_workspace_bytes(batch: int, hq: int, hkv: int, sm_count: int = 0) -> int:
    """Workspace of ``paged_attention_auto`` (sm_count 0: the current device)."""
    return int(_native.load().pkv_auto_workspace_bytes(batch, hq, hkv, sm_count))


def combine_states(states, output, out_indices=None) -> None:
    """Merges ``states[n_parts, B, Hq, 130]`` into ``output`` rows (LSE combine)."""
    _check_tensor(states, "states", torch.float32, 4)
    _check_tensor(output, "output", tuple(_DTYPES), 3)
    n_parts, b, hq, width = states.shape
    if width != STATE_STRIDE:
        raise RuntimeError("states must have 130 values per head")
    if output.size(1) != hq or output.size(2) != HEAD_DIM:
        raise RuntimeError("output shape must match q head dimensions")
    idx_ptr = None
    if out_indices is not None:
        _check_tensor(out_indices, "out_indices", torch.int32, 1)
        if out_indices.size(0) != b:
            raise RuntimeError("out_indices batch mismatch")
        idx_ptr = out_indices.data_ptr()
    lib = _native.load()
    _native.check(lib.pkv_combine_states(
        states.data_ptr(), n_parts, idx_ptr, output.data_ptr(), b, output.size(0), hq,
        HEAD_DIM, _DTYPES[output.dtype], _stream()))


def workspace_bytes(batch: int, hq: int, num_splits: int) -> int:
    """Reference ``persistentkv_workspace_bytes`` (kernels/persistentkv_attention.cuh:891)."""
    return int(_native.load().pkv_workspace_bytes(batch, hq, num_splits))


def workqueue_workspace_bytes(total_partial_slots: int, hq: int) -> int:
    return int(_native.load().pkv_workqueue_workspace_bytes(total_partial_slots, hq))
