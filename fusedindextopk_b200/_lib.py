"""ctypes binding of ``libitk_b200.so`` (the C ABI declared in ``include/itk_b200.h``).

There is no fallback: if the shared library is missing or does not load, every
operator call raises.  Tensors are passed as raw device pointers
(``tensor.data_ptr()``) together with the current torch CUDA stream.
"""

from __future__ import annotations

import ctypes
from ctypes import POINTER, c_char_p, c_int, c_int32, c_longlong, c_size_t, c_uint64, c_void_p
from pathlib import Path
from typing import Any

import os
import struct

# ITK_B200_LIBRARY points the loader at another build of the same library (timing studies).
LIBRARY_PATH = Path(os.environ.get("ITK_B200_LIBRARY") or Path(__file__).resolve().parent / "libitk_b200.so")

TOP_K = 2048
HEADS = 64
HEAD_DIM = 128
BLOCK_Q = 4
REPAIR_CHUNK = 16384
SPILL_U64_PER_ROW = 5632
MAX_KEYS = 262144
MAX_PAIR_SOURCES = 16
MAX_CTAS = 256
STATIC_MAX_ROWS = 256
STATUS_WAIT_EXPIRED = 1
MAX_PLAN_REQUESTS = 16384
MAX_ATTENTION_KEYS = (1 << 31) - 1024
ELEMENT_BF16 = 0
ELEMENT_FP16 = 1
SERVING_STATUS = {
    1: "a bounded wait of the attention kernel expired", 2: "lengths that are negative, decrease or exceed their buffers",
    4: "a page or slot outside its pool", 8: "a page plan ran out of pages", 16: "misaligned shared memory",
}

EXPORTED_SYMBOLS = (
    "itk_version", "itk_last_error", "itk_init", "itk_resource_report", "itk_workspace_bytes",
    "itk_gather_sampled_kv", "itk_sample_thresholds", "itk_fused_topk", "itk_update_chunk_ranges",
    "itk_repair_produce", "itk_chunk_local_topk", "itk_merge_topk_pairs", "itk_finalize_repair",
    "itk_merge_candidate_lists", "itk_fused_topk_static", "itk_quantize_rows_e4m3",
    "itk_gather_sampled_kv_paged", "itk_repair_produce_paged", "itk_merge_shard_lists",
    "itk_compact_flagged_rows", "itk_repair_merge_chunk", "itk_flagged_scope_begin", "itk_flagged_scope_end",
    "itk_serving_status", "itk_plan_pages", "itk_append_tokens", "itk_attention", "itk_attention_workspace_bytes",
)


class ItkError(RuntimeError):
    """A C-ABI call returned a negative status."""


class WorkspaceSizes(ctypes.Structure):
    _fields_ = [
        ("spill_bytes", c_size_t), ("repair_pairs_bytes", c_size_t), ("pairs_bytes", c_size_t),
        ("counts_bytes", c_size_t), ("flags_bytes", c_size_t), ("thresholds_bytes", c_size_t),
        ("chunk_ranges_bytes", c_size_t), ("repair_chunks", c_int),
    ]


class FusedArgs(ctypes.Structure):
    _fields_ = [
        ("q", c_void_p), ("kv", c_void_p), ("kv_scales", c_void_p), ("weights", c_void_p),
        ("k_start", c_void_p), ("k_end", c_void_p), ("thresholds", c_void_p),
        ("out_ids", c_void_p), ("out_pairs", c_void_p), ("out_counts", c_void_p),
        ("failure_flags", c_void_p), ("spill", c_void_p),
        ("shard_pairs", c_void_p), ("shard_counts", c_void_p), ("shard_flags", c_void_p), ("diag_logits", c_void_p),
        ("diag_stride", c_longlong), ("trace", c_void_p), ("status", c_void_p),
        ("wait_limit_ns", ctypes.c_ulonglong), ("withhold_loads", c_int),
        ("rows", c_int), ("keys", c_int), ("key_lo", c_int), ("key_hi", c_int), ("shards", c_int),
        ("split_blocks", c_int), ("block_begin", c_int), ("block_stride", c_int), ("num_blocks", c_int),
        ("force_compute", c_int), ("max_ctas", c_int), ("exit_when_no_keys", c_int),
        ("tile_table", c_void_p), ("physical_keys", c_int),
        ("sampled_kv", c_void_p), ("sampled_scales", c_void_p), ("sample_ids", c_void_p), ("thresholds_out", c_void_p),
        ("samples", c_int), ("sample_rank", c_int), ("target_candidates", c_int),
    ]


class PagePlanArgs(ctypes.Structure):
    _fields_ = [
        ("table", c_void_p), ("old", c_void_p), ("fresh", c_void_p), ("free_pages", c_void_p),
        ("slots", c_void_p), ("cu_q", c_void_p), ("lengths", c_void_p), ("flat", c_void_p),
        ("k_start", c_void_p), ("k_end", c_void_p), ("pages_needed", c_void_p), ("table_stride", c_longlong),
        ("requests", c_int), ("table_pages", c_int), ("page_size", c_int), ("free_count", c_int), ("rows", c_int),
    ]


class AppendArgs(ctypes.Structure):
    _fields_ = [
        ("slots", c_void_p), ("k", c_void_p), ("v", c_void_p), ("k_pool", c_void_p), ("v_pool", c_void_p),
        ("index_source", c_void_p), ("index_pool", c_void_p), ("index_scales", c_void_p),
        ("k_token_stride", c_longlong), ("k_head_stride", c_longlong),
        ("v_token_stride", c_longlong), ("v_head_stride", c_longlong),
        ("k_page_stride", c_longlong), ("k_row_stride", c_longlong), ("k_pool_head_stride", c_longlong),
        ("v_page_stride", c_longlong), ("v_row_stride", c_longlong), ("v_pool_head_stride", c_longlong),
        ("index_stride", c_longlong),
        ("index_dtype", c_int), ("tokens", c_int), ("kv_heads", c_int), ("dim", c_int), ("pages", c_int),
        ("page_size", c_int),
    ]


class KvSegment(ctypes.Structure):
    _fields_ = [
        ("table_stride", c_longlong),
        ("k_page_stride", c_longlong), ("k_row_stride", c_longlong), ("k_head_stride", c_longlong),
        ("v_page_stride", c_longlong), ("v_row_stride", c_longlong), ("v_head_stride", c_longlong),
        ("pages", c_int), ("page_size", c_int), ("table_pages", c_int),
    ]


class AttentionArgs(ctypes.Structure):
    _fields_ = [
        ("q", c_void_p), ("out", c_void_p), ("lse", c_void_p), ("cu_q", c_void_p), ("cu_k", c_void_p),
        ("lens_k", c_void_p), ("workspace", c_void_p), ("workspace_bytes", c_size_t),
        ("k", c_void_p), ("v", c_void_p), ("table", c_void_p),
        ("k_prefix", c_void_p), ("v_prefix", c_void_p), ("prefix_table", c_void_p),
        ("q_token_stride", c_longlong), ("q_head_stride", c_longlong),
        ("out_token_stride", c_longlong), ("out_head_stride", c_longlong), ("wait_limit_ns", ctypes.c_ulonglong),
        ("own", KvSegment), ("prefix", KvSegment), ("scale", ctypes.c_float), ("element", c_int),
        ("tokens", c_int), ("heads", c_int), ("kv_heads", c_int), ("dim", c_int), ("requests", c_int),
        ("prefix_keys", c_int), ("causal", c_int), ("clear_tail", c_int), ("withhold_loads", c_int),
    ]


_library: ctypes.CDLL | None = None


def load_library() -> ctypes.CDLL:
    """Load the shared library once; raise if it is not there."""

    global _library
    if _library is not None:
        return _library
    if not LIBRARY_PATH.exists():
        raise ItkError(
            f"{LIBRARY_PATH} is missing: build it with `python -m fusedindextopk_b200.build` "
            "(there is no CPU or PyTorch fallback)"
        )
    library = ctypes.CDLL(str(LIBRARY_PATH))
    library.itk_version.restype = c_char_p
    library.itk_last_error.restype = c_char_p
    library.itk_init.argtypes = [c_int]
    library.itk_resource_report.argtypes = [c_char_p, c_size_t]
    library.itk_workspace_bytes.argtypes = [c_int, c_int, c_int, POINTER(WorkspaceSizes)]
    library.itk_gather_sampled_kv.argtypes = [c_void_p] * 5 + [c_int, c_int, c_void_p]
    library.itk_sample_thresholds.argtypes = (
        [c_void_p] * 8 + [c_int] * 8 + [c_void_p, c_longlong, c_void_p, c_void_p, c_void_p]
    )
    library.itk_fused_topk.argtypes = [POINTER(FusedArgs), c_void_p]
    library.itk_fused_topk_static.argtypes = [POINTER(FusedArgs), c_void_p]
    library.itk_update_chunk_ranges.argtypes = [c_void_p] * 4 + [c_int, c_int, c_void_p]
    library.itk_repair_produce.argtypes = [c_void_p] * 8 + [c_int] * 7 + [c_void_p, c_void_p]
    library.itk_chunk_local_topk.argtypes = [c_void_p] * 7 + [c_int, c_int, c_void_p]
    library.itk_merge_topk_pairs.argtypes = [c_void_p] * 6 + [c_int, c_int, c_void_p]
    library.itk_finalize_repair.argtypes = [c_void_p] * 7 + [c_int, c_void_p]
    library.itk_merge_candidate_lists.argtypes = (
        [POINTER(c_void_p), POINTER(c_void_p), c_int, c_void_p, c_void_p, c_void_p, c_int, c_void_p]
    )
    library.itk_merge_shard_lists.argtypes = (
        [POINTER(c_void_p), POINTER(c_void_p), c_int, c_void_p, c_void_p, c_void_p, c_int]
        + [c_void_p] * 4 + [c_int] * 5 + [c_void_p, c_void_p, c_void_p]
    )
    library.itk_flagged_scope_begin.argtypes = [c_void_p, c_int, c_void_p, POINTER(c_void_p)]
    library.itk_flagged_scope_end.argtypes = [c_void_p, c_void_p]
    library.itk_compact_flagged_rows.argtypes = [c_void_p] * 5 + [c_int, c_int] + [c_void_p] * 6
    library.itk_repair_merge_chunk.argtypes = (
        [c_void_p] * 5 + [c_int, c_int, c_void_p, c_void_p, c_int, c_int, c_int] + [c_void_p] * 5
    )
    library.itk_gather_sampled_kv_paged.argtypes = [c_void_p] * 6 + [c_int, c_int, c_int, c_void_p]
    library.itk_repair_produce_paged.argtypes = [c_void_p] * 8 + [c_int] * 7 + [c_void_p, c_int, c_void_p, c_void_p]
    library.itk_quantize_rows_e4m3.argtypes = [c_void_p, c_int] + [c_void_p] * 4 + [c_longlong, c_void_p]
    library.itk_serving_status.argtypes = [POINTER(c_int), c_int]
    # (the argument blocks of these three are passed as raw memory: see CallTemplate)
    library.itk_plan_pages.argtypes = [c_void_p, c_void_p]
    library.itk_append_tokens.argtypes = [c_void_p, c_void_p]
    library.itk_attention.argtypes = [c_void_p, c_void_p]
    library.itk_attention_workspace_bytes.argtypes = [POINTER(AttentionArgs), POINTER(c_size_t)]
    for name in EXPORTED_SYMBOLS:
        function = getattr(library, name)
        if name not in ("itk_version", "itk_last_error"):
            function.restype = c_int
    _library = library
    return library


def check(status: int) -> None:
    if status != 0:
        message = load_library().itk_last_error().decode(errors="replace")
        raise ItkError(f"libitk_b200 error {status}: {message}")


def ptr(tensor: Any) -> int | None:
    """Device address of a tensor, or NULL for ``None``."""

    return None if tensor is None else int(tensor.data_ptr())


def current_stream(torch: Any, device: Any) -> int:
    return int(torch.cuda.current_stream(device).cuda_stream)


def version() -> str:
    return load_library().itk_version().decode()


def resource_report() -> dict[str, str]:
    """Registers / shared memory / launch shape of the kernels on the current device."""

    buffer = ctypes.create_string_buffer(8192)
    check(load_library().itk_resource_report(buffer, len(buffer)))
    report: dict[str, str] = {}
    for line in buffer.value.decode().splitlines():
        if "=" in line:
            key, value = line.split("=", 1)
            report[key] = value
    return report


def workspace_sizes(rows: int, keys: int, shards: int = 1) -> WorkspaceSizes:
    sizes = WorkspaceSizes()
    check(load_library().itk_workspace_bytes(rows, keys, shards, ctypes.byref(sizes)))
    return sizes


class CallTemplate:
    """What a call with these shapes, strides and types always passes: a checked argument block without its pointers.

    The serving calls are short, and reading and checking the metadata of half a dozen tensors takes longer than the
    launch.  A call whose tensors have the metadata of an earlier one takes that one's block and fills in the addresses.
    Nothing about addresses or contents is kept.
    """

    LIMIT = 1024

    def __init__(self, args: ctypes.Structure, **extra: Any) -> None:
        self.bytes = bytes(args)
        self.__dict__.update(extra)

    def fill(self, words: Any) -> bytes:
        """A copy of the block with the 64-bit words it begins with put in."""

        return _WORDS[len(words)].pack(*words) + self.bytes[8 * len(words):]

    @classmethod
    def keep(cls, templates: dict, key: Any, template: "CallTemplate") -> "CallTemplate":
        if len(templates) >= cls.LIMIT:
            templates.clear()
        templates[key] = template
        return template


_WORDS = [struct.Struct("<%dQ" % n) for n in range(32)]


def metadata(torch: Any, tensors: tuple) -> tuple:
    # (the device by its number, which is quicker; what is not on a GPU has -1 and is refused, so it is never kept)
    if torch.autograd.forward_ad._current_level >= 0 and any(
            torch.autograd.forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise ValueError("there is no forward-mode derivative: detach")
    return tuple([(t.shape, t.stride(), t.dtype, t.get_device()) for t in tensors])


def refuse_gradients(torch: Any, *tensors: Any) -> None:
    """Raise where a call would drop the gradients that its tensors ask for."""

    if torch.is_grad_enabled():
        for t in tensors:
            if t.requires_grad:
                raise ValueError("there is no backward pass: call it under torch.no_grad() or detach")


def launch(torch: Any, function: Any, block: Any, device: Any, written: tuple = ()) -> None:
    """Calls a C entry on the current stream of ``device``; ``written`` are the caller's tensors that it writes to."""

    index = device.index
    if torch._C._cuda_getDevice() == index:
        status = function(block, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(device):
            status = function(block, torch._C._cuda_getCurrentRawStream(index))
    if status:
        check(status)
    if written:         # a graph that has saved one of them finds that it has changed
        torch._C._increment_version(written)


def check_serving_status(device: Any = None) -> None:
    """Raise when a page plan, an append or an attention call on ``device`` met something it had to clamp, skip or give up.

    Synchronises the device and clears what it reports.  One word per device: it does not say which call it was.
    """

    import torch

    status = c_int(0)
    with torch.cuda.device(device):
        check(load_library().itk_serving_status(ctypes.byref(status), 1))
    if status.value:
        raise ItkError("serving status: " + "; ".join(text for bit, text in SERVING_STATUS.items() if status.value & bit))


def pointer_table(tensors: list[Any]) -> Any:
    table = (c_void_p * len(tensors))()
    for index, tensor in enumerate(tensors):
        table[index] = tensor.data_ptr()
    return table


__all__ = [
    "AppendArgs", "AttentionArgs", "BLOCK_Q", "ELEMENT_BF16", "ELEMENT_FP16", "EXPORTED_SYMBOLS", "FusedArgs", "HEADS",
    "HEAD_DIM", "ItkError", "KvSegment", "LIBRARY_PATH", "MAX_ATTENTION_KEYS", "MAX_KEYS", "MAX_PAIR_SOURCES", "MAX_PLAN_REQUESTS", "PagePlanArgs",
    "SERVING_STATUS", "REPAIR_CHUNK", "SPILL_U64_PER_ROW", "STATUS_WAIT_EXPIRED", "TOP_K", "WorkspaceSizes",
    "check", "check_serving_status", "current_stream", "load_library", "pointer_table", "ptr", "resource_report", "version",
    "workspace_sizes", "c_int32", "c_uint64",
]
