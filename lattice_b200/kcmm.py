"""ctypes binding of the B200 KCMM library (`libkcmm.so`).

Mirrors the reference's Python seam (ref scripts/kcmm/bindings.py:17-429):
the same class names (`KcmmError`, `KcmmConfig`, `KcmmMetrics`,
`KcmmPoolStats`, `BlockLocation`, `KcmmLibrary`, `KcmmPool`), the same
struct layouts with the same layout assertion, and pool methods with the same
names, argument meaning and error behaviour (a failing call raises
`KcmmError` carrying the pool's last error).  Methods for the B200 additions
(bf16 decode, fused norm/rope/append, refcount/CoW, swap) follow the same
pattern.

There is no fallback: if the native library is missing the import of
`KcmmLibrary()` raises.  Device buffers are passed as integer addresses, so
any framework (torch here, in tests and the bench) can own them.
"""
from __future__ import annotations

import ctypes
import gc
import os
import weakref
from pathlib import Path

_PKG = Path(__file__).resolve().parent


class KcmmError(RuntimeError):
    """A KCMM C API call reported failure."""


class KcmmConfig(ctypes.Structure):
    _fields_ = [
        ("block_size", ctypes.c_size_t),
        ("max_blocks", ctypes.c_size_t),
        ("cpu_cache_path", ctypes.c_char * 256),
        ("tiering", ctypes.c_int32),
        ("eviction_policy", ctypes.c_int32),
        ("prefetch_window", ctypes.c_size_t),
        ("max_batch_blocks", ctypes.c_size_t),
        ("device_ordinal", ctypes.c_size_t),
        ("num_layers", ctypes.c_size_t),
        ("kv_heads", ctypes.c_size_t),
        ("head_dim", ctypes.c_size_t),
        ("max_batch", ctypes.c_size_t),
        ("max_seq_len", ctypes.c_size_t),
        ("low_watermark_threshold", ctypes.c_float),
        ("background_evict_interval_ms", ctypes.c_uint64),
        ("attention_sink_blocks", ctypes.c_size_t),
        ("recent_window_blocks", ctypes.c_size_t),
    ]


class KcmmMetrics(ctypes.Structure):
    _fields_ = [
        ("ifr", ctypes.c_double),
        ("pme", ctypes.c_double),
        ("bu", ctypes.c_double),
        ("rfi", ctypes.c_double),
        ("gpu_blocks", ctypes.c_uint64),
        ("cpu_blocks", ctypes.c_uint64),
        ("nvme_blocks", ctypes.c_uint64),
        ("eviction_count", ctypes.c_uint64),
        ("restoration_count", ctypes.c_uint64),
    ]


class KcmmLatencyHistogram(ctypes.Structure):
    _fields_ = [("count", ctypes.c_uint64), ("sum_us", ctypes.c_uint64),
                ("min_us", ctypes.c_uint64), ("max_us", ctypes.c_uint64),
                ("buckets", ctypes.c_uint64 * 9)]


class KcmmMetricsExt(ctypes.Structure):
    _fields_ = [("base", KcmmMetrics), ("evicted_blocks_total", ctypes.c_uint64),
                ("restored_blocks_total", ctypes.c_uint64),
                ("eviction_failures", ctypes.c_uint64),
                ("restoration_failures", ctypes.c_uint64),
                ("background_eviction_count", ctypes.c_uint64),
                ("eviction_latency", KcmmLatencyHistogram),
                ("restoration_latency", KcmmLatencyHistogram)]


class KcmmPolicyStats(ctypes.Structure):
    _fields_ = [("eviction_count", ctypes.c_uint64), ("restoration_count", ctypes.c_uint64),
                ("evicted_blocks", ctypes.c_uint64), ("restored_blocks", ctypes.c_uint64),
                ("avg_evict_batch_size", ctypes.c_double)]


class KcmmPoolStats(ctypes.Structure):
    _fields_ = [
        ("blocks_in_use", ctypes.c_uint32),
        ("total_blocks", ctypes.c_uint32),
        ("total_physical_blocks", ctypes.c_uint32),
        ("free_physical_blocks", ctypes.c_uint32),
        ("active_sequences", ctypes.c_uint32),
        ("num_layers", ctypes.c_uint32),
        ("blocks_per_superblock", ctypes.c_uint32),
        ("superblock_count", ctypes.c_uint32),
        ("block_size", ctypes.c_uint32),
        ("max_blocks_per_seq", ctypes.c_uint32),
        ("block_bytes", ctypes.c_uint32),
        ("tiering_enabled", ctypes.c_int32),
        ("sharing_enabled", ctypes.c_int32),
        ("physical_idle_ratio", ctypes.c_float),
    ]


class BlockLocation:
    GPU_RESIDENT = 0
    CPU_RESIDENT = 1
    NVME_RESIDENT = 2
    EVICTING = 3
    RESTORING = 4
    _NAMES = {0: "gpu", 1: "cpu", 2: "nvme", 3: "evicting", 4: "restoring"}

    @classmethod
    def name(cls, value: int) -> str:
        return cls._NAMES.get(value, f"unknown({value})")


class CacheFormat:
    """What a pool's pages hold (`kcmm_cache_format_t`)."""
    BITS16 = 0
    KV4 = 1


_DTYPES = {"f16": 0, "bf16": 1, "f32": 2}  # kcmm_dtype_t


class RopeMode:
    REFERENCE = 0
    GPTJ = 1
    NEOX = 2


def assert_layout() -> None:
    """The config struct must match the C header byte for byte on LP64."""
    if ctypes.sizeof(ctypes.c_size_t) != 8:
        return
    expected = {
        "max_seq_len": 336,
        "low_watermark_threshold": 344,
        "background_evict_interval_ms": 352,
        "attention_sink_blocks": 360,
        "recent_window_blocks": 368,
    }
    if ctypes.sizeof(KcmmConfig) != 376:
        raise KcmmError(f"kcmm_config_t size {ctypes.sizeof(KcmmConfig)} != 376")
    for name, off in expected.items():
        got = getattr(KcmmConfig, name).offset
        if got != off:
            raise KcmmError(f"kcmm_config_t.{name} at offset {got}, expected {off}")


def library_path() -> Path:
    env = os.environ.get("KCMM_LIB_PATH")
    path = Path(env) if env else _PKG / "libkcmm.so"
    if not path.exists():
        raise KcmmError(
            f"KCMM native library not found at {path}; build it with "
            "`python -m lattice_b200.build` (nvcc, sm_100a)"
        )
    return path


u32, u64, i32, i64, f32 = (ctypes.c_uint32, ctypes.c_uint64, ctypes.c_int32, ctypes.c_int64,
                         ctypes.c_float)
P = ctypes.c_void_p
pu32 = ctypes.POINTER(ctypes.c_uint32)
pu64 = ctypes.POINTER(ctypes.c_uint64)
pi64 = ctypes.POINTER(ctypes.c_int64)
pu8 = ctypes.POINTER(ctypes.c_uint8)

# name -> (restype, argtypes); every symbol declared in include/kcmm.h
SIGNATURES: dict[str, tuple] = {
    "kcmm_pool_create": (P, [ctypes.POINTER(KcmmConfig)]),
    "kcmm_pool_destroy": (None, [P]),
    "kcmm_get_last_error": (ctypes.c_size_t, [P, ctypes.c_char_p, ctypes.c_size_t]),
    "kcmm_clear_error": (None, [P]),
    "kcmm_alloc_blocks": (i32, [P, u32, pu32]),
    "kcmm_free_blocks": (i32, [P, pu32, u32]),
    "kcmm_register_sequence": (i32, [P, pu32, u32, pu32]),
    "kcmm_unregister_sequence": (i32, [P, u32]),
    "kcmm_touch": (None, [P, u32]),
    "kcmm_cool": (None, [P, u32]),
    "kcmm_update_seq_len": (None, [P, u32, u32]),
    "kcmm_get_seq_len": (u32, [P, u32]),
    "kcmm_append_block_to_sequence": (i32, [P, u32, u32]),
    "kcmm_get_block_table": (i32, [P, u32, pu32, u32, pu32]),
    "kcmm_get_block_va_offset": (u64, [P, u32]),
    "kcmm_get_all_block_offsets_f16": (i32, [P, pu64, u32, pu32]),
    "kcmm_get_all_block_valid": (i32, [P, pu8, u32, pu32]),
    "kcmm_get_block_location": (i32, [P, u32, ctypes.POINTER(ctypes.c_int)]),
    "kcmm_get_block_table_va_offsets": (i32, [P, u32, pu64, u32, pu32]),
    "kcmm_get_va_k": (u64, [P, u32]),
    "kcmm_get_va_v": (u64, [P, u32]),
    "kcmm_block_state_epoch": (u64, [P]),
    "kcmm_append_kv_step": (i32, [P, u32, pu32, pu32, u32, u64, u64]),
    "kcmm_append_kv_slots": (i32, [P, u32, pi64, u32, u64, u64]),
    "kcmm_append_kv_slots_on_stream": (i32, [P, u32, pi64, u32, u64, u64, u64]),
    "kcmm_append_kv_device_slots_on_stream":
        (i32, [P, u32, u64, u64, u64, u32, u32, u64, u64, u64, u64]),
    "kcmm_precompile_vllm_kv_write_f16": (i32, [P]),
    "kcmm_paged_attn_decode_f16":
        (i32, [P, u32, u64, u64, u64, u64, u64, u32, u32, u32, u32, u32, u32, f32]),
    "kcmm_paged_attn_decode_f16_on_stream":
        (i32, [P, u32, u64, u64, u64, u64, u64, u32, u32, u32, u32, u32, u32, f32, u64]),
    "kcmm_paged_attn_decode_f16_on_current_context_stream":
        (i32, [P, u32, u64, u64, u64, u64, u64, u32, u32, u32, u32, u32, u32, f32, u64]),
    "kcmm_precompile_paged_attn_decode_f16": (i32, [P]),
    "kcmm_evict_blocks": (u32, [P, u32]),
    "kcmm_restore_evicted_block": (u64, [P, u32]),
    "kcmm_restore_evicted_blocks": (i32, [P, pu32, u32]),
    "kcmm_is_gpu_resident": (i32, [P, u32]),
    "kcmm_get_metrics": (i32, [P, ctypes.POINTER(KcmmMetrics)]),
    "kcmm_get_pool_stats": (i32, [P, ctypes.POINTER(KcmmPoolStats)]),
    "kcmm_blocks_in_use": (u32, [P]),
    "kcmm_total_blocks": (u32, [P]),
    "kcmm_free_physical_blocks": (u32, [P]),
    "kcmm_has_free_blocks": (i32, [P]),
    "kcmm_active_sequences": (u32, [P]),
    "kcmm_set_eviction_policy": (i32, [P, ctypes.c_char_p]),
    "kcmm_get_eviction_policy": (u32, [P, ctypes.c_char_p, u32]),
    "kcmm_is_tiering_enabled": (i32, [P]),
    "kcmm_hint": (i32, [P, u32, ctypes.c_int]),
    "kcmm_protect": (i32, [P, u32, pu32, u32, ctypes.c_int]),
    "kcmm_share_prefix": (i32, [P, u32, u32, u32, pu32]),
    "kcmm_below_low_watermark": (i32, [P, f32]),
    "kcmm_synchronize": (i32, [P]),
    "kcmm_get_block_size": (u32, [P]),
    "kcmm_get_max_blocks_per_seq": (u32, [P]),
    "kcmm_get_block_bytes": (u32, [P]),
    "kcmm_get_num_layers": (u32, [P]),
    "kcmm_get_max_batch": (u32, [P]),
    "kcmm_get_max_seq_len": (u32, [P]),
    # --- B200 additions ---
    "kcmm_paged_attn_decode_bf16_on_stream":
        (i32, [P, u32, u64, u64, u64, u64, u64, u32, u32, u32, u32, u32, u32, f32, u64]),
    "kcmm_paged_attn_decode_bf16_noalloc_on_stream":
        (i32, [P, u32, u64, u64, u64, u64, u64, u32, u32, u32, u32, u32, u32, f32, u64]),
    "kcmm_paged_prefill_bf16_on_stream":
        (i32, [P, u32, u64, u64, u64, u64, u64, u64, u32, u32, u32, u32, u32, u32, u32, f32,
               u64]),
    "kcmm_paged_prefill_f16_on_stream":
        (i32, [P, u32, u64, u64, u64, u64, u64, u64, u32, u32, u32, u32, u32, u32, u32, f32,
               u64]),
    "kcmm_append_kv_device_slots_bf16_on_stream":
        (i32, [P, u32, u64, u64, u64, u32, u32, u64, u64, u64, u64]),
    "kcmm_fused_norm_rope_append_bf16_on_stream":
        (i32, [P, u32, u64, u64, u64, u32, f32, u64, u32, u64, u64, u64, f32, u32,
               u64, u64, u64, u32, u32, u64, u64]),
    "kcmm_kv4_row_elems": (u32, [u32]),
    **{f"kcmm_kv4_{op}_{dt}_on_stream":
       (i32, [P, u32, u64, u64, u64, u32, u32, u32, u64, i64, u64, i64, u64, u64])
       for op in ("append", "read") for dt in ("bf16", "f16")},
    **{f"kcmm_{op}_{dt}_on_stream":
       (i32, [P, u32, u64, i64, i64, u64, i64, i64, u64, i64, u64, u64, u32, u32, u32, u32, u32,
              u32, f32, u64, u64, i64, u64])
       for op in ("kv4_paged_attn_decode", "paged_attn_decode_weights") for dt in ("bf16", "f16")},
    "kcmm_evict_tokens_on_stream":
        (i32, [P, u32, u32, u32, u64, i64, u64, u64, u32, u32, u32, u32, u32, u64, u64, u64, u64,
               i64, u64, u64, u64, u64]),
    "kcmm_truncate_sequence": (i32, [P, u32, u32]),
    **{f"kcmm_rope_append_{dt}_on_stream":
       (i32, [P, u32, u32, u32, ctypes.c_void_p, u64, i64, i64, u64, i64, i64, u32, u64, i64, u64,
              i64, u64, i64, u64, u64, u64, u32, u32, u64, u64])
       for dt in ("bf16", "f16")},
    **{f"kcmm_prompt_attn_{dt}_on_stream":
       (i32, [P, u64, i64, i64, u64, i64, i64, u64, i64, i64, u64, i64, i64, u64, u64, u32, u32,
              u32, u32, u32, u32, f32, u32, u64])
       for dt in ("bf16", "f16")},
    "kcmm_beam_select_on_stream":
        (i32, [P, u64, u32, i64, u64, u64, u32, u32, u32, u32, u32, u64, u64, u64, u64]),
    "kcmm_beam_gather_on_stream":
        (i32, [P, u64, u64, u64, u64, u32, u32, u32, u64, u64, u64]),
    "kcmm_reorder_sequences_on_stream": (i32, [P, pu32, pu32, u32, u64]),
    "kcmm_block_incref": (i32, [P, u32]),
    "kcmm_block_decref": (i32, [P, u32]),
    "kcmm_block_refcount": (u32, [P, u32]),
    "kcmm_fork_sequence": (i32, [P, u32, pu32]),
    "kcmm_cow_blocks_on_stream": (i32, [P, pu32, pu32, u32, pu32, u64]),
    "kcmm_swap_out_blocks_on_stream": (i32, [P, pu32, u32, u64]),
    "kcmm_swap_in_blocks_on_stream": (i32, [P, pu32, u32, u64]),
    "kcmm_get_kernel_status": (i32, [P]),
    "kcmm_paged_attn_decode_bf16_strided_on_stream":
        (i32, [P, u32, u64, i64, i64, u64, i64, i64, u64, i64, u64, u64, u32, u32, u32, u32, u32,
               u32, f32, u64]),
    "kcmm_paged_attn_decode_f16_strided_on_stream":
        (i32, [P, u32, u64, i64, i64, u64, i64, i64, u64, i64, u64, u64, u32, u32, u32, u32, u32,
               u32, f32, u64]),
    "kcmm_append_kv_device_slots_strided_on_stream":
        (i32, [P, u32, u64, u64, u64, u32, u32, u64, i64, u64, i64, u64, u64]),
    "kcmm_peer_signal_words": (u32, [u32]),
    "kcmm_peer_allgather_on_stream": (i32, [u64, u64, pu64, pu64, u32, u32, u64, u64]),
    "kcmm_peer_wait_on_stream": (i32, [u64, u32, u64, u64, u64]),
    "kcmm_paged_attn_decode_shared_prefix_bf16_on_stream": (
        i32, [P, u32, u64, u64, u64, u64, u64, u32, u32, u32, u32, u32, u32, f32, u64, u64,
              u32, u32, u64]),
    "kcmm_paged_attn_decode_shared_prefix_f16_on_stream": (
        i32, [P, u32, u64, u64, u64, u64, u64, u32, u32, u32, u32, u32, u32, f32, u64, u64,
              u32, u32, u64]),
    "kcmm_paged_attn_decode_bf16_allgather_on_stream": (
        i32, [P, u32, u64, u64, u64, u64, u64, u32, u32, u32, u32, u32, u32, f32, pu64, pu64,
              u32, u32, u64, u64]),
    "kcmm_paged_attn_decode_f16_allgather_on_stream": (
        i32, [P, u32, u64, u64, u64, u64, u64, u32, u32, u32, u32, u32, u32, f32, pu64, pu64,
              u32, u32, u64, u64]),
    "kcmm_get_metrics_ext": (i32, [P, ctypes.c_void_p]),
    "kcmm_get_policy_stats": (i32, [P, ctypes.c_char_p, ctypes.c_void_p]),
    "kcmm_start_background_eviction": (i32, [P]),
    "kcmm_stop_background_eviction": (i32, [P]),
    "kcmm_preview_eviction_victims": (u32, [P, u32, pu32, u32]),
    "kcmm_step_tables_create": (P, [P, u32]),
    "kcmm_step_tables_destroy": (None, [P]),
    "kcmm_step_tables_sync_on_stream": (i32, [P, pu32, u32, u64]),
    "kcmm_step_tables_block_tables": (u64, [P]),
    "kcmm_step_tables_seq_lens": (u64, [P]),
    "kcmm_step_tables_block_offsets": (u64, [P]),
    "kcmm_step_tables_stats": (i32, [P, ctypes.c_void_p]),
    "kcmm_build_info": (ctypes.c_char_p, []),
}


class KcmmRope(ctypes.Structure):
    """The rotation of a model's q and k rows (`kcmm_rope_t`)."""
    _fields_ = [("mode", ctypes.c_uint32), ("rotary_dim", ctypes.c_uint32),
                ("inv_freq_ptr", ctypes.c_uint64), ("positions_ptr", ctypes.c_uint64),
                ("positions_row_stride", ctypes.c_int64), ("axes", ctypes.c_uint32),
                ("layout", ctypes.c_uint32), ("sections", ctypes.c_uint32 * 4)]


def make_rope(*, rotary_dim: int, inv_freq_ptr: int, positions_ptr: int,
              positions_row_stride: int = 0, sections=None, mode: str = "neox",
              layout: str = "sections") -> KcmmRope:
    """A `KcmmRope`: `sections` are the pairs of each axis (None: one axis), `mode` "neox" or
    "gptj", `layout` "sections" or "interleaved"."""
    sections = [rotary_dim // 2] if sections is None else [int(s) for s in sections]
    if not 1 <= len(sections) <= 4:
        raise ValueError(f"1 to 4 axes, not {len(sections)}")
    return KcmmRope({"gptj": RopeMode.GPTJ, "neox": RopeMode.NEOX}[mode], rotary_dim,
                    inv_freq_ptr, positions_ptr, positions_row_stride, len(sections),
                    {"sections": 0, "interleaved": 1}[layout],
                    (ctypes.c_uint32 * 4)(*sections))


class KcmmStepTablesStats(ctypes.Structure):
    _fields_ = [("syncs", ctypes.c_uint64), ("table_entries", ctypes.c_uint64),
                ("offset_entries", ctypes.c_uint64), ("bytes", ctypes.c_uint64),
                ("full_offsets", ctypes.c_uint64)]


class StepTables:
    """Device-resident block tables / lengths / offsets of one ordered batch
    (`kcmm_step_tables_*`); `sync` uploads only what changed."""

    def __init__(self, pool: "KcmmPool", max_batch: int):
        self.pool = pool
        self.lib = pool.lib
        h = self.lib.kcmm_step_tables_create(pool.handle, max_batch)
        if not h:
            raise KcmmError(f"kcmm_step_tables_create: {pool.last_error()}")
        self.handle = ctypes.c_void_p(h)
        self.max_batch = max_batch

    def sync(self, seq_indices, stream_ptr: int = 0) -> None:
        arr = _u32_array(seq_indices)
        rc = self.lib.kcmm_step_tables_sync_on_stream(self.handle, arr, len(seq_indices),
                                                      stream_ptr)
        if rc != 0:
            raise KcmmError(f"kcmm_step_tables_sync_on_stream: {self.pool.last_error()}")

    @property
    def block_tables_ptr(self) -> int:
        return self.lib.kcmm_step_tables_block_tables(self.handle)

    @property
    def seq_lens_ptr(self) -> int:
        return self.lib.kcmm_step_tables_seq_lens(self.handle)

    @property
    def block_offsets_ptr(self) -> int:
        return self.lib.kcmm_step_tables_block_offsets(self.handle)

    def stats(self) -> dict:
        st = KcmmStepTablesStats()
        if self.lib.kcmm_step_tables_stats(self.handle, ctypes.byref(st)) != 0:
            raise KcmmError("kcmm_step_tables_stats failed")
        return {f: getattr(st, f) for f, _ in st._fields_}

    def destroy(self) -> None:
        if self.handle:
            self.lib.kcmm_step_tables_destroy(self.handle)
            self.handle = None


def _u32_array(values):
    values = [int(v) for v in values]
    return (ctypes.c_uint32 * max(1, len(values)))(*values)


def kv4_row_elems(head_dim: int) -> int:
    """The pool head_dim of a 4-bit cache of `head_dim` (`kcmm_kv4_row_elems`)."""
    if head_dim <= 0 or head_dim % 32 != 0 or head_dim > 256:
        raise ValueError(f"the 4-bit cache takes head dims that are multiples of 32 up to 256, "
                         f"not {head_dim}")
    return head_dim * 9 // 32


class KcmmLibrary:
    """Loads `libkcmm.so` and binds every exported function."""

    def __init__(self, path: str | Path | None = None):
        assert_layout()
        self.path = Path(path) if path else library_path()
        self.lib = ctypes.CDLL(str(self.path))
        for name, (res, args) in SIGNATURES.items():
            fn = getattr(self.lib, name)
            fn.restype = res
            fn.argtypes = args

    def create_pool(self, config: KcmmConfig) -> "KcmmPool":
        handle = self.lib.kcmm_pool_create(ctypes.byref(config))
        if not handle:
            raise KcmmError("kcmm_pool_create returned NULL")
        return KcmmPool(self, handle)

    def build_info(self) -> str:
        return self.lib.kcmm_build_info().decode()


def make_config(*, num_layers: int, kv_heads: int, head_dim: int, max_batch: int,
                max_seq_len: int, block_size: int = 16, max_blocks: int = 0,
                tiering: bool = False, eviction_policy: int = 0, device: int = 0,
                cpu_cache_path: str = "") -> KcmmConfig:
    cfg = KcmmConfig()
    cfg.block_size = block_size
    cfg.max_blocks = max_blocks
    cfg.cpu_cache_path = cpu_cache_path.encode()
    cfg.tiering = 1 if tiering else 0
    cfg.eviction_policy = eviction_policy
    cfg.device_ordinal = device
    cfg.num_layers = num_layers
    cfg.kv_heads = kv_heads
    cfg.head_dim = head_dim
    cfg.max_batch = max_batch
    cfg.max_seq_len = max_seq_len
    return cfg


class _Regions:
    """Holds a pool's device memory: a pool that was destroyed releases it when neither the
    pool nor any `RegionAddress` refers to this any more."""

    def __init__(self, lib, handle):
        self.lib, self.handle, self.closed = lib, handle, False

    def __del__(self):
        if self.closed:
            self.lib.kcmm_pool_destroy(self.handle)


class RegionAddress(int):
    """A region's device address.  The region stays mapped while this object lives, so that a
    tensor over it (`__cuda_array_interface__` with this object in "data") may outlive the
    pool; what arithmetic makes of it is a plain int and holds nothing."""

    def __new__(cls, address: int, regions: _Regions):
        self = super().__new__(cls, address)
        self._regions = regions
        return self

    def __reduce__(self):  # a copy, or what was pickled, is a plain int
        return int, (int(self),)


class KcmmPool:
    """One pool handle; every method raises `KcmmError` on a -1 return."""

    def __init__(self, library: KcmmLibrary, handle):
        self.library = library
        self.lib = library.lib
        self.handle = ctypes.c_void_p(handle)
        self._regions = _Regions(self.lib, self.handle)
        self._destroyed = False

    def __enter__(self) -> "KcmmPool":
        return self

    def __exit__(self, *_exc) -> None:
        self.destroy()

    # --- errors ---------------------------------------------------------
    def last_error(self) -> str:
        buf = ctypes.create_string_buffer(4096)
        n = self.lib.kcmm_get_last_error(self.handle, buf, ctypes.sizeof(buf))
        return buf.value.decode("utf-8", errors="replace") if n else ""

    def clear_error(self) -> None:
        self.lib.kcmm_clear_error(self.handle)

    def _check(self, rc: int, op: str) -> None:
        if rc != 0:
            raise KcmmError(f"{op} failed: {self.last_error() or 'unknown KCMM error'}")

    def destroy(self) -> None:
        """Release everything; the regions only once no address of `va_k` / `va_v`, nor a tensor
        over one, is left.  No other call on the pool may follow."""
        if self._destroyed:
            return
        self._destroyed = True
        self._regions.closed = True
        held = weakref.ref(self._regions)
        self._regions = None
        if held() is not None:
            gc.collect()  # the class that hands an address to a tensor lies in a cycle

    # --- blocks and sequences --------------------------------------------
    def alloc_blocks(self, count: int) -> list[int]:
        if count <= 0:
            raise ValueError("count must be positive")
        out = (ctypes.c_uint32 * count)()
        self._check(self.lib.kcmm_alloc_blocks(self.handle, count, out), "kcmm_alloc_blocks")
        return list(out)

    def free_blocks(self, blocks) -> None:
        if len(blocks) == 0:
            return
        arr = _u32_array(blocks)
        self._check(self.lib.kcmm_free_blocks(self.handle, arr, len(blocks)), "kcmm_free_blocks")

    def register_sequence(self, block_table) -> int:
        arr = _u32_array(block_table)
        out = ctypes.c_uint32()
        self._check(self.lib.kcmm_register_sequence(self.handle, arr, len(block_table),
                                                    ctypes.byref(out)),
                    "kcmm_register_sequence")
        return out.value

    def unregister_sequence(self, seq_idx: int) -> None:
        self._check(self.lib.kcmm_unregister_sequence(self.handle, seq_idx),
                    "kcmm_unregister_sequence")

    def append_block_to_sequence(self, seq_idx: int, block_idx: int) -> None:
        self._check(self.lib.kcmm_append_block_to_sequence(self.handle, seq_idx, block_idx),
                    "kcmm_append_block_to_sequence")

    def touch(self, seq_idx: int) -> None:
        self.lib.kcmm_touch(self.handle, seq_idx)

    def cool(self, seq_idx: int) -> None:
        self.lib.kcmm_cool(self.handle, seq_idx)

    def update_seq_len(self, seq_idx: int, length: int) -> None:
        self.lib.kcmm_update_seq_len(self.handle, seq_idx, length)

    def seq_len(self, seq_idx: int) -> int:
        return self.lib.kcmm_get_seq_len(self.handle, seq_idx)

    def block_table(self, seq_idx: int, max_blocks: int = 1 << 16) -> list[int]:
        out = (ctypes.c_uint32 * max_blocks)()
        count = ctypes.c_uint32()
        self._check(self.lib.kcmm_get_block_table(self.handle, seq_idx, out, max_blocks,
                                                  ctypes.byref(count)),
                    "kcmm_get_block_table")
        return list(out[: count.value])

    def block_table_va_offsets(self, seq_idx: int, max_blocks: int = 1 << 16) -> list[int]:
        out = (ctypes.c_uint64 * max_blocks)()
        count = ctypes.c_uint32()
        self._check(self.lib.kcmm_get_block_table_va_offsets(self.handle, seq_idx, out,
                                                             max_blocks, ctypes.byref(count)),
                    "kcmm_get_block_table_va_offsets")
        return list(out[: count.value])

    def all_block_offsets_f16(self, min_entries: int = 0) -> list[int]:
        n = max(self.total_blocks(), min_entries, 1)
        out = (ctypes.c_uint64 * n)()
        count = ctypes.c_uint32()
        self._check(self.lib.kcmm_get_all_block_offsets_f16(self.handle, out, n,
                                                            ctypes.byref(count)),
                    "kcmm_get_all_block_offsets_f16")
        vals = list(out[: count.value])
        return vals + [0] * (min_entries - len(vals)) if min_entries > len(vals) else vals

    def all_block_valid_flags(self, min_entries: int = 0) -> list[int]:
        n = max(self.total_blocks(), min_entries, 1)
        out = (ctypes.c_uint8 * n)()
        count = ctypes.c_uint32()
        self._check(self.lib.kcmm_get_all_block_valid(self.handle, out, n, ctypes.byref(count)),
                    "kcmm_get_all_block_valid")
        vals = list(out[: count.value])
        return vals + [0] * (min_entries - len(vals)) if min_entries > len(vals) else vals

    def block_va_offset(self, block_idx: int) -> int:
        return self.lib.kcmm_get_block_va_offset(self.handle, block_idx)

    def block_location(self, block_idx: int) -> str:
        loc = ctypes.c_int()
        self._check(self.lib.kcmm_get_block_location(self.handle, block_idx, ctypes.byref(loc)),
                    "kcmm_get_block_location")
        return BlockLocation.name(loc.value)

    def is_gpu_resident(self, block_idx: int) -> bool:
        return bool(self.lib.kcmm_is_gpu_resident(self.handle, block_idx))

    def total_blocks(self) -> int:
        return self.lib.kcmm_total_blocks(self.handle)

    def blocks_in_use(self) -> int:
        return self.lib.kcmm_blocks_in_use(self.handle)

    def free_physical_blocks(self) -> int:
        return self.lib.kcmm_free_physical_blocks(self.handle)

    def active_sequences(self) -> int:
        return self.lib.kcmm_active_sequences(self.handle)

    def block_state_epoch(self) -> int:
        return self.lib.kcmm_block_state_epoch(self.handle)

    def va_k(self, layer: int) -> RegionAddress:
        """Base of a layer's K region, which stays mapped while the address is held."""
        return self._region_address("kcmm_get_va_k", layer)

    def va_v(self, layer: int) -> RegionAddress:
        """Base of a layer's V region, which stays mapped while the address is held."""
        return self._region_address("kcmm_get_va_v", layer)

    def _region_address(self, op: str, layer: int) -> RegionAddress:
        if self._destroyed:
            raise KcmmError(f"{op}: the pool is destroyed")
        va = getattr(self.lib, op)(self.handle, layer)
        if not va:
            raise KcmmError(f"{op}: layer {layer} out of bounds")
        return RegionAddress(va, self._regions)

    def stats(self) -> dict:
        s = KcmmPoolStats()
        self._check(self.lib.kcmm_get_pool_stats(self.handle, ctypes.byref(s)),
                    "kcmm_get_pool_stats")
        return {name: getattr(s, name) for name, _ in s._fields_}

    def metrics(self) -> dict:
        m = KcmmMetrics()
        self._check(self.lib.kcmm_get_metrics(self.handle, ctypes.byref(m)), "kcmm_get_metrics")
        return {name: getattr(m, name) for name, _ in m._fields_}

    def kernel_status(self) -> int:
        """Sticky device diagnostics (bit 0 wait timeout, bit 1 bad offset), then cleared."""
        return self.lib.kcmm_get_kernel_status(self.handle)

    def synchronize(self) -> None:
        self._check(self.lib.kcmm_synchronize(self.handle), "kcmm_synchronize")

    # --- KV append --------------------------------------------------------
    def append_kv_step(self, layer: int, seq_indices, positions, k_src_ptr: int,
                       v_src_ptr: int) -> None:
        n = len(seq_indices)
        self._check(self.lib.kcmm_append_kv_step(self.handle, layer, _u32_array(seq_indices),
                                                 _u32_array(positions), n, k_src_ptr, v_src_ptr),
                    "kcmm_append_kv_step")

    def append_kv_slots(self, layer: int, slot_mapping, k_src_ptr: int, v_src_ptr: int,
                        stream_ptr: int | None = None) -> None:
        n = len(slot_mapping)
        arr = (ctypes.c_int64 * max(1, n))(*[int(s) for s in slot_mapping])
        if stream_ptr is None:
            rc = self.lib.kcmm_append_kv_slots(self.handle, layer, arr, n, k_src_ptr, v_src_ptr)
        else:
            rc = self.lib.kcmm_append_kv_slots_on_stream(self.handle, layer, arr, n, k_src_ptr,
                                                         v_src_ptr, stream_ptr)
        self._check(rc, "kcmm_append_kv_slots")

    def append_kv_device_slots_on_stream(self, layer: int, *, slot_mapping_ptr: int,
                                         block_offsets_f16_ptr: int, valid_blocks_ptr: int,
                                         block_offsets_f16_len: int, batch: int,
                                         k_src_ptr: int, v_src_ptr: int, status_ptr: int,
                                         stream_ptr: int) -> None:
        self._check(self.lib.kcmm_append_kv_device_slots_on_stream(
            self.handle, layer, slot_mapping_ptr, block_offsets_f16_ptr, valid_blocks_ptr,
            block_offsets_f16_len, batch, k_src_ptr, v_src_ptr, status_ptr, stream_ptr),
            "kcmm_append_kv_device_slots_on_stream")

    def fused_norm_rope_append_bf16(self, layer: int, *, x_ptr: int, weight_ptr: int,
                                    normed_ptr: int, hidden: int, eps: float, q_ptr: int,
                                    num_q_heads: int, k_ptr: int, v_ptr: int,
                                    positions_ptr: int, rope_theta: float, rope_mode: int,
                                    slot_mapping_ptr: int, block_offsets_f16_ptr: int,
                                    valid_blocks_ptr: int, block_offsets_f16_len: int,
                                    num_tokens: int, status_ptr: int, stream_ptr: int) -> None:
        self._check(self.lib.kcmm_fused_norm_rope_append_bf16_on_stream(
            self.handle, layer, x_ptr, weight_ptr, normed_ptr, hidden, eps, q_ptr, num_q_heads,
            k_ptr, v_ptr, positions_ptr, rope_theta, rope_mode, slot_mapping_ptr,
            block_offsets_f16_ptr, valid_blocks_ptr, block_offsets_f16_len, num_tokens,
            status_ptr, stream_ptr), "kcmm_fused_norm_rope_append_bf16_on_stream")

    # --- 4-bit cache ---------------------------------------------------------
    def kv4_append(self, layer: int, *, slot_mapping_ptr: int, block_offsets_f16_ptr: int,
                   block_offsets_f16_len: int, num_tokens: int, head_dim: int, k_src_ptr: int,
                   v_src_ptr: int, k_row_stride: int = 0, v_row_stride: int = 0,
                   valid_blocks_ptr: int = 0, status_ptr: int = 0, dtype: str = "bf16",
                   stream_ptr: int = 0) -> None:
        """Quantise rows of K and V into the slots of a 4-bit cache."""
        op = f"kcmm_kv4_append_{dtype}_on_stream"
        self._check(getattr(self.lib, op)(
            self.handle, layer, slot_mapping_ptr, block_offsets_f16_ptr, valid_blocks_ptr,
            block_offsets_f16_len, num_tokens, head_dim, k_src_ptr, k_row_stride, v_src_ptr,
            v_row_stride, status_ptr, stream_ptr), op)

    def kv4_read(self, layer: int, *, slot_mapping_ptr: int, block_offsets_f16_ptr: int,
                 block_offsets_f16_len: int, num_tokens: int, head_dim: int, k_dst_ptr: int,
                 v_dst_ptr: int, k_row_stride: int = 0, v_row_stride: int = 0,
                 valid_blocks_ptr: int = 0, status_ptr: int = 0, dtype: str = "bf16",
                 stream_ptr: int = 0) -> None:
        """The 16-bit values of a 4-bit cache's slots."""
        op = f"kcmm_kv4_read_{dtype}_on_stream"
        self._check(getattr(self.lib, op)(
            self.handle, layer, slot_mapping_ptr, block_offsets_f16_ptr, valid_blocks_ptr,
            block_offsets_f16_len, num_tokens, head_dim, k_dst_ptr, k_row_stride, v_dst_ptr,
            v_row_stride, status_ptr, stream_ptr), op)

    def _decode_weights(self, kind, layer, query_ptr, out_ptr, block_tables_ptr, seq_lens_ptr,
                        block_offsets_f16_ptr, batch, num_q_heads, kv_heads, head_dim, block_size,
                        max_blocks_per_seq, scale, q_stride_token=0, q_stride_head=0,
                        out_stride_token=0, out_stride_head=0, block_tables_row_stride=0,
                        weights_in_ptr=0, weights_out_ptr=0, weights_row_stride=0, dtype="bf16",
                        stream_ptr=0):
        op = f"kcmm_{kind}_{dtype}_on_stream"
        self._check(getattr(self.lib, op)(
            self.handle, layer, query_ptr, q_stride_token, q_stride_head, out_ptr,
            out_stride_token, out_stride_head, block_tables_ptr, block_tables_row_stride,
            seq_lens_ptr, block_offsets_f16_ptr, batch, num_q_heads, kv_heads, head_dim,
            block_size, max_blocks_per_seq, scale, weights_in_ptr, weights_out_ptr,
            weights_row_stride, stream_ptr), op)

    def kv4_paged_attn_decode(self, layer: int, **kw) -> None:
        """Decode attention over a 4-bit cache.  Keywords as `paged_attn_decode` (without
        `noalloc` / `current_context`), optional strides `q_stride_token`, `q_stride_head`,
        `out_stride_token`, `out_stride_head`, `block_tables_row_stride` (0 = dense), and
        optional `weights_in_ptr`, `weights_out_ptr`, `weights_row_stride`."""
        self._decode_weights("kv4_paged_attn_decode", layer, **kw)

    def paged_attn_decode_weights(self, layer: int, **kw) -> None:
        """`kv4_paged_attn_decode` over the 16-bit cache, the weights required."""
        self._decode_weights("paged_attn_decode_weights", layer, **kw)

    # --- eviction by accumulated attention weight -----------------------------
    def evict_tokens(self, layer: int, *, head_dim: int, block_tables_ptr: int,
                     seq_lens_ptr: int, block_offsets_f16_ptr: int, batch: int,
                     max_blocks_per_seq: int, budget: int, sinks: int, recent: int,
                     weights_in_ptr: int, weights_out_ptr: int, weights_row_stride: int,
                     positions_in_ptr: int, positions_out_ptr: int, next_positions_ptr: int,
                     kept_lens_ptr: int, new_lens_ptr: int,
                     cache_format: int = CacheFormat.BITS16, block_tables_row_stride: int = 0,
                     stream_ptr: int = 0) -> None:
        """Cut one layer's cached tokens to `budget` per kv head; `weights_row_stride` is the
        row stride of the positions too.  `truncate_sequence` afterwards."""
        self._check(self.lib.kcmm_evict_tokens_on_stream(
            self.handle, layer, cache_format, head_dim, block_tables_ptr,
            block_tables_row_stride, seq_lens_ptr, block_offsets_f16_ptr, batch,
            max_blocks_per_seq, budget, sinks, recent, weights_in_ptr, weights_out_ptr,
            positions_in_ptr, positions_out_ptr, weights_row_stride, next_positions_ptr,
            kept_lens_ptr, new_lens_ptr, stream_ptr), "kcmm_evict_tokens_on_stream")

    def truncate_sequence(self, seq_idx: int, length: int) -> None:
        self._check(self.lib.kcmm_truncate_sequence(self.handle, seq_idx, length),
                    "kcmm_truncate_sequence")

    # --- rotation and append, attention over packed prompts --------------------
    def rope_append(self, layer: int, *, rope: KcmmRope, head_dim: int, k_ptr: int, v_ptr: int,
                    slot_mapping_ptr: int, block_offsets_f16_ptr: int,
                    block_offsets_f16_len: int, num_tokens: int, num_q_heads: int = 0,
                    q_ptr: int = 0, q_out_ptr: int = 0, k_out_ptr: int = 0,
                    q_stride_token: int = 0, q_stride_head: int = 0,
                    q_out_stride_token: int = 0, q_out_stride_head: int = 0,
                    k_row_stride: int = 0, v_row_stride: int = 0, k_out_row_stride: int = 0,
                    cache_format: int = CacheFormat.BITS16, valid_blocks_ptr: int = 0,
                    status_ptr: int = 0, dtype: str = "bf16", stream_ptr: int = 0) -> None:
        """Rotate q and k by `rope` (`make_rope`) and append k and v to the cache."""
        op = f"kcmm_rope_append_{dtype}_on_stream"
        self._check(getattr(self.lib, op)(
            self.handle, layer, cache_format, head_dim, ctypes.byref(rope), q_ptr, q_stride_token,
            q_stride_head, q_out_ptr, q_out_stride_token, q_out_stride_head, num_q_heads, k_ptr,
            k_row_stride, v_ptr, v_row_stride, k_out_ptr, k_out_row_stride, slot_mapping_ptr,
            block_offsets_f16_ptr, valid_blocks_ptr, block_offsets_f16_len, num_tokens,
            status_ptr, stream_ptr), op)

    def prompt_attn(self, *, query_ptr: int, key_ptr: int, value_ptr: int, out_ptr: int,
                    q_start_ptr: int, k_start_ptr: int, batch: int, num_q_tokens: int,
                    num_k_tokens: int, num_q_heads: int, kv_heads: int, head_dim: int,
                    scale: float, causal: bool = True, q_stride_token: int = 0,
                    q_stride_head: int = 0, k_stride_token: int = 0, k_stride_head: int = 0,
                    v_stride_token: int = 0, v_stride_head: int = 0, out_stride_token: int = 0,
                    out_stride_head: int = 0, dtype: str = "bf16", stream_ptr: int = 0) -> None:
        """Attention of packed sequences over packed K and V rows."""
        op = f"kcmm_prompt_attn_{dtype}_on_stream"
        self._check(getattr(self.lib, op)(
            self.handle, query_ptr, q_stride_token, q_stride_head, key_ptr, k_stride_token,
            k_stride_head, value_ptr, v_stride_token, v_stride_head, out_ptr, out_stride_token,
            out_stride_head, q_start_ptr, k_start_ptr, batch, num_q_tokens, num_k_tokens,
            num_q_heads, kv_heads, head_dim, scale, int(causal), stream_ptr), op)

    # --- beam search -----------------------------------------------------------
    def beam_select(self, *, logits_ptr: int, dtype: str, scores_in_ptr: int, batch: int,
                    beams: int, vocab: int, n_select: int, scores_out_ptr: int,
                    parents_out_ptr: int, tokens_out_ptr: int, row_stride: int = 0, finished_ptr: int = 0, eos_token: int = 0,
                    stream_ptr: int = 0) -> None:
        """The `n_select` best continuations of each request's beams."""
        self._check(self.lib.kcmm_beam_select_on_stream(
            self.handle, logits_ptr, _DTYPES[dtype], row_stride, scores_in_ptr, finished_ptr,
            eos_token, batch, beams, vocab, n_select, scores_out_ptr, parents_out_ptr,
            tokens_out_ptr, stream_ptr), "kcmm_beam_select_on_stream")

    def beam_gather(self, *, src_ptr: int, dst_ptr: int, row_bytes: int, parents_ptr: int,
                    batch: int, beams: int, n_select: int, tokens_ptr: int = 0,
                    token_index: int = 0, stream_ptr: int = 0) -> None:
        """dst row (b, j) = src row (b, parents[b][j])."""
        self._check(self.lib.kcmm_beam_gather_on_stream(
            self.handle, src_ptr, dst_ptr, row_bytes, parents_ptr, batch, beams, n_select,
            tokens_ptr, token_index, stream_ptr), "kcmm_beam_gather_on_stream")

    def reorder_sequences(self, seq_indices, parents, stream_ptr: int = 0) -> None:
        """seq_indices[i] continues what seq_indices[parents[i]] holds now."""
        if len(parents) != len(seq_indices):
            raise ValueError(f"{len(seq_indices)} sequences have {len(parents)} parents")
        self._check(self.lib.kcmm_reorder_sequences_on_stream(
            self.handle, _u32_array(seq_indices), _u32_array(parents), len(seq_indices),
            stream_ptr), "kcmm_reorder_sequences_on_stream")

    # --- decode attention --------------------------------------------------
    def paged_attn_decode(self, layer: int, *, query_ptr: int, out_ptr: int,
                          block_tables_ptr: int, seq_lens_ptr: int,
                          block_offsets_f16_ptr: int, batch: int, num_q_heads: int,
                          kv_heads: int, head_dim: int, block_size: int,
                          max_blocks_per_seq: int, scale: float, dtype: str = "bf16",
                          stream_ptr: int | None = 0, current_context: bool = False,
                          noalloc: bool = False) -> None:
        """`noalloc=True` (bf16 only) calls the entry point whose scratch is a static
        per-device array instead of a stream-ordered allocation."""
        args = (self.handle, layer, query_ptr, out_ptr, block_tables_ptr, seq_lens_ptr,
                block_offsets_f16_ptr, batch, num_q_heads, kv_heads, head_dim, block_size,
                max_blocks_per_seq, scale)
        if noalloc:
            if dtype != "bf16":
                raise ValueError("the no-allocation decode entry point is bf16 only")
            rc = self.lib.kcmm_paged_attn_decode_bf16_noalloc_on_stream(*args, stream_ptr or 0)
            op = "kcmm_paged_attn_decode_bf16_noalloc_on_stream"
        elif dtype == "bf16":
            rc = self.lib.kcmm_paged_attn_decode_bf16_on_stream(*args, stream_ptr or 0)
            op = "kcmm_paged_attn_decode_bf16_on_stream"
        elif stream_ptr is None:
            rc = self.lib.kcmm_paged_attn_decode_f16(*args)
            op = "kcmm_paged_attn_decode_f16"
        elif current_context:
            rc = self.lib.kcmm_paged_attn_decode_f16_on_current_context_stream(*args, stream_ptr)
            op = "kcmm_paged_attn_decode_f16_on_current_context_stream"
        else:
            rc = self.lib.kcmm_paged_attn_decode_f16_on_stream(*args, stream_ptr)
            op = "kcmm_paged_attn_decode_f16_on_stream"
        self._check(rc, op)

    def paged_prefill(self, layer: int, *, query_ptr: int, out_ptr: int, block_tables_ptr: int,
                      query_start_loc_ptr: int, context_lens_ptr: int,
                      block_offsets_f16_ptr: int, batch: int, max_query_len: int,
                      num_q_heads: int, kv_heads: int, head_dim: int, block_size: int,
                      max_blocks_per_seq: int, scale: float, dtype: str = "bf16",
                      stream_ptr: int = 0) -> None:
        op = f"kcmm_paged_prefill_{dtype}_on_stream"
        fn = getattr(self.lib, op)
        self._check(fn(self.handle, layer, query_ptr, out_ptr, block_tables_ptr,
                       query_start_loc_ptr, context_lens_ptr, block_offsets_f16_ptr, batch,
                       max_query_len, num_q_heads, kv_heads, head_dim, block_size,
                       max_blocks_per_seq, scale, stream_ptr), op)

    def precompile_paged_attn_decode_f16(self) -> None:
        self._check(self.lib.kcmm_precompile_paged_attn_decode_f16(self.handle),
                    "kcmm_precompile_paged_attn_decode_f16")

    def precompile_vllm_kv_write_f16(self) -> None:
        self._check(self.lib.kcmm_precompile_vllm_kv_write_f16(self.handle),
                    "kcmm_precompile_vllm_kv_write_f16")

    # --- sharing / copy-on-write ------------------------------------------
    def incref(self, block_idx: int) -> None:
        self._check(self.lib.kcmm_block_incref(self.handle, block_idx), "kcmm_block_incref")

    def decref(self, block_idx: int) -> None:
        self._check(self.lib.kcmm_block_decref(self.handle, block_idx), "kcmm_block_decref")

    def refcount(self, block_idx: int) -> int:
        return self.lib.kcmm_block_refcount(self.handle, block_idx)

    def fork_sequence(self, src_seq: int) -> int:
        out = ctypes.c_uint32()
        self._check(self.lib.kcmm_fork_sequence(self.handle, src_seq, ctypes.byref(out)),
                    "kcmm_fork_sequence")
        return out.value

    def share_prefix(self, src_seq: int, dst_seq: int, num_blocks: int) -> list[int]:
        out = (ctypes.c_uint32 * max(1, num_blocks))()
        self._check(self.lib.kcmm_share_prefix(self.handle, src_seq, dst_seq, num_blocks, out),
                    "kcmm_share_prefix")
        return list(out[:num_blocks])

    def cow_blocks(self, seq_indices, logical_blocks, stream_ptr: int = 0) -> list[int]:
        n = len(seq_indices)
        out = (ctypes.c_uint32 * max(1, n))()
        self._check(self.lib.kcmm_cow_blocks_on_stream(self.handle, _u32_array(seq_indices),
                                                       _u32_array(logical_blocks), n, out,
                                                       stream_ptr),
                    "kcmm_cow_blocks_on_stream")
        return list(out[:n])

    # --- tiering -------------------------------------------------------------
    def evict_blocks(self, count: int) -> int:
        return self.lib.kcmm_evict_blocks(self.handle, count)

    def restore_evicted_block(self, block_idx: int) -> int:
        va = self.lib.kcmm_restore_evicted_block(self.handle, block_idx)
        if va == 0 and self.last_error():
            raise KcmmError(f"kcmm_restore_evicted_block failed: {self.last_error()}")
        return va

    def restore_evicted_blocks(self, blocks) -> None:
        self._check(self.lib.kcmm_restore_evicted_blocks(self.handle, _u32_array(blocks),
                                                         len(blocks)),
                    "kcmm_restore_evicted_blocks")

    def swap_out(self, blocks, stream_ptr: int = 0) -> None:
        self._check(self.lib.kcmm_swap_out_blocks_on_stream(self.handle, _u32_array(blocks),
                                                            len(blocks), stream_ptr),
                    "kcmm_swap_out_blocks_on_stream")

    def swap_in(self, blocks, stream_ptr: int = 0) -> None:
        self._check(self.lib.kcmm_swap_in_blocks_on_stream(self.handle, _u32_array(blocks),
                                                           len(blocks), stream_ptr),
                    "kcmm_swap_in_blocks_on_stream")

    def metrics_ext(self) -> dict:
        m = KcmmMetricsExt()
        self._check(self.lib.kcmm_get_metrics_ext(self.handle, ctypes.byref(m)),
                    "kcmm_get_metrics_ext")

        def hist(h):
            return {"count": h.count, "sum_us": h.sum_us, "min_us": h.min_us,
                    "max_us": h.max_us, "buckets": list(h.buckets)}
        out = {name: getattr(m.base, name) for name, _ in m.base._fields_}
        out.update({name: getattr(m, name) for name, _ in m._fields_[1:6]})
        out["eviction_latency"] = hist(m.eviction_latency)
        out["restoration_latency"] = hist(m.restoration_latency)
        return out

    def policy_stats(self, policy: str) -> dict | None:
        st = KcmmPolicyStats()
        if self.lib.kcmm_get_policy_stats(self.handle, policy.encode(), ctypes.byref(st)) != 0:
            return None
        return {name: getattr(st, name) for name, _ in st._fields_}

    def start_background_eviction(self) -> None:
        self._check(self.lib.kcmm_start_background_eviction(self.handle),
                    "kcmm_start_background_eviction")

    def stop_background_eviction(self) -> None:
        self._check(self.lib.kcmm_stop_background_eviction(self.handle),
                    "kcmm_stop_background_eviction")

    def preview_eviction_victims(self, count: int) -> list[int]:
        buf = (ctypes.c_uint32 * max(1, count))()
        n = self.lib.kcmm_preview_eviction_victims(self.handle, count, buf, max(1, count))
        return list(buf[:n])

    def set_eviction_policy(self, name: str) -> None:
        self._check(self.lib.kcmm_set_eviction_policy(self.handle, name.encode()),
                    "kcmm_set_eviction_policy")

    def eviction_policy(self) -> str:
        buf = ctypes.create_string_buffer(64)
        self.lib.kcmm_get_eviction_policy(self.handle, buf, 64)
        return buf.value.decode()
