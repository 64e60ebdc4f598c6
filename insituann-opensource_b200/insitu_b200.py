"""Python binding of libinsitu_b200.so (ctypes over the C ABI in include/insitu_b200.h).

The objects mirror the reference's host API for the IVF query path:
``Index`` is IVFIndexContext, ``Batch`` is IVFQueryBatchContext
(cuda/search/ivf_search_separated.cu:31-93), ``Batch.stage1_prepare`` /
``stage2_compute`` / ``get_results`` are the pipeline stages of
cuda/search/ivf_search.cuh:276-327 and ``CoarseRouter`` wraps the
CoarseHandle / coarse_search routing API of cuda/search/cpu_fine/cpu_fine.h:232-278.

There is no CPU fallback: every search runs in the CUDA library, and the
module raises if the library or a CUDA device is missing.
"""
from __future__ import annotations

import ctypes as C
import os
from typing import Optional

import numpy as np

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(HERE, "libinsitu_b200.so")

IVF_OK = 0
ERRORS = {-1: "EINVAL", -2: "ECUDA", -3: "ESTATE", -4: "ENOMEM", -5: "EOVERFLOW", -6: "EUNSUPPORTED"}

# every exported symbol, as declared in include/insitu_b200.h and include/cuda_wrapper.h
EXPORTS = [
    "ivf_create_index_context", "ivf_destroy_index_context", "ivf_load_dataset", "ivf_create_batch_context",
    "ivf_destroy_batch_context", "ivf_pipeline_stage1_prepare", "ivf_pipeline_stage2_compute",
    "ivf_pipeline_get_results", "ivf_pipeline_sync_batch",
    "ivf_create_index_context_wrapper", "ivf_destroy_index_context_wrapper", "ivf_load_dataset_wrapper",
    "ivf_create_batch_context_wrapper", "ivf_destroy_batch_context_wrapper",
    "ivf_pipeline_stage1_prepare_wrapper", "ivf_pipeline_stage2_compute_wrapper",
    "ivf_pipeline_get_results_wrapper", "ivf_pipeline_sync_batch_wrapper", "ivf_check_index_initialized_wrapper",
    "ivf_register_index_instance", "ivf_get_index_instance", "ivf_unregister_index_instance",
    "coarse_handle_init", "coarse_handle_release", "coarse_search", "coarse_get_last_timing",
    "ivf_u8_load", "ivf_pq_load", "ivf_set_shard", "ivf_pq_publish_delta", "ivf_pq_clear_delta",
    "ivf_pq_delta_mode",
    "ivf_route", "ivf_set_probes", "ivf_get_probes", "ivf_u8_search", "ivf_pq_search", "ivf_get_results_i32",
    "ivf_pipeline_stage1_prepare_device", "ivf_get_results_device", "ivf_batch_stream",
    "ivf_route_keys", "ivf_route_merge", "ivf_route_merge_shards", "ivf_set_deleted", "ivf_pq_search_shard", "ivf_pq_merge_shards",
    "ivf_u8_search_shard", "ivf_u8_merge_shards", "ivf_pq_shard_scan", "ivf_pq_shard_bounds",
    "ivf_pq_shard_select", "ivf_pq_shard_kappa", "ivf_pq_shard_rerank", "ivf_pq_shard_final",
    "ivf_last_error", "ivf_global_last_error",
    "ivf_kernel_launches", "ivf_batch_profile", "ivf_batch_stage_ms", "ivf_u8_search_noalloc",
    "ivf_load_centroids", "ivf_assign", "ivf_build_reorder", "ivf_kmeans_update", "ivf_pq_train", "ivf_pq_encode",
    "ivf_sq_write", "ivf_sq_read", "ivf_sq_matmul", "ivf_sq_matmul_work", "ivf_sq_scores",
    "ivf_sq_scores_work", "ivf_sq_status",
    "ivf_read_centroids", "ivf_read_assign", "ivf_read_codebook", "ivf_read_codes", "ivf_read_u8bin",
    "ivf_read_fbin", "ivf_read_gt", "ivf_write_centroids", "ivf_write_assign", "ivf_write_codebook",
    "ivf_write_codes", "ivf_pq_load_files", "ivf_pq_insert",
    "cuda_is_available", "cuda_malloc", "cuda_alloc_pinned", "cuda_free_pinned", "cuda_free", "cuda_memcpy_h2d",
    "cuda_memcpy_d2h", "cuda_memcpy_async_h2d", "cuda_memcpy_async_d2h", "cuda_cleanup_memory",
    "cuda_pipeline_init", "cuda_pipeline_flush", "cuda_pipeline_flush_vectors_only", "cuda_pipeline_free",
    "cuda_device_synchronize", "cuda_get_last_error_string", "cuda_check_last_error",
]

vp = C.c_void_p
i32 = C.c_int
i64 = C.c_longlong

_SIGS = {
    "ivf_create_index_context": ([], vp),
    "ivf_destroy_index_context": ([vp], None),
    "ivf_load_dataset": ([vp, vp, vp, vp, i32, i32, i32], i32),
    "ivf_create_batch_context": ([i32, i32, i32, i32, i32], vp),
    "ivf_destroy_batch_context": ([vp], None),
    "ivf_pipeline_stage1_prepare": ([vp, vp, i32], None),
    "ivf_pipeline_stage2_compute": ([vp, vp, i32, i32, i32, i32], None),
    "ivf_pipeline_get_results": ([vp, vp, vp, i32, i32], None),
    "ivf_pipeline_sync_batch": ([vp], None),
    "ivf_check_index_initialized_wrapper": ([vp], i32),
    "ivf_register_index_instance": ([C.c_uint, vp], None),
    "ivf_get_index_instance": ([C.c_uint], vp),
    "ivf_unregister_index_instance": ([C.c_uint], None),
    "coarse_handle_init": ([vp, vp, i32, i32], None),
    "coarse_handle_release": ([vp], None),
    "coarse_search": ([vp, vp, i32, i32, i32, vp, vp, vp, vp], None),
    "coarse_get_last_timing": ([], vp),
    "ivf_u8_load": ([vp, vp, vp, vp, vp, vp, i32, i64, i32], i32),
    "ivf_pq_load": ([vp, vp, vp, i32, i32, i32, vp, vp, vp, vp, vp, vp, i32, i64, i32], i32),
    "ivf_set_shard": ([vp, i32, vp, vp], i32),
    "ivf_pq_publish_delta": ([vp, vp, vp, vp, vp, vp, vp, vp, i64], i32),
    "ivf_pq_clear_delta": ([vp], i32),
    "ivf_pq_delta_mode": ([vp], i32),
    "ivf_route": ([vp, vp, i32, i32], i32),
    "ivf_set_probes": ([vp, vp, i32, i32], i32),
    "ivf_get_probes": ([vp, vp, i32, i32], i32),
    "ivf_u8_search": ([vp, vp, i32, i32, i32, i32], i32),
    "ivf_pq_search": ([vp, vp, i32, i32, i32, i32, i32, i32, i32], i32),
    "ivf_get_results_i32": ([vp, vp, vp, i32, i32], i32),
    "ivf_pipeline_stage1_prepare_device": ([vp, vp, i32], i32),
    "ivf_get_results_device": ([vp, vp, vp, i32, i32], i32),
    "ivf_batch_stream": ([vp], vp),
    "ivf_route_keys": ([vp, vp, i32, i32, vp], i32),
    "ivf_route_merge": ([vp, vp, i32, i32, i32], i32),
    "ivf_route_merge_shards": ([vp, vp, i32, i32, i32], i32),
    "ivf_set_deleted": ([vp, vp, i64], i32),
    "ivf_pq_search_shard": ([vp, vp, i32, i32, i32, i32, vp, vp, vp, vp], i32),
    "ivf_pq_merge_shards": ([vp, vp, vp, i32, i32, vp, vp, i32, i32, i32, i32, i32], i32),
    "ivf_u8_search_shard": ([vp, vp, i32, i32, i32, vp], i32),
    "ivf_u8_merge_shards": ([vp, vp, i32, i32, i32], i32),
    "ivf_pq_shard_scan": ([vp, vp, i32, i32, i32, i32], i32),
    "ivf_pq_shard_bounds": ([vp], vp),
    "ivf_pq_shard_select": ([vp, vp, i32, i32, i32, vp], i32),
    "ivf_pq_shard_kappa": ([vp, vp, i32, i32, i32, vp], i32),
    "ivf_pq_shard_rerank": ([vp, vp, i32, i32, vp, vp, i32, vp], i32),
    "ivf_pq_shard_final": ([vp, vp, i32, i32, i32, i32], i32),
    "ivf_last_error": ([vp], C.c_char_p),
    "ivf_global_last_error": ([], C.c_char_p),
    "cuda_is_available": ([], C.c_bool),
    "ivf_kernel_launches": ([], C.c_ulonglong),
    "ivf_batch_profile": ([vp, i32], i32),
    "ivf_batch_stage_ms": ([vp, vp, i32], i32),
    "ivf_u8_search_noalloc": ([vp, vp, vp, i32, i32, i32, vp, vp, vp], i32),
    "ivf_load_centroids": ([vp, vp, i32, i32], i32),
    "ivf_assign": ([vp, vp, vp, i32, i64, vp], i32),
    "ivf_build_reorder": ([vp, i64, i32, vp, vp, vp, vp], i32),
    "ivf_kmeans_update": ([vp, i32, i64, i32, vp, i32, vp, vp], i32),
    "ivf_pq_train": ([vp, i32, i64, i32, vp, vp, i32, i32, vp, vp], i32),
    "ivf_pq_encode": ([vp, i32, i64, i32, vp, vp, vp, vp, i32, vp, vp], i32),
    "ivf_sq_write": ([vp, i32, i64, i32, i64, vp, i32, i32, vp, i64, vp, i64, i64, vp, vp], i32),
    "ivf_sq_read": ([vp, i64, vp, i64, i64, i32, i32, vp, i64, i32, vp, i32, i64, vp], i32),
    "ivf_sq_matmul": ([vp, i64, vp, i64, vp, i64, vp, i64, i32, vp, vp, i32, i64, vp, C.c_size_t, vp], i32),
    "ivf_sq_matmul_work": ([vp, i64, i64, vp, i64, i64, i32], C.c_size_t),
    "ivf_sq_scores": ([vp, i32, i64, i64, vp, i64, vp, i64, i32, vp, vp, i32, i64, vp, C.c_size_t, vp], i32),
    "ivf_sq_scores_work": ([i64, vp, i64, i64, i32], C.c_size_t),
    "ivf_sq_status": ([vp], i32),
    "ivf_read_centroids": ([C.c_char_p, vp, i64, vp, vp], i64),
    "ivf_read_assign": ([C.c_char_p, vp, i64, vp], i64),
    "ivf_read_codebook": ([C.c_char_p, vp, i64, vp, vp, vp], i64),
    "ivf_read_codes": ([C.c_char_p, vp, i64, vp, vp], i64),
    "ivf_read_u8bin": ([C.c_char_p, vp, i64, vp, vp], i64),
    "ivf_read_fbin": ([C.c_char_p, vp, i64, vp, vp], i64),
    "ivf_read_gt": ([C.c_char_p, vp, i64, vp, vp], i64),
    "ivf_write_centroids": ([C.c_char_p, vp, i32, i32], i32),
    "ivf_write_assign": ([C.c_char_p, vp, i64], i32),
    "ivf_write_codebook": ([C.c_char_p, vp, i32, i32, i32], i32),
    "ivf_write_codes": ([C.c_char_p, vp, i64, i32], i32),
    "ivf_pq_load_files": ([vp, C.c_char_p, C.c_char_p, C.c_char_p, C.c_char_p, C.c_char_p], i32),
    "ivf_pq_insert": ([vp, vp, i32, vp, i64], i32),
}

_SQ_SCAN_ROWS = 512      # IVF_SQ_SCAN_ROWS

STAGES = ("route", "worklist", "scan", "select", "rerank")

_lib = None


class InsituError(RuntimeError):
    def __init__(self, code: int, msg: str):
        super().__init__(f"{ERRORS.get(code, code)}: {msg}")
        self.code = code


def library_path() -> str:
    return LIB_PATH


def kernel_launches() -> int:
    """kernels launched by libinsitu_b200 in this process so far"""
    return int(load_library().ivf_kernel_launches())


def load_library(require_device: bool = False):
    """Loads libinsitu_b200.so (raises when it was not built)."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise RuntimeError(f"{LIB_PATH} is missing: build it with `make -C {HERE}`")
        L = C.CDLL(LIB_PATH)
        for name, (args, res) in _SIGS.items():
            fn = getattr(L, name)
            fn.argtypes = args
            fn.restype = res
        _lib = L
    if require_device and not _lib.cuda_is_available():
        raise RuntimeError("libinsitu_b200 needs a CUDA device; none is visible")
    return _lib


def _p(a) -> Optional[int]:
    """Address of a numpy array or of a torch tensor's data (None passes NULL)."""
    if a is None:
        return None
    if hasattr(a, "data_ptr"):
        return a.data_ptr()
    return a.ctypes.data


_TORCH_DT = {np.uint8: "uint8", np.int32: "int32", np.int64: "int64", np.float32: "float32"}


def _c(a, dt):
    """C-contiguous array of dtype dt; torch tensors (host or device) stay torch tensors."""
    if a is None:
        return None
    if hasattr(a, "data_ptr"):
        import torch

        t = a.to(getattr(torch, _TORCH_DT[dt]))
        return t.contiguous()
    return np.ascontiguousarray(a, dtype=dt)


class Index:
    """Device-resident IVF index (uint8 exact or residual PQ)."""

    def __init__(self):
        self.L = load_library(require_device=True)
        self.h = self.L.ivf_create_index_context()
        if not self.h:
            raise InsituError(-4, self.L.ivf_global_last_error().decode())
        self.kind = None
        self.d = None

    def _check(self, rc):
        if rc != IVF_OK:
            raise InsituError(rc, self.L.ivf_last_error(self.h).decode())

    def load_u8(self, base_u8, offsets, counts, reorder_to_original, centroids):
        base_u8 = _c(base_u8, np.uint8)
        n, d = base_u8.shape
        offsets, counts = _c(offsets, np.int64), _c(counts, np.int32)
        r2o = _c(reorder_to_original, np.int32)
        cent = _c(centroids, np.float32)
        self._check(self.L.ivf_u8_load(self.h, _p(base_u8), _p(offsets), _p(counts), _p(r2o), _p(cent),
                                       counts.shape[0], n, d))
        self.kind, self.d, self.nlist = "u8", d, counts.shape[0]
        return self

    def load_pq(self, centroids, codebook, codes, offsets, counts, reorder_to_original, base_u8=None,
                base_f32=None):
        cent = _c(centroids, np.float32)
        cb = _c(codebook, np.float32)
        M, K, dsub = cb.shape
        codes = _c(codes, np.uint8)
        offsets, counts = _c(offsets, np.int64), _c(counts, np.int32)
        r2o = _c(reorder_to_original, np.int32)
        bu, bf = _c(base_u8, np.uint8), _c(base_f32, np.float32)
        n = codes.shape[0]
        d = cent.shape[1]
        self._check(self.L.ivf_pq_load(self.h, _p(cent), _p(cb), M, K, dsub, _p(codes), _p(offsets), _p(counts),
                                       _p(r2o), _p(bu), _p(bf), counts.shape[0], n, d))
        self.kind, self.d, self.nlist, self.f32 = "pq", d, counts.shape[0], bf is not None
        return self

    def load_pq_files(self, centroids_path, codebook_path, codes_path, assign_path, base_u8bin_path):
        """a residual-PQ index from the reference's files (ivf_pq_load_files)"""
        self._check(self.L.ivf_pq_load_files(self.h, centroids_path.encode(), codebook_path.encode(),
                                             codes_path.encode(), assign_path.encode(), base_u8bin_path.encode()))
        self.kind = "pq"
        return self

    def set_shard(self, nlist_global, local_to_global, key_offsets=None):
        l2g = _c(local_to_global, np.int32)
        ko = _c(key_offsets, np.int64)
        self._check(self.L.ivf_set_shard(self.h, nlist_global, _p(l2g), _p(ko)))
        return self

    def publish_delta(self, codes, ids, counts, offsets, raw_u8=None, raw_f32=None, key_offsets=None):
        codes = _c(codes, np.uint8)
        ids = _c(ids, np.int32)
        counts, offsets = _c(counts, np.int32), _c(offsets, np.int64)
        ko = _c(key_offsets, np.int64)
        ru, rf = _c(raw_u8, np.uint8), _c(raw_f32, np.float32)
        self._check(self.L.ivf_pq_publish_delta(self.h, _p(codes), _p(ids), _p(counts), _p(offsets), _p(ko),
                                                _p(ru), _p(rf), codes.shape[0]))
        return self

    def clear_delta(self):
        self._check(self.L.ivf_pq_clear_delta(self.h))

    def delta_mode(self):
        """how the published delta is searched: None, "direct", "mix" or "seg" (ivf_pq_delta_mode)"""
        r = self.L.ivf_pq_delta_mode(self.h)
        if r < 0:
            self._check(r)
        return [None, "direct", "mix", "seg"][r]

    def insert(self, rows, ids):
        """online insert of device rows (torch uint8 / float32 [n, d]) with ids (int32 [n]) into the delta"""
        import torch

        rows = rows.contiguous()
        ids = np.ascontiguousarray(ids, dtype=np.int32)
        self._check(self.L.ivf_pq_insert(self.h, rows.data_ptr(), 1 if rows.dtype == torch.uint8 else 0, _p(ids),
                                         rows.shape[0]))
        return self

    def set_deleted(self, deleted=None):
        """per-position delete mask (uint8 [n], nonzero = deleted), or None to clear it."""
        m = None if deleted is None else _c(deleted, np.uint8)
        self._check(self.L.ivf_set_deleted(self.h, _p(m), 0 if m is None else m.shape[0]))
        return self

    def close(self):
        if self.h:
            self.L.ivf_destroy_index_context(self.h)
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class Batch:
    """One query batch: a CUDA stream plus scratch (IVFQueryBatchContext)."""

    def __init__(self, max_nq, d, max_nprobe, max_k, nlist):
        self.L = load_library(require_device=True)
        self.h = self.L.ivf_create_batch_context(max_nq, d, max_nprobe, max_k, nlist)
        if not self.h:
            raise InsituError(-4, self.L.ivf_global_last_error().decode())
        self.d = d

    def _check(self, rc):
        if rc != IVF_OK:
            raise InsituError(rc, self.L.ivf_last_error(self.h).decode())

    def last_error(self) -> str:
        return self.L.ivf_last_error(self.h).decode()

    @property
    def stream(self) -> int:
        return self.L.ivf_batch_stream(self.h) or 0

    # ---- reference pipeline ----
    def stage1_prepare(self, q_host):
        """q_host must stay alive until the stream has consumed it (sync or get_results)."""
        self._q_keep = _c(q_host, np.float32)
        self.L.ivf_pipeline_stage1_prepare(self.h, _p(self._q_keep), self._q_keep.shape[0])
        self._raise_if_error()

    def stage1_prepare_ptr(self, host_ptr: int, nq: int):
        self.L.ivf_pipeline_stage1_prepare(self.h, host_ptr, nq)
        self._raise_if_error()

    def stage1_prepare_device(self, d_ptr: int, nq: int):
        self._check(self.L.ivf_pipeline_stage1_prepare_device(self.h, d_ptr, nq))

    def stage2_compute(self, index: Index, nq, nprobe, k, distance_mode=0):
        self.L.ivf_pipeline_stage2_compute(self.h, index.h, nq, nprobe, k, distance_mode)
        self._raise_if_error()

    def get_results(self, nq, k):
        dist = np.empty((nq, k), np.float32)
        ids = np.empty((nq, k), np.int32)
        self.L.ivf_pipeline_get_results(self.h, _p(dist), _p(ids), nq, k)
        self._raise_if_error()
        return ids, dist

    def get_results_into(self, dist_ptr: int, ids_ptr: int, nq, k):
        self.L.ivf_pipeline_get_results(self.h, dist_ptr, ids_ptr, nq, k)
        self._raise_if_error()

    def get_results_i32(self, nq, k):
        dist = np.empty((nq, k), np.int32)
        ids = np.empty((nq, k), np.int32)
        self._check(self.L.ivf_get_results_i32(self.h, _p(ids), _p(dist), nq, k))
        return ids, dist

    def get_results_device(self, d_dist: int, d_ids: int, nq, k):
        self._check(self.L.ivf_get_results_device(self.h, d_dist, d_ids, nq, k))

    def sync(self):
        self.L.ivf_pipeline_sync_batch(self.h)
        self._raise_if_error()

    def _raise_if_error(self):
        msg = self.last_error()
        if msg:
            raise InsituError(-1, msg)

    # ---- observability ----
    def profile(self, enable=True):
        self._check(self.L.ivf_batch_profile(self.h, 1 if enable else 0))

    def stage_ms(self) -> dict:
        out = np.zeros(len(STAGES), np.float64)
        rc = self.L.ivf_batch_stage_ms(self.h, _p(out), len(STAGES))
        if rc < 0:
            self._check(rc)
        return dict(zip(STAGES, out.tolist()))

    # ---- explicit entry points ----
    def route(self, index: Index, nq, nprobe):
        self._check(self.L.ivf_route(self.h, index.h, nq, nprobe))

    def set_probes(self, probes):
        probes = _c(probes, np.int32)
        self._probes_keep = probes
        self._check(self.L.ivf_set_probes(self.h, _p(probes), probes.shape[0], probes.shape[1]))

    def get_probes(self, nq, nprobe):
        out = np.empty((nq, nprobe), np.int32)
        self._check(self.L.ivf_get_probes(self.h, _p(out), nq, nprobe))
        return out

    def u8_search(self, index: Index, nq, nprobe, k, route=True):
        self._check(self.L.ivf_u8_search(self.h, index.h, nq, nprobe, k, 1 if route else 0))

    def pq_search(self, index: Index, nq, nprobe, k, rerank_n=512, overlay=True, delta_topk=16, route=True):
        self._check(self.L.ivf_pq_search(self.h, index.h, nq, nprobe, k, rerank_n, 1 if overlay else 0,
                                         delta_topk, 1 if route else 0))

    # ---- shard exchange (device pointers) ----
    def route_keys(self, index: Index, nq, nprobe, d_keys: int):
        self._check(self.L.ivf_route_keys(self.h, index.h, nq, nprobe, d_keys))

    def route_merge(self, d_keys: int, n_in, nq, nprobe):
        self._check(self.L.ivf_route_merge(self.h, d_keys, n_in, nq, nprobe))

    def route_merge_shards(self, d_keys: int, n_shards, nq, nprobe):
        """d_keys: the shards' sorted routing keys as all-gathered, [n_shards][nq][nprobe]."""
        self._check(self.L.ivf_route_merge_shards(self.h, d_keys, n_shards, nq, nprobe))

    def pq_search_shard(self, index: Index, nq, nprobe, rerank_n, delta_topk, d_adc, d_exact, d_dadc=None,
                        d_dexact=None):
        self._check(self.L.ivf_pq_search_shard(self.h, index.h, nq, nprobe, rerank_n, delta_topk, d_adc, d_exact,
                                               d_dadc, d_dexact))

    def pq_merge_shards(self, d_adc, d_exact, n_main, rerank_n, d_dadc, d_dexact, n_delta, delta_topk, nq, k,
                        exact_is_int):
        self._check(self.L.ivf_pq_merge_shards(self.h, d_adc, d_exact, n_main, rerank_n, d_dadc, d_dexact, n_delta,
                                               delta_topk, nq, k, 1 if exact_is_int else 0))

    # phased sharded PQ search (see the header): device pointers as ints
    def pq_shard_scan(self, index: Index, nq, nprobe, rerank_n, pass_):
        self._check(self.L.ivf_pq_shard_scan(self.h, index.h, nq, nprobe, rerank_n, pass_))

    def pq_shard_bounds(self) -> int:
        """device address of the [nq] int64 rank-R bounds"""
        return int(self.L.ivf_pq_shard_bounds(self.h) or 0)

    def pq_shard_select(self, index: Index, nq, nprobe, rerank_n, d_adc):
        self._check(self.L.ivf_pq_shard_select(self.h, index.h, nq, nprobe, rerank_n, d_adc))

    def pq_shard_kappa(self, d_adc_all, n_shards, n_owned, rerank_n, d_kappa):
        """owner: d_adc_all [n_shards][n_owned][R] -> d_kappa [n_owned], the R-th smallest key of the union"""
        self._check(self.L.ivf_pq_shard_kappa(self.h, d_adc_all, n_shards, n_owned, rerank_n, d_kappa))

    def pq_shard_rerank(self, index: Index, nq, rerank_n, d_adc, d_kappa, k, d_topk):
        """this shard's exact top-k [nq, k] (keys) of its stage-1 keys <= d_kappa[q]"""
        self._check(self.L.ivf_pq_shard_rerank(self.h, index.h, nq, rerank_n, d_adc, d_kappa, k, d_topk))

    def pq_shard_final(self, d_topk_all, n_shards, n_owned, k, exact_is_int):
        """owner: d_topk_all [n_shards][n_owned][k] -> the batch results of its n_owned queries"""
        self._check(self.L.ivf_pq_shard_final(self.h, d_topk_all, n_shards, n_owned, k, 1 if exact_is_int else 0))

    def u8_search_shard(self, index: Index, nq, nprobe, k, d_keys):
        self._check(self.L.ivf_u8_search_shard(self.h, index.h, nq, nprobe, k, d_keys))

    def u8_merge_shards(self, d_keys, n_in, nq, k):
        self._check(self.L.ivf_u8_merge_shards(self.h, d_keys, n_in, nq, k))

    def close(self):
        if self.h:
            self.L.ivf_destroy_batch_context(self.h)
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


# ---- the reference's index file formats (host code, no device needed) ----
def _err(L):
    return L.ivf_global_last_error().decode()


def read_centroids(path):
    L = load_library()
    nl, d = C.c_int(0), C.c_int(0)
    if L.ivf_read_centroids(path.encode(), None, 0, C.byref(nl), C.byref(d)) < 0:
        raise InsituError(-1, _err(L))
    out = np.empty((nl.value, d.value), np.float32)
    if L.ivf_read_centroids(path.encode(), _p(out), out.size, C.byref(nl), C.byref(d)) < 0:
        raise InsituError(-1, _err(L))
    return out


def read_assign(path):
    L = load_library()
    n = C.c_longlong(0)
    if L.ivf_read_assign(path.encode(), None, 0, C.byref(n)) < 0:
        raise InsituError(-1, _err(L))
    out = np.empty(n.value, np.int32)
    if L.ivf_read_assign(path.encode(), _p(out), out.size, C.byref(n)) < 0:
        raise InsituError(-1, _err(L))
    return out


def read_codebook(path):
    L = load_library()
    M, K, ds = C.c_int(0), C.c_int(0), C.c_int(0)
    if L.ivf_read_codebook(path.encode(), None, 0, C.byref(M), C.byref(K), C.byref(ds)) < 0:
        raise InsituError(-1, _err(L))
    out = np.empty((M.value, K.value, ds.value), np.float32)
    if L.ivf_read_codebook(path.encode(), _p(out), out.size, C.byref(M), C.byref(K), C.byref(ds)) < 0:
        raise InsituError(-1, _err(L))
    return out


def read_codes(path):
    L = load_library()
    n, M = C.c_longlong(0), C.c_int(0)
    if L.ivf_read_codes(path.encode(), None, 0, C.byref(n), C.byref(M)) < 0:
        raise InsituError(-1, _err(L))
    out = np.empty((n.value, M.value), np.uint8)
    if L.ivf_read_codes(path.encode(), _p(out), out.size, C.byref(n), C.byref(M)) < 0:
        raise InsituError(-1, _err(L))
    return out


def read_bin(path, dtype=np.uint8):
    """DiskANN u8bin (dtype uint8) or fbin (float32) [n, d]"""
    L = load_library()
    n, d = C.c_longlong(0), C.c_int(0)
    fn = L.ivf_read_u8bin if dtype == np.uint8 else L.ivf_read_fbin
    if fn(path.encode(), None, 0, C.byref(n), C.byref(d)) < 0:
        raise InsituError(-1, _err(L))
    out = np.empty((n.value, d.value), dtype)
    if fn(path.encode(), _p(out), out.size, C.byref(n), C.byref(d)) < 0:
        raise InsituError(-1, _err(L))
    return out


def read_gt(path):
    L = load_library()
    n, k = C.c_longlong(0), C.c_int(0)
    if L.ivf_read_gt(path.encode(), None, 0, C.byref(n), C.byref(k)) < 0:
        raise InsituError(-1, _err(L))
    out = np.empty((n.value, k.value), np.int32)
    if L.ivf_read_gt(path.encode(), _p(out), out.size, C.byref(n), C.byref(k)) < 0:
        raise InsituError(-1, _err(L))
    return out


def write_index_files(prefix, centroids=None, assign=None, codebook=None, codes=None):
    """writes the given arrays in the reference formats as prefix + {centroids,assign,codebook,codes}.bin"""
    L = load_library()
    rc = 0
    if centroids is not None:
        c = _c(centroids, np.float32)
        rc |= L.ivf_write_centroids((prefix + "centroids.bin").encode(), _p(c), c.shape[0], c.shape[1])
    if assign is not None:
        a = _c(assign, np.int32)
        rc |= L.ivf_write_assign((prefix + "assign.bin").encode(), _p(a), a.shape[0])
    if codebook is not None:
        cb = _c(codebook, np.float32)
        rc |= L.ivf_write_codebook((prefix + "codebook.bin").encode(), _p(cb), *cb.shape)
    if codes is not None:
        cd = _c(codes, np.uint8)
        rc |= L.ivf_write_codes((prefix + "codes.bin").encode(), _p(cd), cd.shape[0], cd.shape[1])
    if rc:
        raise InsituError(-1, _err(L))


class Builder:
    """GPU index build through the C ABI (device tensors in and out).

    ``assign`` is the exact routing with n_probes = 1; ``kmeans`` runs Lloyd
    iterations of assign + ivf_kmeans_update; ``reorder``, ``pq_train`` and
    ``pq_encode`` wrap the other build entry points.  Work runs on the current
    torch stream of the tensors' device."""

    def __init__(self, d: int, batch_rows: int = 65536):
        self.L = load_library(require_device=True)
        self.d = d
        self.batch_rows = batch_rows

    def _stream(self):
        import torch

        return torch.cuda.current_stream().cuda_stream

    def _check(self, rc, ctx=None):
        if rc != IVF_OK:
            msg = (self.L.ivf_last_error(ctx) if ctx else self.L.ivf_global_last_error()).decode()
            raise InsituError(rc, msg)

    def assign(self, x, centroids):
        """nearest centroid (int32 [n]) of the rows of x (uint8 or fp32 device tensor)."""
        import torch

        n = x.shape[0]
        nlist = centroids.shape[0]
        out = torch.empty(n, dtype=torch.int32, device=x.device)
        idx = self.L.ivf_create_index_context()
        b = self.L.ivf_create_batch_context(min(self.batch_rows, max(n, 1)), self.d, 1, 1, nlist)
        try:
            c = centroids.float().contiguous()
            self._check(self.L.ivf_load_centroids(idx, c.data_ptr(), nlist, self.d), idx)
            torch.cuda.current_stream().synchronize()
            self._check(self.L.ivf_assign(b, idx, x.contiguous().data_ptr(), 1 if x.dtype == torch.uint8 else 0,
                                          n, out.data_ptr()), b)
            self.L.ivf_pipeline_sync_batch(b)
        finally:
            self.L.ivf_destroy_batch_context(b)
            self.L.ivf_destroy_index_context(idx)
        return out

    def kmeans_update(self, x, assign, centroids):
        import torch

        self._check(self.L.ivf_kmeans_update(x.contiguous().data_ptr(), 1 if x.dtype == torch.uint8 else 0,
                                             x.shape[0], self.d, assign.data_ptr(), centroids.shape[0],
                                             centroids.data_ptr(), self._stream()))
        return centroids

    def kmeans(self, x, init_centroids, iters):
        """Lloyd k-means from init_centroids (fp32 [nlist, d], updated copy returned)."""
        cent = init_centroids.float().clone().contiguous()
        for _ in range(iters):
            a = self.assign(x, cent)
            self.kmeans_update(x, a, cent)
        return cent

    def reorder(self, assign, nlist):
        """(counts int32 [nlist], offsets int64 [nlist], order int32 [n]) as device tensors."""
        import torch

        n = assign.shape[0]
        counts = torch.empty(nlist, dtype=torch.int32, device=assign.device)
        offsets = torch.empty(nlist, dtype=torch.int64, device=assign.device)
        order = torch.empty(max(n, 1), dtype=torch.int32, device=assign.device)
        self._check(self.L.ivf_build_reorder(assign.data_ptr(), n, nlist, counts.data_ptr(), offsets.data_ptr(),
                                             order.data_ptr(), self._stream()))
        return counts, offsets, order[:n]

    def pq_train(self, x, centroids, assign, codebook, iters):
        import torch

        M = codebook.shape[0]
        self._check(self.L.ivf_pq_train(x.contiguous().data_ptr(), 1 if x.dtype == torch.uint8 else 0, x.shape[0],
                                        self.d, centroids.data_ptr(), assign.data_ptr(), M, iters,
                                        codebook.data_ptr(), self._stream()))
        return codebook

    def pq_encode(self, x, centroids, assign, codebook, rows=None):
        import torch

        M = codebook.shape[0]
        n = rows.shape[0] if rows is not None else x.shape[0]
        codes = torch.empty((n, M), dtype=torch.uint8, device=x.device)
        self._check(self.L.ivf_pq_encode(x.contiguous().data_ptr(), 1 if x.dtype == torch.uint8 else 0, n, self.d,
                                         None if rows is None else rows.data_ptr(), centroids.data_ptr(),
                                         assign.data_ptr(), codebook.data_ptr(), M, codes.data_ptr(),
                                         self._stream()))
        return codes


def _sq_fail(rc):
    raise InsituError(rc, load_library().ivf_global_last_error().decode())


_SQ_TYPES: dict = {}     # torch dtype -> IVF_SQ_*


def _sq_type(dtype):
    """IVF_SQ_* of a torch dtype."""
    t = _SQ_TYPES.get(dtype)
    if t is None:
        import torch

        _SQ_TYPES.update({torch.float32: 0, torch.float16: 1, torch.bfloat16: 2})
        t = _SQ_TYPES.get(dtype)
        if t is None:
            raise ValueError(f"scalar-quantised rows are read and written as float32, float16 or bfloat16, not {dtype}")
    return t


def _sq_need(ok, msg):
    if not ok:
        raise ValueError(msg)


# The checks below are on the path of calls of a few microseconds: messages are
# made only where a check fails.

def _sq_2d(t, name, device=None):
    """(tensor with unit steps inside its rows, distance between rows, rows, row width) of a 2-D device tensor"""
    if t.dim() != 2:
        raise ValueError(f"{name} must be 2-D, got shape {tuple(t.shape)}")
    if not t.is_cuda or (device is not None and t.device != device):
        raise ValueError(f"{name} is on {t.device}, not on {device or 'a CUDA device'}")
    n, d = t.shape
    ld, step = t.stride()
    if (step != 1 and d > 1) or (ld < d and n > 1):
        t = t.contiguous()
        ld = d
    return t, (ld if n > 1 and ld > 0 else max(d, 1)), n, d


def _sq_1d(t, name, n, dtype, device):
    if t.dim() != 1 or t.shape[0] != n:
        raise ValueError(f"{name} must have shape ({n},), got {tuple(t.shape)}")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, not on {device}")
    if t.dtype != dtype:
        import torch

        if dtype != torch.int64 or t.dtype != torch.int32:
            raise ValueError(f"{name} must be {dtype}, got {t.dtype}")
        t = t.to(dtype)
    return t.contiguous()


def _sq_out(out, n, d, dtype, device):
    """(output tensor, distance between its rows)"""
    if out is None:
        import torch

        return torch.empty((n, d), dtype=dtype, device=device), d or 1
    if tuple(out.shape) != (n, d):
        raise ValueError(f"out must have shape {(n, d)}, got {tuple(out.shape)}")
    if out.dtype != dtype or out.device != device:
        raise ValueError(f"out must be {dtype} on {device}")
    ld, step = out.stride()
    if (d > 1 and step != 1) or (n > 1 and ld < d):
        raise ValueError("out must have unit steps inside its rows, and rows that do not overlap")
    return out, (ld if n > 1 and ld > 0 else max(d, 1))


def _sq_capturing(device):
    """whether torch's current stream of that device, the one that _sq_call uses, is being captured"""
    import torch

    if torch.cuda.current_device() != device.index:
        with torch.cuda.device(device):
            return torch.cuda.is_current_stream_capturing()
    return torch.cuda.is_current_stream_capturing()


def _sq_call(fn, device, *args):
    """fn(*args, stream) with the tensors' device current, on torch's current stream of that device"""
    import torch

    if torch.cuda.current_device() != device.index:
        with torch.cuda.device(device):
            rc = fn(*args, torch.cuda.current_stream(device).cuda_stream)
    else:
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(device.index))
    if rc != IVF_OK:
        _sq_fail(rc)


def sq_status(device=None):
    """Waits for the current stream of the device and raises InsituError when a product on it (sq_matmul,
    SQRows.scores) gave up a wait on the device since the last such report: its outputs are not valid."""
    import torch

    load_library(require_device=True)
    device = torch.device("cuda" if device is None else device)
    if device.index is None:
        device = torch.device("cuda", torch.cuda.current_device())
    _sq_call(load_library().ivf_sq_status, device)


def sq_matmul(a, a_scale, b, b_scale, bias=None, dtype=None, out=None):
    """8-bit matrix product with a scale per token and per channel (ivf_sq_matmul):

        out[i, j] = (sum_t a[i, t] * b[j, t]) * a_scale[i] * b_scale[j] + bias[j]

    a int8 [m, k] and b int8 [n, k] (rows at any distance; 16-byte aligned rows
    are fastest), a_scale fp32 [m], b_scale fp32 [n], bias fp32 [n] or None.
    dtype: torch.float32 (default), float16 or bfloat16.  The sum is exact, the
    rest fp32 in the order written (a sum times a_scale that leaves fp32's range
    stays lost) and rounded once.  Runs on the current torch stream of the
    tensors' device; no gradient flows."""
    import torch

    L = load_library()
    if a.dtype != torch.int8 or b.dtype != torch.int8:
        raise ValueError("a and b must be int8")
    a, lda, m, k = _sq_2d(a, "a")
    dev = a.device
    b, ldb, n, kb = _sq_2d(b, "b", dev)
    if k != kb:
        raise ValueError(f"a has rows of {k} values, b of {kb}")
    a_scale = _sq_1d(a_scale, "a_scale", m, torch.float32, dev)
    b_scale = _sq_1d(b_scale, "b_scale", n, torch.float32, dev)
    if bias is not None:
        bias = _sq_1d(bias, "bias", n, torch.float32, dev)
    dtype = dtype or (torch.float32 if out is None else out.dtype)
    t = _sq_type(dtype)
    out, ldo = _sq_out(out, m, n, dtype, dev)
    pa, pb, need, work = a.data_ptr(), b.data_ptr(), 0, None
    if (pa | pb | lda | ldb) & 15:                       # rows that the library may have to copy first
        need = L.ivf_sq_matmul_work(pa, lda, m, pb, ldb, n, k)
        work = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
    _sq_call(L.ivf_sq_matmul, dev, pa, lda, a_scale.data_ptr(), m, pb, ldb, b_scale.data_ptr(), n, k,
             None if bias is None else bias.data_ptr(), out.data_ptr(), t, ldo,
             None if work is None else work.data_ptr(), need)
    return out


class SQRows:
    """A store of scalar-quantised rows: `capacity` slots of `d` values at 8 or 4
    bits with one fp32 scale per `group` values (0: per row), in device tensors.

    ``write`` quantises floating rows into slots (online inserts, a cache that
    grows), ``read`` turns slots back into values, ``scores`` multiplies floating
    queries with every row by 8-bit products.  With L = 127 (8 bits) or 7 (4
    bits): scale = max |x| / L, code = round-half-even(x / scale), value = code *
    scale.  A group with a NaN or an infinity reads back as NaN.

    ``codes``  int8 [capacity, >= d] or uint8 [capacity, >= ceil(d / 2)] (two
    codes a byte, the even one in the low half); ``scales`` fp32 [capacity,
    groups].  Slots never written are zeros: they read as zeros and score 0 (see
    ``scores``).

    Work runs on the current torch stream of the store's device; two writes of
    one store must be ordered.  No gradient flows through any call."""

    def __init__(self, capacity: int, d: int, bits: int = 8, group: int = 0, device=None):
        import torch

        load_library(require_device=True)
        _sq_need(bits in (8, 4), "bits must be 8 or 4")
        _sq_need(capacity >= 0 and d >= 1 and group >= 0, "need capacity >= 0, d >= 1, group >= 0")
        ld = ((d * bits + 7) // 8 + 15) // 16 * 16
        device = torch.device("cuda" if device is None else device)
        codes = torch.zeros((capacity, ld), dtype=torch.int8 if bits == 8 else torch.uint8, device=device)
        scales = torch.zeros((capacity, -(-d // group) if group else 1), dtype=torch.float32, device=device)
        self._adopt(codes, scales, d, bits, group)

    @classmethod
    def from_arrays(cls, codes, scales, d: int, bits: int = 8, group: int = 0) -> "SQRows":
        """a store over existing device tensors (as ``codes`` and ``scales`` above), which it shares"""
        load_library(require_device=True)
        rows = cls.__new__(cls)
        rows._adopt(codes, scales, d, bits, group)
        return rows

    def _adopt(self, codes, scales, d, bits, group):
        import torch

        _sq_need(bits in (8, 4), "bits must be 8 or 4")
        _sq_need(1 <= d <= 1 << 20, "need 1 <= d <= 2^20")
        _sq_need(0 <= group < 1 << 31 and group % 16 == 0, "group must be 0 or a multiple of 16 below 2^31")
        _sq_need(codes.dim() == 2 and scales.dim() == 2 and codes.shape[0] == scales.shape[0],
                 "codes and scales must be 2-D with a row per slot")
        _sq_need(codes.is_cuda and scales.device == codes.device, "codes and scales must be on one CUDA device")
        _sq_need(codes.dtype == (torch.int8 if bits == 8 else torch.uint8) and scales.dtype == torch.float32,
                 "codes must be int8 (8 bits) or uint8 (4 bits), scales float32")
        n = codes.shape[0]
        _sq_need(codes.shape[1] >= (d * bits + 7) // 8, "codes rows are shorter than d values")
        _sq_need(scales.shape[1] == (-(-d // group) if group else 1), "scales must have a column per group")
        for t in (codes, scales):
            _sq_need((t.shape[1] <= 1 or t.stride(1) == 1) and (n <= 1 or t.stride(0) >= t.shape[1]),
                     "codes and scales must have unit steps inside their rows, and rows that do not overlap")
        self.L = load_library()
        self._codes, self._scales = codes, scales
        self.capacity, self.d, self.bits, self.group = n, d, bits, group
        self.device = codes.device
        self._ldc = codes.stride(0) if n > 1 else max(codes.shape[1], codes.stride(0))
        self._lds = scales.stride(0) if n > 1 else max(scales.shape[1], scales.stride(0))
        self._groups = scales.shape[1]
        self._claim = None               # scratch of large writes, kept (4 bytes a slot), and the stream it is of
        self._claim_stream = None
        self._work = {}                  # tokens -> bytes of scratch that scores needs

    @property
    def codes(self):
        return self._codes

    @property
    def scales(self):
        return self._scales

    def _slots(self, slots, n):
        import torch

        if slots is None:
            if n > self.capacity:
                raise ValueError(f"{n} rows for {self.capacity} slots")
            return None
        return _sq_1d(slots, "slots", n, torch.int64, self.device)

    def _rows(self, x):
        """(x with unit steps inside its rows, distance between rows, rows, type) of floating rows as wide as the store's"""
        x, ldx, n, d = _sq_2d(x, "x", self.device)
        if d != self.d:
            raise ValueError(f"x has rows of {d} values, the store of {self.d}")
        return x, ldx, n, _sq_type(x.dtype)

    def write(self, x, slots=None):
        """rows x [n, d] (fp32, fp16 or bf16) into slots [n] (None: slots 0 .. n - 1).

        A row whose slot is outside the store is left out; of rows with one
        slot the last stays; other slots are left as they were."""
        x, ldx, n, t = self._rows(x)
        slots = self._slots(slots, n)
        claim = None
        if slots is not None and n > _SQ_SCAN_ROWS:
            import torch

            # a captured write takes scratch of its own: the graph may run beside others, and outlive the store
            capturing = _sq_capturing(self.device)
            claim = None if capturing else self._claim
            if claim is None:
                claim = torch.empty(max(self.capacity, 1), dtype=torch.int32, device=self.device)
                if not capturing:
                    self._claim = claim
                    self._claim_stream = torch._C._cuda_getCurrentRawStream(self.device.index)
            elif torch._C._cuda_getCurrentRawStream(self.device.index) != self._claim_stream:
                # the store may be dropped while this write runs: its scratch is not handed out before it ends
                claim.record_stream(torch.cuda.current_stream(self.device))
        _sq_call(self.L.ivf_sq_write, self.device, x.data_ptr(), t, n, self.d, ldx,
                 None if slots is None else slots.data_ptr(), self.bits, self.group, self._codes.data_ptr(), self._ldc,
                 self._scales.data_ptr(), self._lds, self.capacity, None if claim is None else claim.data_ptr())
        return self

    def read(self, slots=None, dtype=None, out=None):
        """values [n, d] of slots [n] (None: every slot); a slot outside the store reads as zeros.
        dtype: torch.float32 (default), float16 or bfloat16."""
        import torch

        dtype = dtype or (torch.float32 if out is None else out.dtype)
        t = _sq_type(dtype)
        n = self.capacity if slots is None else slots.shape[0]
        slots = self._slots(slots, n)
        out, ldo = _sq_out(out, n, self.d, dtype, self.device)
        _sq_call(self.L.ivf_sq_read, self.device, self._codes.data_ptr(), self._ldc, self._scales.data_ptr(), self._lds,
                 self.capacity, self.bits, self.group, None if slots is None else slots.data_ptr(), n, self.d,
                 out.data_ptr(), t, ldo)
        return out

    def scores(self, x, bias=None, dtype=None, out=None):
        """[m, capacity] products of floating rows x [m, d] with every row of an
        8-bit store with one scale a row (group 0): x is quantised one scale a
        row as ``write`` does it, then multiplied as by sq_matmul.  bias fp32
        [capacity] or None; dtype of the scores: torch.float32 (default),
        float16 or bfloat16.

        A slot never written scores 0, above every negative score.  Where the
        best rows of a store that is not full are looked for, give a bias of
        minus infinity for its empty slots and 0 for the others."""
        import torch

        if self.bits != 8 or self._groups != 1:
            raise ValueError("scores needs an 8-bit store with one scale a row")
        if self._lds != 1 and self.capacity > 1:
            raise ValueError("scores needs dense scales")
        x, ldx, m, t = self._rows(x)
        if bias is not None:
            bias = _sq_1d(bias, "bias", self.capacity, torch.float32, self.device)
        dtype = dtype or (torch.float32 if out is None else out.dtype)
        to = _sq_type(dtype)
        out, ldo = _sq_out(out, m, self.capacity, dtype, self.device)
        need = self._work.get(m)
        if need is None:
            need = self.L.ivf_sq_scores_work(m, self._codes.data_ptr(), self._ldc, self.capacity, self.d)
            if len(self._work) < 256:
                self._work[m] = need
        work = torch.empty(need, dtype=torch.uint8, device=self.device) if need else None
        _sq_call(self.L.ivf_sq_scores, self.device, x.data_ptr(), t, ldx, m, self._codes.data_ptr(), self._ldc,
                 self._scales.data_ptr(), self.capacity, self.d, None if bias is None else bias.data_ptr(), out.data_ptr(),
                 to, ldo, None if work is None else work.data_ptr(), need)
        return out


class CoarseTiming(C.Structure):
    _fields_ = [(n, C.c_double) for n in ("query_h2d_ms", "seq_init_ms", "query_norm_ms", "gemm_ms", "topk_ms",
                                          "cluster_d2h_ms", "coarse_compute_ms", "coarse_total_ms")]


class _CoarseHandle(C.Structure):
    _fields_ = [("d_centers", vp), ("d_centers_norm", vp), ("cublas_handle", vp), ("n_total_clusters", i32),
                ("dim", i32), ("distance_mode_cached", i32)]


class CoarseRouter:
    """CoarseHandle + coarse_search (cpu_fine.h:232-278): host queries in, host probe ids out."""

    def __init__(self, d_centers_ptr: int, nlist: int, dim: int):
        self.L = load_library(require_device=True)
        self.h = _CoarseHandle()
        self.L.coarse_handle_init(C.byref(self.h), d_centers_ptr, nlist, dim)
        if not self.h.cublas_handle:
            raise InsituError(-1, self.L.ivf_global_last_error().decode())

    def search(self, q, nprobe):
        q = _c(q, np.float32)
        out = np.full((q.shape[0], nprobe), -7, np.int32)
        t = [C.c_double(0), C.c_double(0), C.c_double(0)]
        self.L.coarse_search(C.byref(self.h), _p(q), q.shape[0], nprobe, 0, _p(out), C.byref(t[0]),
                             C.byref(t[1]), C.byref(t[2]))
        err = self.L.ivf_global_last_error().decode()
        if (out == -7).any() and err:
            raise InsituError(-1, err)
        return out

    def last_timing(self) -> CoarseTiming:
        return CoarseTiming.from_address(self.L.coarse_get_last_timing())

    def close(self):
        if self.h.cublas_handle:
            self.L.coarse_handle_release(C.byref(self.h))

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass
