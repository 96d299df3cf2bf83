"""Python mirror of the reference's host API, over the C ABI of libgann.so.

``GustANN`` follows ``gustann::GustANN`` (``src/ssd_search.hpp:29-83``): same
method names, argument meaning and order. Errors raise :class:`GustANNError`
(a ``RuntimeError``, as ``CHECK_CUDA`` throws ``std::runtime_error`` in
``src/common_cuda.cuh:10-17``) carrying the C status code.

The library is loaded from the package directory (``_lib/libgann.so``); there
is no fallback: if it is missing, importing this module raises.
"""
from __future__ import annotations

import ctypes as C
import functools
import os
from dataclasses import dataclass

import numpy as np

from .formats import FLOAT, UINT8

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_HERE, "_lib", "libgann.so")

PART_BLOB_BYTES = 512   # GANN_PART_BLOB_BYTES
GANN_OK, GANN_EINVAL, GANN_EIO, GANN_ENOMEM, GANN_ECUDA, GANN_ETIMEDOUT, GANN_EUNSUPPORTED, GANN_ESTATE = range(8)
STATUS_NAMES = ["OK", "EINVAL", "EIO", "ENOMEM", "ECUDA", "ETIMEDOUT", "EUNSUPPORTED", "ESTATE"]

# Every symbol include/gann.h declares.
EXPORTS = ["gann_open", "gann_open_device", "gann_search", "gann_search_device", "gann_close", "gann_last_error",
           "gann_index_info", "gann_probe_lut", "gann_probe_entry", "gann_pivot_sample", "gann_set_option",
           "gann_search_noalloc", "gann_part_export", "gann_part_attach", "gann_hop_begin", "gann_hop_requests",
           "gann_hop_step", "gann_hop_finish", "gann_hop_free", "gann_read_pages", "gann_exact_knn",
           "gann_robust_prune", "gann_sort_unique_rows", "gann_quantize_rows", "gann_matmul_i8",
           "gann_beam_select_workspace", "gann_beam_select", "gann_reorder_states"]
GANN_OPT_ADC_MODE, GANN_OPT_PIVOT_WARPS, GANN_OPT_NEIGHBOUR_CODES = 1, 2, 3
LAYOUT_AUTO, LAYOUT_SEPARATE, LAYOUT_NEIGHBOUR_CODES = 0, 1, 2
ADC_AUTO, ADC_TABLE, ADC_PIVOT, ADC_FILTERED = 0, 1, 2, 3
METRIC_L2, METRIC_IP = 0, 1
F32, F16, BF16 = 1, 2, 3   # gann_float
MAX_BEAMS = 128            # beams of a group, and candidates kept


class GustANNError(RuntimeError):
    def __init__(self, code: int, msg: str):
        self.code = code
        name = STATUS_NAMES[code] if 0 <= code < len(STATUS_NAMES) else str(code)
        super().__init__(f"GANN_{name}: {msg}")


class _Config(C.Structure):
    _fields_ = [("index_file", C.c_char_p), ("pq_file_prefix", C.c_char_p), ("nav_graph_prefix", C.c_char_p),
                ("dtype", C.c_int32), ("use_gpu_mem", C.c_int32), ("device", C.c_int32),
                ("layout", C.c_int32), ("part_count", C.c_int32), ("part_index", C.c_int32),
                ("metric", C.c_int32), ("reserved", C.c_int32 * 1)]


class _Stats(C.Structure):
    _fields_ = [("run_time", C.c_double), ("total_time", C.c_double), ("hops", C.c_int64),
                ("adc_evals", C.c_int64), ("capped_queries", C.c_int64), ("bytes_touched", C.c_int64)]


class _DeviceIndex(C.Structure):
    _fields_ = [("vectors", C.c_void_p), ("vec_stride", C.c_int64), ("adjacency", C.c_void_p),
                ("adj_stride", C.c_int32), ("max_degree", C.c_int32), ("codes", C.c_void_p),
                ("code_stride", C.c_int32), ("pq_chunks", C.c_int32), ("pivots", C.c_void_p),
                ("centroid", C.c_void_p), ("chunk_offsets", C.c_void_p), ("num_points", C.c_int64),
                ("dim", C.c_int32), ("dtype", C.c_int32), ("medoid", C.c_int64), ("device", C.c_int32),
                ("metric", C.c_int32), ("reserved", C.c_int32 * 2)]


class _Info(C.Structure):
    _fields_ = [("num_points", C.c_int64), ("dim", C.c_int32), ("max_degree", C.c_int32),
                ("pq_chunks", C.c_int32), ("dtype", C.c_int32), ("medoid", C.c_int64),
                ("node_len", C.c_int32), ("nodes_per_page", C.c_int32), ("nav_points", C.c_int32),
                ("nav_start", C.c_int32), ("device_bytes", C.c_int64)]


class _State(C.Structure):
    """gann_state: 13 words of 8 bytes."""

    _fields_ = [("src", C.c_void_p), ("dst", C.c_void_p), ("src_group", C.c_int64), ("src_beam", C.c_int64),
                ("src_stride", C.c_int64 * 2), ("dst_group", C.c_int64), ("dst_beam", C.c_int64),
                ("dst_stride", C.c_int64 * 2), ("size", C.c_int64 * 2), ("row_bytes", C.c_int64)]


def _load() -> C.CDLL:
    if not os.path.exists(LIB_PATH):
        raise ImportError(f"{LIB_PATH} is not built; run `python -m gustann_b200.build`")
    lib = C.CDLL(LIB_PATH)
    vp, i64, i32, fp, ip = C.c_void_p, C.c_int64, C.c_int32, C.c_void_p, C.c_void_p
    lib.gann_open.argtypes = [C.POINTER(_Config), C.POINTER(vp)]
    lib.gann_open_device.argtypes = [C.POINTER(_DeviceIndex), C.POINTER(vp)]
    lib.gann_search.argtypes = [vp, fp, i64, i32, i32, ip, fp, ip, C.POINTER(_Stats)]
    lib.gann_search_device.argtypes = [vp, vp, i64, i32, i32, vp, vp, vp, vp, vp]
    lib.gann_close.argtypes = [vp]
    lib.gann_last_error.restype = C.c_char_p
    lib.gann_index_info.argtypes = [vp, C.POINTER(_Info)]
    lib.gann_probe_lut.argtypes = [vp, fp, i64, fp]
    lib.gann_probe_entry.argtypes = [vp, fp, i64, ip, ip]
    lib.gann_pivot_sample.argtypes = [i64, i64, C.c_uint32, ip]
    lib.gann_set_option.argtypes = [vp, i32, i64]
    lib.gann_search_noalloc.argtypes = [C.POINTER(_DeviceIndex), vp, i64, i32, i32, vp, vp, vp, vp]
    lib.gann_part_export.argtypes = [vp, vp, i64]
    lib.gann_part_attach.argtypes = [vp, i32, C.c_char_p, i64]
    lib.gann_hop_begin.argtypes = [vp, fp, i64, i32, i32, C.POINTER(vp)]
    lib.gann_hop_requests.argtypes = [vp, ip, C.POINTER(i64)]
    lib.gann_hop_step.argtypes = [vp, vp]
    lib.gann_hop_finish.argtypes = [vp, ip, fp, ip]
    lib.gann_hop_free.argtypes = [vp]
    lib.gann_read_pages.argtypes = [C.c_char_p, ip, i64, i32, vp, i32]
    lib.gann_exact_knn.argtypes = [vp, i64, i64, i32, i32, vp, i64, i64, i32, i32, vp, vp, i32, vp]
    lib.gann_robust_prune.argtypes = [vp, i64, i64, i32, i32, vp, i64, vp, vp, i32, i32, C.c_float, vp, vp, i32, vp]
    lib.gann_sort_unique_rows.argtypes = [vp, vp, i64, i32, vp, vp, i32, vp]
    lib.gann_quantize_rows.argtypes = [vp, i64, i64, i32, i32, vp, i64, vp, i32, vp]
    lib.gann_matmul_i8.argtypes = [vp, i64, i64, vp, vp, i64, i64, vp, vp, i32, vp, i64, i32, i32, vp]
    lib.gann_beam_select_workspace.argtypes = [i64, i32, i32, i32, i32, i32, C.POINTER(i64)]
    lib.gann_beam_select.argtypes = [vp, i32, i64, i64, vp, vp, i64, i32, i32, i32, i32, i32, vp, vp, vp, vp, i64,
                                     i32, vp]
    lib.gann_reorder_states.argtypes = [vp, i32, vp, i64, i32, i32, i32, vp]
    for name in EXPORTS:
        if name != "gann_last_error":
            getattr(lib, name).restype = C.c_int
    return lib


lib = _load()


def _check(rc: int) -> None:
    if rc != GANN_OK:
        raise GustANNError(rc, lib.gann_last_error().decode(errors="replace"))


def _ptr(a: np.ndarray):
    return a.ctypes.data_as(C.c_void_p)


@dataclass
class GustANNConfig:
    """``gustann::GustANNConfig`` (``src/ssd_search.hpp:18-23``)."""

    index_file: str
    pq_file_prefix: str
    nav_graph_prefix: str = ""


@dataclass
class GustANNStats:
    """``gustann::GustANNStats`` plus the counters of ``gann_stats``."""

    run_time: float = 0.0
    total_time: float = 0.0
    hops: int = 0
    adc_evals: int = 0
    capped_queries: int = 0
    bytes_touched: int = 0


class GustANN:
    """Drop-in for ``gustann::GustANN`` on one B200 (``device``). ``metric``
    (an extension; the reference is L2-only) is :data:`METRIC_L2` or
    :data:`METRIC_IP` (distances -<q, x>)."""

    def __init__(self, data_type: int = FLOAT, device: int = 0, layout: int = 0, metric: int = METRIC_L2):
        if data_type not in (UINT8, FLOAT):
            raise GustANNError(GANN_EINVAL, "data type must be UINT8 (0) or FLOAT (1)")
        self.data_type = data_type
        self.device = device
        self.layout = layout
        self.metric = metric
        self._h = None
        self.dim = 0

    # --------------------------------------------------------------- init
    def init_pure_mem(self, config: GustANNConfig, use_gpu_mem: bool, part_count: int = 0,
                      part_index: int = 0) -> None:
        """``GustANN::init_pure_mem`` (``src/ssd_search.cu:108-112``). With
        ``part_count`` > 1 the node records are split by id range and this
        handle loads range ``part_index`` (-1: every range, on this device);
        other processes' ranges are added with :meth:`attach_part`."""
        self.close()
        cfg = _Config(config.index_file.encode(), config.pq_file_prefix.encode(),
                      (config.nav_graph_prefix or "").encode(), self.data_type, int(bool(use_gpu_mem)),
                      self.device, self.layout, part_count, part_index, self.metric)
        h = C.c_void_p()
        _check(lib.gann_open(C.byref(cfg), C.byref(h)))
        self._h = h
        self.dim = self.info()["dim"]

    @classmethod
    def from_device(cls, vectors, adjacency, codes, pivots: np.ndarray, centroid: np.ndarray,
                    chunk_offsets: np.ndarray, medoid: int, max_degree: int, device: int = 0,
                    metric: int = METRIC_L2) -> "GustANN":
        """Search over caller-owned CUDA tensors (``gann_open_device``): ``vectors``
        [n, d] uint8/float32, ``adjacency`` [n, stride] int32 (-1 = empty slot),
        ``codes`` [n, code_stride] uint8. The tensors must stay alive and may be
        rewritten between searches."""
        dt = UINT8 if vectors.dtype.itemsize == 1 else FLOAT
        g = cls(dt, device, metric=metric)
        piv = np.ascontiguousarray(pivots, np.float32)
        cen = np.ascontiguousarray(centroid, np.float32)
        off = np.ascontiguousarray(chunk_offsets, np.uint32)
        d = _DeviceIndex(vectors.data_ptr(), vectors.stride(0) * vectors.element_size(), adjacency.data_ptr(),
                         adjacency.stride(0), max_degree, codes.data_ptr(), codes.stride(0), len(off) - 1,
                         _ptr(piv), _ptr(cen), _ptr(off), vectors.shape[0], vectors.shape[1], dt, medoid, device,
                         metric)
        h = C.c_void_p()
        _check(lib.gann_open_device(C.byref(d), C.byref(h)))
        g._h = h
        g.dim = int(vectors.shape[1])
        g._keep = (vectors, adjacency, codes)
        return g

    def init_bam(self, *args, **kwargs) -> None:
        raise GustANNError(GANN_EUNSUPPORTED, "init_bam: BaM search is not provided by this build")

    # ------------------------------------------------------------- search
    def search(self, qdata: np.ndarray, num_queries: int, topk: int, ef_search: int, nns: np.ndarray,
               distances: np.ndarray, found_cnt: np.ndarray, stats: GustANNStats | None = None) -> None:
        """``GustANN::search`` (``src/ssd_search.cu:114-140``): fills ``nns``,
        ``distances`` (squared L2) and ``found_cnt`` in place."""
        self._need()
        q = np.ascontiguousarray(qdata, dtype=np.float32)
        if q.size < num_queries * self.dim:
            raise GustANNError(GANN_EINVAL, "search: qdata holds fewer than num_queries rows")
        for arr, dt, n in ((nns, np.int32, num_queries * topk), (distances, np.float32, num_queries * topk),
                           (found_cnt, np.int32, num_queries)):
            if arr.dtype != dt or not arr.flags.c_contiguous or arr.size < n:
                raise GustANNError(GANN_EINVAL, "search: output arrays must be contiguous int32/float32 of the right size")
        if getattr(self, "_hybrid", None) is not None:
            import time
            t0 = time.perf_counter()
            batch = self._hybrid[0] or max(num_queries, 1)
            rounds = 0
            for lo in range(0, num_queries, batch):
                hi = min(num_queries, lo + batch)
                n_, d_, f_, r_ = self.hop_search(q.reshape(-1, self.dim)[lo:hi], topk, ef_search,
                                                 threads=self._hybrid[1])
                nns.reshape(-1, topk)[lo:hi] = n_
                distances.reshape(-1, topk)[lo:hi] = d_
                found_cnt.reshape(-1)[lo:hi] = f_
                rounds += r_
            if stats is not None:
                stats.run_time = stats.total_time = time.perf_counter() - t0
                stats.hops = rounds
            return
        st = _Stats()
        _check(lib.gann_search(self._h, _ptr(q), num_queries, topk, ef_search, _ptr(nns), _ptr(distances),
                               _ptr(found_cnt), C.byref(st)))
        if stats is not None:
            for f, _ in _Stats._fields_:
                setattr(stats, f, getattr(st, f))

    def query(self, qdata: np.ndarray, topk: int, ef_search: int, stats: GustANNStats | None = None):
        """Convenience form of :meth:`search` returning ``(nns, distances, found_cnt)``."""
        q = np.ascontiguousarray(qdata, dtype=np.float32).reshape(-1, self.dim if self.dim else qdata.shape[-1])
        nq = q.shape[0]
        nns = np.zeros((nq, topk), np.int32)
        dist = np.zeros((nq, topk), np.float32)
        found = np.zeros(nq, np.int32)
        self.search(q, nq, topk, ef_search, nns, dist, found, stats)
        return nns, dist, found

    def search_device(self, d_queries: int, num_queries: int, topk: int, ef_search: int, d_nns: int,
                      d_distances: int, d_found_cnt: int, d_hops: int = 0, stream: int = 0) -> None:
        """Device-pointer search (``gann_search_device``); pointers are ints
        (e.g. ``tensor.data_ptr()``), ``stream`` a ``cudaStream_t`` handle."""
        self._need()
        _check(lib.gann_search_device(self._h, d_queries, num_queries, topk, ef_search, d_nns, d_distances,
                                      d_found_cnt, d_hops or None, stream or None))

    # ------------------------------------------------------------- probes
    def probe_lut(self, qdata: np.ndarray) -> np.ndarray:
        self._need()
        q = np.ascontiguousarray(qdata, dtype=np.float32).reshape(-1, self.dim)
        m = self.info()["pq_chunks"]
        out = np.zeros((q.shape[0], m, 256), np.float32)
        _check(lib.gann_probe_lut(self._h, _ptr(q), q.shape[0], _ptr(out)))
        return out

    def probe_entry(self, qdata: np.ndarray):
        self._need()
        q = np.ascontiguousarray(qdata, dtype=np.float32).reshape(-1, self.dim)
        s = np.zeros(q.shape[0], np.int32)
        e = np.zeros(q.shape[0], np.int32)
        _check(lib.gann_probe_entry(self._h, _ptr(q), q.shape[0], _ptr(s), _ptr(e)))
        return s, e

    def init_hybrid(self, config: GustANNConfig, hybrid_config=None) -> None:
        """``GustANN::init_hybrid`` (``src/ssd_search.cu:81-106``): node records
        stay in the index file; :meth:`search` and :meth:`query` then run the
        host-driven hop search (:meth:`hop_search`). ``hybrid_config`` may carry
        ``mini_batch`` and ``thread_cnt`` (``HybridExecutorConfig``)."""
        self.close()
        cfg = _Config(config.index_file.encode(), config.pq_file_prefix.encode(),
                      (config.nav_graph_prefix or "").encode(), self.data_type, 2, self.device, 1, 0, 0,
                      self.metric)
        h = C.c_void_p()
        _check(lib.gann_open(C.byref(cfg), C.byref(h)))
        self._h = h
        self.dim = self.info()["dim"]
        self._index_file = config.index_file
        self._hybrid = (getattr(hybrid_config, "mini_batch", 0) or 0, getattr(hybrid_config, "thread_cnt", 0) or 0)

    def hop_search(self, queries: np.ndarray, topk: int, ef_search: int, index_file: str | None = None,
                   threads: int = 0, read_pages=None):
        """Host-driven search, one hop per round (``gann_hop_*``): between hops
        the 4 KB page of every query's requested node is read from
        ``index_file`` (``gann_read_pages``), or by ``read_pages(ids, pages)``
        when given. Returns ``(nns, distances, found_cnt, rounds)``."""
        self._need()
        q = np.ascontiguousarray(queries, dtype=np.float32).reshape(-1, self.dim)
        nq = q.shape[0]
        index_file = index_file or getattr(self, "_index_file", None)
        npp = self.info()["nodes_per_page"]
        b = C.c_void_p()
        _check(lib.gann_hop_begin(self._h, _ptr(q), nq, topk, ef_search, C.byref(b)))
        try:
            ids = np.full(nq, -1, np.int32)
            pages = np.zeros((nq, 4096), np.uint8)
            active = C.c_int64()
            rounds = 0
            while True:
                _check(lib.gann_hop_requests(b, _ptr(ids), C.byref(active)))
                if active.value == 0:
                    break
                if read_pages is not None:
                    read_pages(ids, pages)
                else:
                    _check(lib.gann_read_pages(index_file.encode(), _ptr(ids), nq, npp, _ptr(pages), threads))
                _check(lib.gann_hop_step(b, _ptr(pages)))
                rounds += 1
            nns = np.zeros((nq, topk), np.int32)
            dist = np.zeros((nq, topk), np.float32)
            found = np.zeros(nq, np.int32)
            _check(lib.gann_hop_finish(b, _ptr(nns), _ptr(dist), _ptr(found)))
        finally:
            lib.gann_hop_free(b)
        return nns, dist, found, rounds

    def export_part(self) -> bytes:
        """``gann_part_export``: an opaque blob naming this handle's record
        range for :meth:`attach_part` in another process."""
        self._need()
        buf = C.create_string_buffer(PART_BLOB_BYTES)
        _check(lib.gann_part_export(self._h, buf, PART_BLOB_BYTES))
        return buf.raw

    def attach_part(self, part: int, blob: bytes) -> None:
        """``gann_part_attach``: map record range ``part`` exported by another
        process (peer access over NVLink)."""
        self._need()
        if len(blob) < PART_BLOB_BYTES:
            raise GustANNError(GANN_EINVAL, "blob too short")
        _check(lib.gann_part_attach(self._h, part, blob, PART_BLOB_BYTES))

    def set_option(self, option: int, value: int) -> None:
        """``gann_set_option``: ADC mode (0 auto, 1 table, 2 pivot) or pivot warps."""
        self._need()
        _check(lib.gann_set_option(self._h, option, value))

    def info(self) -> dict:
        self._need()
        inf = _Info()
        _check(lib.gann_index_info(self._h, C.byref(inf)))
        return {f: getattr(inf, f) for f, _ in _Info._fields_}

    # ---------------------------------------------------------- lifetime
    def close(self) -> None:
        if self._h is not None:
            lib.gann_close(self._h)
            self._h = None
        self._hybrid = None

    def _need(self) -> None:
        if self._h is None:
            raise GustANNError(GANN_ESTATE, "GustANN used before init_pure_mem")

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.close()


def exact_knn(base, queries, k: int, metric: int = METRIC_L2, stream: int = 0):
    """Exact ``k`` nearest rows of ``base`` for every row of ``queries``
    (``gann_exact_knn``): CUDA tensors of one dtype (uint8 or float32), rows
    16-byte aligned. Returns ``(ids int32 [nq, k], dists float32 [nq, k])`` on
    the same device, ascending by (distance, id); L2 distances are squared."""
    import torch
    if base.dtype != queries.dtype or base.dtype not in (torch.uint8, torch.float32):
        raise GustANNError(GANN_EINVAL, "exact_knn: base and queries must both be uint8 or float32")
    if not (base.is_cuda and queries.is_cuda) or base.device != queries.device:
        raise GustANNError(GANN_EINVAL, "exact_knn: tensors must be on one CUDA device")
    if base.stride(1) != 1 or queries.stride(1) != 1:
        raise GustANNError(GANN_EINVAL, "exact_knn: rows must be contiguous")
    dt = UINT8 if base.dtype == torch.uint8 else FLOAT
    nq = queries.shape[0]
    ids = torch.empty((nq, k), dtype=torch.int32, device=base.device)
    dists = torch.empty((nq, k), dtype=torch.float32, device=base.device)
    es = base.element_size()
    _check(lib.gann_exact_knn(base.data_ptr(), base.shape[0], base.stride(0) * es, base.shape[1], dt,
                              queries.data_ptr(), queries.stride(0) * es, nq, k, metric, ids.data_ptr(),
                              dists.data_ptr(), base.device.index or 0, stream or None))
    return ids, dists


def robust_prune(vectors, points, cand, cand_dist, r: int, alpha: float, stream: int = 0):
    """RobustPrune of many points on the GPU (``gann_robust_prune``):
    ``vectors`` [n, d] uint8/float32 CUDA tensor (rows 16-byte aligned),
    ``points`` [b] int32, ``cand`` [b, k] int32 candidates nearest-first (-1
    empty), ``cand_dist`` [b, k] float32 squared distances to the point.
    Returns (kept [b, r] int32 nearest-first, -1 padded; their distances)."""
    import torch
    if vectors.dtype not in (torch.uint8, torch.float32) or vectors.stride(1) != 1:
        raise GustANNError(GANN_EINVAL, "robust_prune: vectors must be uint8/float32 with contiguous rows")
    dt = UINT8 if vectors.dtype == torch.uint8 else FLOAT
    pts = points.to(torch.int32).contiguous()
    ci = cand.to(torch.int32).contiguous()
    cd = cand_dist.to(torch.float32).contiguous()
    b, k = ci.shape
    out = torch.empty((b, r), dtype=torch.int32, device=vectors.device)
    outd = torch.empty((b, r), dtype=torch.float32, device=vectors.device)
    _check(lib.gann_robust_prune(vectors.data_ptr(), vectors.shape[0], vectors.stride(0) * vectors.element_size(),
                                 vectors.shape[1], dt, pts.data_ptr(), b, ci.data_ptr(), cd.data_ptr(), k, r,
                                 float(alpha), out.data_ptr(), outd.data_ptr(), vectors.device.index or 0,
                                 stream or None))
    return out, outd


def sort_unique_rows(ids, dists, stream: int = 0):
    """Rows of (id, distance) candidates sorted by (distance, id) with empty
    slots (id < 0) and repeated ids removed, -1/+inf padded
    (``gann_sort_unique_rows``). CUDA tensors [rows, k], k <= 256; returns
    (ids int32, dists float32) of the same shape."""
    import torch
    i = ids.to(torch.int32).contiguous()
    d = dists.to(torch.float32).contiguous()
    rows, k = i.shape
    oi = torch.empty_like(i)
    od = torch.empty_like(d)
    _check(lib.gann_sort_unique_rows(i.data_ptr(), d.data_ptr(), rows, k, oi.data_ptr(), od.data_ptr(),
                                     i.device.index or 0, stream or None))
    return oi, od


def _fail(msg: str):
    raise GustANNError(GANN_EINVAL, msg)


_torch = None
_FLOATS = {}   # torch dtype -> gann_float


def _get_torch():
    """torch, imported with the first call that takes tensors."""
    global _torch
    if _torch is None:
        import torch
        _FLOATS.update({torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16})
        _torch = torch
    return _torch


def _float_code(dtype, who: str) -> int:
    code = _FLOATS.get(dtype)
    if code is None:
        _fail(f"{who}: dtype must be float32, float16 or bfloat16")
    return code


def _on_cuda(who: str, *tensors):
    """The tensors' common device and its index."""
    dev = tensors[0].device
    for t in tensors:
        if t.device != dev or not t.is_cuda:
            _fail(f"{who}: tensors must be on one CUDA device")
    return dev, dev.index


def _stream_scope(device, stream: int):
    """Makes ``stream`` (a ``cudaStream_t``, 0 the default stream) torch's
    current one, so that a call's outputs and workspaces are allocated on the
    stream it runs on."""
    torch = _get_torch()
    return torch.cuda.stream(torch.cuda.ExternalStream(stream, device) if stream
                             else torch.cuda.default_stream(device))


def _extent(t):
    """First byte of a tensor and the byte behind its last one."""
    span = sum((n - 1) * s for n, s in zip(t.shape, t.stride())) + 1 if t.numel() else 0
    return t.data_ptr(), t.data_ptr() + span * t.element_size()


def _disjoint(a, b) -> bool:
    """Two tensors share no memory (sufficient test): one lies behind the other,
    or they lie side by side in every period of their strides, largest first, as
    slices of one array do."""
    (a0, a1), (b0, b1) = _extent(a), _extent(b)
    if a1 <= b0 or b1 <= a0 or a0 == a1 or b0 == b1:
        return True
    if a0 > b0:
        a, b, a0, b0 = b, a, b0, a0
    gap = b0 - a0     # from a's start to b's, within the period
    left = sorted(((s * a.element_size(), n) for n, s in zip(a.shape, a.stride()) if n > 1), reverse=True)
    right = sorted(((s * b.element_size(), n) for n, s in zip(b.shape, b.stride()) if n > 1), reverse=True)
    la, lb = a.element_size(), b.element_size()     # bytes of one element
    while left or right:
        period = max(d[0][0] for d in (left, right) if d)
        if period == 0:
            return False
        for d in (left, right):   # a tensor without this stride has one period
            if d and d[0][0] == period:
                d.pop(0)
        gap %= period
        wa, wb = (sum((n - 1) * s for s, n in d) + e for d, e in ((left, la), (right, lb)))
        if gap + wb > period:     # count from b's start instead
            gap = (period - gap) % period
            left, right, la, lb, wa, wb = right, left, lb, la, wb, wa
        if wa > period or gap + wb > period:
            return False
        if gap >= wa:
            return True
    return False


def quantize_rows(x, stream: int | None = None):
    """Rows of ``x`` [n, d] (float32, float16 or bfloat16 CUDA tensor, contiguous
    rows) as 8-bit codes with one scale each (``gann_quantize_rows``): ``scale =
    max|x| * float32(1/127)``, ``code = x / scale`` to the nearest integer. Returns ``(codes
    int8 [n, d], scales float32 [n])``; the codes' rows start on 16-byte
    boundaries, as :func:`matmul_i8` wants them. A row with a NaN or an
    infinity gets scale NaN and codes 0. ``stream``: a ``cudaStream_t``, or
    None for torch's current stream; tensors made on other streams must stay
    alive until it has passed the call. No gradients are recorded, here and in
    the three calls below."""
    torch = _get_torch()
    if x.dim() != 2:
        _fail("quantize_rows: x must have two dimensions")
    dt = _float_code(x.dtype, "quantize_rows")
    dev, index = _on_cuda("quantize_rows", x)
    n, d = x.shape
    step, inner = x.stride()
    if inner != 1 and d > 1:
        _fail("quantize_rows: rows must be contiguous")
    if stream is not None:
        with _stream_scope(dev, stream):
            return quantize_rows(x)
    pad = (d + 15) // 16 * 16
    codes = torch.empty_strided((n, d), (pad, 1), dtype=torch.int8, device=dev)
    scales = torch.empty(n, dtype=torch.float32, device=dev)
    _check(lib.gann_quantize_rows(x.data_ptr(), n, step * x.element_size(), d, dt, codes.data_ptr(), pad,
                                  scales.data_ptr(), index, torch._C._cuda_getCurrentRawStream(index)))
    return codes, scales


def _i8_rows(name: str, codes, scales):
    if codes.dtype != _torch.int8 or codes.dim() != 2:
        _fail(f"matmul_i8: {name} must be int8 with two dimensions")
    n, k = codes.shape
    stride, inner = codes.stride()
    if scales.dtype != _torch.float32 or scales.shape != (n,) or (n > 1 and scales.stride(0) != 1):
        _fail(f"matmul_i8: {name}'s scales must be contiguous float32, one a row")
    if inner != 1 and k > 1:
        _fail(f"matmul_i8: rows of {name} must be contiguous")
    if n <= 1:
        stride = (k + 15) // 16 * 16
    if n and (stride % 16 or codes.data_ptr() % 16):
        _fail(f"matmul_i8: rows of {name} must start on 16-byte boundaries, as quantize_rows lays them out")
    return n, k, stride


def matmul_i8(a, a_scales, b, b_scales, bias=None, dtype=None, out=None, stream: int | None = None):
    """``out[i, j] = (a[i] . b[j]) * a_scales[i] * b_scales[j] + bias[j]`` of 8-bit
    rows (``gann_matmul_i8``): ``a`` [m, k] and ``b`` [n, k] int8 CUDA tensors
    whose rows start on 16-byte boundaries (:func:`quantize_rows` makes them),
    scales float32 [m] and [n], ``bias`` float32 [n] or None. Sums are exact.
    Returns ``out`` [m, n] of ``dtype`` (float32 unless given; float16 and
    bfloat16 too), or fills ``out`` when it is given (contiguous rows).
    Queries against base rows: their scores; tokens against the rows of a
    weight matrix: a linear layer. A GPU that does not serve the kernel for
    about 4 s leaves NaN in what it has not made. ``stream`` as in
    :func:`quantize_rows`."""
    torch = _get_torch()
    m, k, sa = _i8_rows("a", a, a_scales)
    n, kb, sb = _i8_rows("b", b, b_scales)
    if k != kb:
        _fail("matmul_i8: a and b must have the same number of columns")
    ins = [a, a_scales, b, b_scales]
    if bias is not None:
        if bias.dtype != torch.float32 or bias.shape != (n,) or (n > 1 and bias.stride(0) != 1):
            _fail("matmul_i8: bias must be contiguous float32, one a row of b")
        ins.append(bias)
    dev, index = _on_cuda("matmul_i8", *ins)
    if out is not None:
        _on_cuda("matmul_i8", a, out)
        if out.shape != (m, n) or (dtype is not None and out.dtype != dtype):
            _fail("matmul_i8: out must be [m, n] of the given dtype")
        if (n > 1 and out.stride(1) != 1) or (m > 1 and out.stride(0) < n):
            _fail("matmul_i8: rows of out must be contiguous and apart from each other")
        if not all(_disjoint(out, t) for t in ins):
            _fail("matmul_i8: out overlaps an input")
        dtype = out.dtype
    elif dtype is None:
        dtype = torch.float32
    dt = _float_code(dtype, "matmul_i8")
    if stream is not None:
        with _stream_scope(dev, stream):
            return matmul_i8(a, a_scales, b, b_scales, bias, dtype, out)
    if out is None:
        out = torch.empty(m, n, dtype=dtype, device=dev)
    _check(lib.gann_matmul_i8(a.data_ptr(), m, sa, a_scales.data_ptr(), b.data_ptr(), n, sb, b_scales.data_ptr(),
                              None if bias is None else bias.data_ptr(), k, out.data_ptr(),
                              out.stride(0) if m > 1 else n, dt, index, torch._C._cuda_getCurrentRawStream(index)))
    return out


@functools.lru_cache(maxsize=1024)
def _select_workspace(g, w, v, k, dt, soft) -> int:
    need = C.c_int64()
    _check(lib.gann_beam_select_workspace(g, w, v, k, dt, soft, C.byref(need)))
    return need.value


def beam_select(scores, logits, k: int, log_softmax: bool = False, finished=None, end_token: int = 0,
                stream: int | None = None):
    """The best ``k`` continuations of each group's beams (``gann_beam_select``):
    ``scores`` [g, w] float32, ``logits`` [g, w, v] float32, float16 or bfloat16
    (any strides with v contiguous). A candidate is worth ``scores[g, b] +
    logits[g, b, t]``, or with ``log_softmax`` ``scores[g, b] +
    log_softmax(logits[g, b])[t]``; the largest come first, compared in 64 bits,
    equal ones in ascending order of (b, t) (with ``log_softmax`` a beam's own
    candidates by ``scores + logits``, then t; those of different beams may trade
    places where their values are within 2^-17). Logits that are NaN or infinite are masked;
    beams whose score is not finite are dead. ``finished`` [g, w] bool: such a
    beam has one candidate, ``end_token`` at its own score. Returns ``(scores
    float32, parents int32, tokens int32)``, each [g, k], filled up with
    -inf, -1, -1. w and k at most 128. ``stream`` as in :func:`quantize_rows`."""
    torch = _get_torch()
    if logits.dim() != 3 or scores.dtype != torch.float32 or scores.shape != logits.shape[:2]:
        _fail("beam_select: need logits [g, w, v] and float32 scores [g, w]")
    dt = _float_code(logits.dtype, "beam_select")
    g, w, v = logits.shape
    if finished is None:
        dev, index = _on_cuda("beam_select", scores, logits)
    else:
        if finished.dtype not in (torch.bool, torch.uint8) or finished.shape != (g, w):
            _fail("beam_select: finished must be bool [g, w]")
        dev, index = _on_cuda("beam_select", scores, logits, finished)
    gs, bs, inner = logits.stride()
    if inner != 1 and v > 1:
        _fail("beam_select: the last dimension of logits must be contiguous")
    if stream is not None:
        with _stream_scope(dev, stream):
            return beam_select(scores, logits, k, log_softmax, finished, end_token)
    soft = 1 if log_softmax else 0
    need = _select_workspace(g, w, v, k, dt, soft)
    scores = scores.contiguous()
    if finished is not None:
        finished = finished.contiguous()
    ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
    out_s = torch.empty(g, k, dtype=torch.float32, device=dev)
    out_p = torch.empty(g, k, dtype=torch.int32, device=dev)
    out_t = torch.empty_like(out_p)
    _check(lib.gann_beam_select(logits.data_ptr(), dt, gs, bs, scores.data_ptr(),
                                None if finished is None else finished.data_ptr(), g, w, v, k, soft, end_token,
                                out_s.data_ptr(), out_p.data_ptr(), out_t.data_ptr(),
                                None if ws is None else ws.data_ptr(), need, index,
                                torch._C._cuda_getCurrentRawStream(index)))
    return out_s, out_p, out_t


def _state_layout(src, dst):
    """The dimensions behind (group, beam) of two tensors of one shape as at most
    two strided dimensions and a run of contiguous bytes (None if they do not
    fit)."""
    es = src.element_size()
    dims = [(n, a, b) for n, a, b in zip(src.shape[2:], src.stride()[2:], dst.stride()[2:]) if n != 1]
    run = 1
    while dims and dims[-1][1] == run and dims[-1][2] == run:
        run *= dims.pop()[0]
    if not dims:
        return [1, 1], [0, 0], [0, 0], run * es
    merged = []
    for n, a, b in dims:
        if merged and merged[-1][1] == n * a and merged[-1][2] == n * b:
            merged[-1] = (merged[-1][0] * n, a, b)
        else:
            merged.append((n, a, b))
    if len(merged) > 2:
        return None
    merged = [(1, 0, 0)] * (2 - len(merged)) + merged
    return [m[0] for m in merged], [m[1] * es for m in merged], [m[2] * es for m in merged], run * es


def _apart(t) -> bool:
    """No two elements of the tensor share memory (sufficient test)."""
    span = 1
    for s, n in sorted((s, n) for n, s in zip(t.shape, t.stride()) if n > 1):
        if s < span:
            return False
        span = s * (n - 1) + span
    return True


def reorder_states(states, parents, out=None, stream: int | None = None):
    """The states that follow the selected beams (``gann_reorder_states``):
    ``out[g, j] = states[g, parents[g, j]]``. ``states``: a CUDA tensor [g, w, ...] of any
    type, or a list of them, each moved; behind (g, w) its dimensions may be
    strided as far as they are a contiguous run and two strided dimensions (a
    slice of a cache's positions, or layers and heads). ``parents`` int32 [g, k], as
    :func:`beam_select` returns; a parent outside [0, w) gives zeros. Without
    ``out`` new tensors [g, k, ...] are returned; ``out`` gives the targets,
    and may be ``states`` itself: in place (k <= w; beams from k on stay as they were).
    Slices of one array (keys and values) may be states and targets side by
    side; other overlaps are refused. ``stream`` as in :func:`quantize_rows`."""
    torch = _get_torch()
    one = torch.is_tensor(states)
    srcs = [states] if one else list(states)
    if parents.dim() != 2 or parents.dtype != torch.int32:
        _fail("reorder_states: parents must be int32 [g, k]")
    g, k = parents.shape
    dev, index = _on_cuda("reorder_states", parents, *srcs)
    if not srcs:
        return []
    w = srcs[0].shape[1] if srcs[0].dim() > 1 else 0
    for s in srcs:
        if s.dim() < 2 or s.shape[0] != g or s.shape[1] != w:
            _fail("reorder_states: every state must be [g, w, ...] with the groups of parents")
    if out is not None:
        dsts = [out] if torch.is_tensor(out) else list(out)
        _check_targets(srcs, dsts, parents, g, k)
    if stream is not None:
        with _stream_scope(dev, stream):
            return reorder_states(srcs[0] if one else srcs, parents, None if out is None else dsts)
    if out is None:
        # the memory of a conjugate or negative view holds other values
        srcs = [s.resolve_conj().resolve_neg() for s in srcs]
        dsts = [torch.empty(g, k, *s.shape[2:], dtype=s.dtype, device=dev) for s in srcs]
    table = []
    for s, d in zip(srcs, dsts):
        lay = _state_layout(s, d)
        if lay is None:
            _fail("reorder_states: a state has more than two strided dimensions behind (g, w)")
        size, ss, ds, row = lay
        es, a, b = s.element_size(), s.stride(), d.stride()
        table += [s.data_ptr(), d.data_ptr(), a[0] * es, a[1] * es, *ss, b[0] * es, b[1] * es, *ds, *size, row]
    parents = parents.contiguous()
    _check(lib.gann_reorder_states((C.c_int64 * len(table))(*table), len(srcs), parents.data_ptr(), g, w, k, index,
                                   torch._C._cuda_getCurrentRawStream(index)))
    return dsts[0] if one else dsts


def _check_targets(srcs, dsts, parents, g, k):
    if len(dsts) != len(srcs):
        _fail("reorder_states: one target for each state")
    _on_cuda("reorder_states", parents, *dsts)
    for s, d in zip(srcs, dsts):
        same = d.data_ptr() == s.data_ptr() and d.shape == s.shape and d.stride() == s.stride()
        if d.dtype != s.dtype or d.shape != ((g,) + (s.shape[1] if same else k,) + s.shape[2:]):
            _fail("reorder_states: a target must be [g, k, ...] of its state's type, or the state itself")
        if d.is_conj() != s.is_conj() or d.is_neg() != s.is_neg():
            _fail("reorder_states: a state and its target must both be conjugate (or negative) views or neither")
        if same and k > s.shape[1]:
            _fail("reorder_states: in place needs k <= w")
        # in place a group's rows are read before any is written, so no other
        # group's may lie among them, in beams that are only read neither
        if not _apart(d) or (d.data_ptr() == s.data_ptr() and not _apart(s)):
            _fail("reorder_states: elements of a target share memory")
    # every target apart from every other array, but for its own state in place
    spans = sorted([(*_extent(d), i, True) for i, d in enumerate(dsts)] +
                   [(*_extent(s), i, False) for i, s in enumerate(srcs)] + [(*_extent(parents), -1, False)])
    before = []   # those that end behind the start of the present one
    for a, b, i, target in spans:
        if b == a:
            continue
        t = parents if i < 0 else dsts[i] if target else srcs[i]
        before = [x for x in before if x[0] > a]
        for _, j, other, u in before:
            own = i == j and dsts[i].data_ptr() == srcs[i].data_ptr()
            if (target or other) and not own and not _disjoint(t, u):
                _fail("reorder_states: a target overlaps another array")
        before.append((b, i, target, t))


def pivot_sample(n: int, s: int, seed: int = 114514) -> np.ndarray:
    """Sorted pivot-graph sample ids (``bin/gen_small_file.cpp:18-40`` sampling)."""
    out = np.zeros(s, np.int32)
    _check(lib.gann_pivot_sample(n, s, seed, _ptr(out)))
    return out
