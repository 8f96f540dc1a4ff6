"""ctypes binding of ``libspork_b200.so`` for torch tensors.

Function names follow the reference's launch functions (``matmul_sm90`` /
``matmul_sm80_supports`` / ``matmul_baseline`` in gemm/gemm_sm90.h:14,
gemm/gemm_sm80.h:5-6, gemm/gemm_baseline.h:5); argument meaning is that of the
harness's hot call ``GPU_Tensors{M,N,K,d_a,d_bCol,d_c,0,1,0}``
(gemm/gemm_test.cu:365): ``a`` is (M, K), ``b`` is (N, K), both fp16 and
contiguous; ``c`` is (M, N) fp32.
"""
from __future__ import annotations

import contextlib
import ctypes
import os
import struct
import threading

_HERE = os.path.dirname(os.path.abspath(__file__))
# SPORK_B200_LIBRARY selects another build of the library (the range-checked debug build
# libspork_b200_checked.so of `python -m spork_b200.build --checked`).
_LIB_PATH = os.environ.get("SPORK_B200_LIBRARY") or os.path.join(_HERE, "libspork_b200.so")

# Fixture codes of init_test_data: 0..2 are the reference's TestDataCode (gemm/gemm_test.h:6-11).
DATA_RANDOM, DATA_IDENTITY, DATA_TILED_NUMBERS, DATA_UNIFORM_PM1, DATA_NORMAL, DATA_NORMAL_BM = range(6)
# The reference's two hash constants (gemm/gemm_test.cu:73,86) seed the A and B operands.
SEED_A = 20010106
SEED_B = 19980724

ERR_BASE = 10000
_ERR_NAMES = {
    10001: "bad argument (null or misaligned pointer, unknown variant)",
    10002: "unsupported shape (GEMM: K must be a multiple of 8; attention: see the entry point's head dimensions and page sizes)",
    10003: "current device is not an sm_100 (B200-class) GPU",
    10004: "driver call failed (tensor map encode)",
    10005: "a bounded device-side wait ran out",
    10006: "size beyond the fixed capacity of this entry point",
    10007: "a range check of the debug build failed on the device",
}


class SporkError(RuntimeError):
    def __init__(self, code: int, what: str):
        self.code = code
        detail = _ERR_NAMES.get(code, f"cudaError_t {code}" if code < ERR_BASE else "unknown")
        super().__init__(f"{what} failed with code {code}: {detail}")


def library_path() -> str:
    return _LIB_PATH


_lib = None


def lib() -> ctypes.CDLL:
    """Load the C-ABI library; raises (never falls back) if it has not been built."""
    global _lib
    if _lib is None:
        if not os.path.exists(_LIB_PATH):
            raise FileNotFoundError(
                f"{_LIB_PATH} is missing: build it with `python -m spork_b200.build` (needs nvcc); "
                "there is no CPU fallback")
        L = ctypes.CDLL(_LIB_PATH)
        u32, i32, vp = ctypes.c_uint32, ctypes.c_int, ctypes.c_void_p
        L.spork_gemm_sm100_supports.argtypes = [u32, u32, u32]
        L.spork_gemm_sm100_supports.restype = i32
        L.spork_gemm_sm100_f16f32.argtypes = [u32, u32, u32, vp, vp, vp, i32, vp]
        L.spork_gemm_sm100_f16f32.restype = i32
        L.spork_gemm_sm100_tf32f32.argtypes = [u32, u32, u32, vp, vp, vp, i32, i32, vp]
        L.spork_gemm_sm100_tf32f32.restype = i32
        L.spork_gemm_sm100_f16f32_ex.argtypes = [u32, u32, u32, vp, vp, vp, i32, i32, i32, i32, vp]
        L.spork_gemm_sm100_f16f32_ex.restype = i32
        L.spork_gemm_sm100_f16f32_batched.argtypes = [u32, u32, u32, u32, vp, vp, vp, i32, i32, vp]
        L.spork_gemm_sm100_f16f32_batched.restype = i32
        L.spork_gemm_sm100_f16f32_static.argtypes = [u32, u32, u32, vp, vp, vp, i32, vp]
        L.spork_gemm_sm100_f16f32_static.restype = i32
        L.spork_selftest_bounded_wait.argtypes = [u32, vp]
        L.spork_selftest_bounded_wait.restype = i32
        L.spork_selftest_range_check.argtypes = [i32, vp]
        L.spork_selftest_range_check.restype = i32
        L.spork_gemm_sm100_last_clock_mhz.argtypes = [vp, ctypes.POINTER(ctypes.c_double)]
        L.spork_gemm_sm100_last_clock_mhz.restype = i32
        L.spork_gemm_sm100_tune.argtypes = [i32, i32, i32, i32]
        L.spork_gemm_sm100_tune.restype = i32
        L.spork_gemm_sm100_ring_model.argtypes = [u32, u32, u32, i32, i32, i32, i32, i32, i32, i32, u32, u32, i32,
                                                  ctypes.POINTER(ctypes.c_uint64)]
        L.spork_gemm_sm100_ring_model.restype = i32
        L.spork_gemm_sm100_choice.argtypes = [u32, u32, u32, i32, i32, i32, i32, ctypes.POINTER(i32)]
        L.spork_gemm_sm100_choice.restype = i32
        L.spork_gemm_sm100_tmap_cache_stats.argtypes = [ctypes.POINTER(ctypes.c_uint64), ctypes.POINTER(ctypes.c_uint64)]
        L.spork_gemm_sm100_tmap_cache_stats.restype = i32
        L.spork_gemm_sm100_stream_k_counters.argtypes = [ctypes.POINTER(u32), vp]
        L.spork_gemm_sm100_stream_k_counters.restype = i32
        L.spork_gemm_sm100_trace.argtypes = [vp, u32]
        L.spork_gemm_sm100_trace.restype = i32
        L.spork_gemm_sm100_tuning.argtypes = [ctypes.POINTER(i32), i32]
        L.spork_gemm_sm100_tuning.restype = i32
        L.spork_gemm_sm100_status.argtypes = [vp, ctypes.POINTER(u32)]
        L.spork_gemm_sm100_status.restype = i32
        L.spork_gemm_sm100_htod_f16f32.argtypes = [u32, u32, u32, vp, vp, vp]
        L.spork_gemm_sm100_htod_f16f32.restype = i32
        L.spork_init_test_data_f16.argtypes = [vp, u32, u32, i32, u32, i32, vp]
        L.spork_init_test_data_f16.restype = i32
        L.spork_init_test_data_f16_at.argtypes = [vp, u32, u32, i32, u32, i32, u32, u32, vp]
        L.spork_init_test_data_f16_at.restype = i32
        L.spork_gemm_baseline_f16f32.argtypes = [u32, u32, u32, vp, vp, vp, vp]
        L.spork_gemm_baseline_f16f32.restype = i32
        L.spork_compare_f32.argtypes = [vp, vp, u32, u32, vp, vp]
        L.spork_compare_f32.restype = i32
        if hasattr(L, "spork_attn_sm100_fwd_f16"):
            L.spork_attn_sm100_supports.argtypes = [i32, i32, i32]
            L.spork_attn_sm100_supports.restype = i32
            L.spork_attn_sm100_fwd_f16.argtypes = [i32, i32, i32, vp, vp, vp, vp, ctypes.c_float, vp]
            L.spork_attn_sm100_fwd_f16.restype = i32
            L.spork_attn_sm100_fwd_bf16.argtypes = [i32, i32, i32, vp, vp, vp, vp, ctypes.c_float, vp]
            L.spork_attn_sm100_fwd_bf16.restype = i32
            L.spork_attn_sm100_fwd_ex.argtypes = [i32, i32, i32, vp, vp, vp, vp, ctypes.c_float, i32, i32, vp]
            L.spork_attn_sm100_fwd_ex.restype = i32
            L.htod_f32_attn_sm100_fwd.argtypes = [i32, i32, vp, vp, vp, vp]
            L.htod_f32_attn_sm100_fwd.restype = None
        cp = ctypes.c_char_p  # packed argument structures: read before the call returns
        L.spork_paged_sm100_tables.argtypes = [cp, vp]
        L.spork_paged_sm100_tables.restype = i32
        L.spork_paged_sm100_store.argtypes = [cp, vp]
        L.spork_paged_sm100_store.restype = i32
        L.spork_attn_sm100_paged.argtypes = [cp, vp]
        L.spork_attn_sm100_paged.restype = i32
        L.spork_attn_sm100_paged_supports.argtypes = [i32, i32, i32, i32]
        L.spork_attn_sm100_paged_supports.restype = i32
        L.spork_attn_sm100_paged_workspace.argtypes = [i32, i32, i32]
        L.spork_attn_sm100_paged_workspace.restype = ctypes.c_int64
        L.spork_attn_sm100_paged_plan.argtypes = [ctypes.POINTER(i32)] + [i32] * 8 + [ctypes.POINTER(i32), i32]
        L.spork_attn_sm100_paged_plan.restype = i32
        L.spork_b200_version.restype = ctypes.c_char_p
        _lib = L
    return _lib


def version() -> str:
    return lib().spork_b200_version().decode()


def _check(rc: int, what: str) -> None:
    if rc != 0:
        raise SporkError(rc, what)


def _stream_ptr(stream) -> int:
    import torch

    if stream is None:
        stream = torch.cuda.current_stream()
    return int(stream.cuda_stream)


def _dev_ptr(t, dtype, what: str) -> int:
    import torch

    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise TypeError(f"{what} must be a CUDA tensor")
    if t.dtype != dtype:
        raise TypeError(f"{what} must be {dtype}, got {t.dtype}")
    if not t.is_contiguous():
        raise ValueError(f"{what} must be contiguous")
    return int(t.data_ptr())


class _OnDevice:
    """``with _OnDevice(t.device)``: the launch runs with that GPU current.  Nothing is switched (and nothing
    is paid) when it already is, the usual case."""

    __slots__ = ("_ctx",)

    def __init__(self, device):
        import torch

        index = device if isinstance(device, int) else torch.device(device).index
        current = torch.cuda.current_device()
        self._ctx = None if index is None or index == current else torch.cuda.device(index)

    def __enter__(self):
        if self._ctx is not None:
            self._ctx.__enter__()
        return self

    def __exit__(self, *exc):
        if self._ctx is not None:
            return self._ctx.__exit__(*exc)
        return False


def _same_device(first, *others) -> None:
    """All operands of a launch must live on one GPU: the kernel runs on the first one's device and would
    otherwise read or write addresses that mean nothing there."""
    for t in others:
        if t.device != first.device:
            raise ValueError(f"tensors are on different devices: {first.device} and {t.device}")


def matmul_sm100_supports(M: int, N: int, K: int) -> bool:
    return bool(lib().spork_gemm_sm100_supports(M, N, K))


def matmul_sm100(a, b, c=None, *, variant: int = 0, block_n: int | None = None, cta_group: int | None = None,
                 split_k: int = 1, max_ctas: int = 0, stream=None):
    """c[M,N] (fp32) = a[M,K] (fp16) @ b[N,K]^T (fp16); asynchronous on ``stream``.

    ``variant`` 0/64/128/256 picks the output-tile width like the reference's
    n64/n128/n256 kernels.  ``block_n``/``cta_group``/``split_k``/``max_ctas``
    select the explicit-tunables entry point instead; ``split_k=0`` alone leaves
    tile and K mode (whole tiles, split-K or stream-K) to the library.
    """
    import torch

    M, K = a.shape
    N, K2 = b.shape
    if K != K2:
        raise ValueError(f"inner dimensions differ: a is {tuple(a.shape)}, b is {tuple(b.shape)}")
    if c is None:
        c = torch.empty((M, N), dtype=torch.float32, device=a.device)
    if tuple(c.shape) != (M, N):
        raise ValueError(f"c must be {(M, N)}, got {tuple(c.shape)}")
    _same_device(a, b, c)
    pa = _dev_ptr(a, torch.float16, "a")
    pb = _dev_ptr(b, torch.float16, "b")
    pc = _dev_ptr(c, torch.float32, "c")
    with _OnDevice(a.device):
        sp = _stream_ptr(stream)
        if block_n is None and cta_group is None and split_k == 1 and max_ctas == 0:
            rc = lib().spork_gemm_sm100_f16f32(M, N, K, pa, pb, pc, variant, sp)
        else:
            bn = block_n if block_n is not None else (variant or (64 if N <= 64 else 128 if N <= 128 else 256))
            cg = cta_group or 2
            if block_n is None and cta_group is None and variant == 0 and split_k == 0:
                cg = 0  # fully automatic: the library picks the tile and the K mode
            rc = lib().spork_gemm_sm100_f16f32_ex(M, N, K, pa, pb, pc, bn, cg, split_k, max_ctas, sp)
    _check(rc, "spork_gemm_sm100_f16f32")
    return c


def matmul_sm100_batched(a, b, c=None, *, variant: int = 0, split_k: int = 1, stream=None):
    """c[L,M,N] (fp32) = a[L,M,K] (fp16) @ b[L,N,K]^T (fp16), one launch for the whole batch.

    The batch dimension of the reference's generated entry points (xgemm_Sm90.py:45-48).
    """
    import torch

    L, M, K = a.shape
    L2, N, K2 = b.shape
    if K != K2 or L != L2:
        raise ValueError(f"shapes do not match: a is {tuple(a.shape)}, b is {tuple(b.shape)}")
    if c is None:
        c = torch.empty((L, M, N), dtype=torch.float32, device=a.device)
    if tuple(c.shape) != (L, M, N):
        raise ValueError(f"c must be {(L, M, N)}, got {tuple(c.shape)}")
    _same_device(a, b, c)
    pa = _dev_ptr(a, torch.float16, "a")
    pb = _dev_ptr(b, torch.float16, "b")
    pc = _dev_ptr(c, torch.float32, "c")
    with _OnDevice(a.device):
        rc = lib().spork_gemm_sm100_f16f32_batched(L, M, N, K, pa, pb, pc, variant, split_k, _stream_ptr(stream))
    _check(rc, "spork_gemm_sm100_f16f32_batched")
    return c


def matmul_sm100_tf32(a, b, c=None, *, variant: int = 0, split_k: int = 1, stream=None):
    """c[M,N] = a[M,K] @ b[N,K]^T with fp32 operands read as tf32 (the reference's own operand type)."""
    import torch

    M, K = a.shape
    N, K2 = b.shape
    if K != K2:
        raise ValueError(f"inner dimensions differ: a is {tuple(a.shape)}, b is {tuple(b.shape)}")
    if c is None:
        c = torch.empty((M, N), dtype=torch.float32, device=a.device)
    if tuple(c.shape) != (M, N):
        raise ValueError(f"c must be {(M, N)}, got {tuple(c.shape)}")
    _same_device(a, b, c)
    pa, pb, pc = (_dev_ptr(t, torch.float32, n) for t, n in ((a, "a"), (b, "b"), (c, "c")))
    with _OnDevice(a.device):
        rc = lib().spork_gemm_sm100_tf32f32(M, N, K, pa, pb, pc, variant, split_k, _stream_ptr(stream))
    _check(rc, "spork_gemm_sm100_tf32f32")
    return c


def last_clock_mhz(stream=None) -> float:
    """SM clock the most recent GEMM or attention launch on the current device ran at (measured inside the kernel)."""
    mhz = ctypes.c_double(0.0)
    _check(lib().spork_gemm_sm100_last_clock_mhz(_stream_ptr(stream), ctypes.byref(mhz)), "last_clock_mhz")
    return float(mhz.value)


def tune(stages: int = 0, group_m: int = 0, l2_hints: int = 0, backoff_ns: int = 0, *, experiment: int = 0,
         k_atoms: int = 0, wide: int = 0, wide_skew: int = 0, wide_group_m: int = 0,
         no_early_launch: bool = False, keep_wide_tiles: bool = False) -> None:
    """Process-wide tuning knobs of later GEMM launches (see spork_gemm_sm100_tune in the header).

    ``l2_hints`` may carry the packed upper bits itself (the C form); the keyword arguments are OR-ed in."""
    packed = l2_hints | ((experiment & 15) << 4) | ((k_atoms & 3) << 8) | ((wide & 3) << 10) | \
        ((wide_skew & 15) << 12) | ((wide_group_m & 255) << 16) | (int(bool(no_early_launch)) << 24) | \
        (int(bool(keep_wide_tiles)) << 25)
    _check(lib().spork_gemm_sm100_tune(stages, group_m, packed, backoff_ns), "spork_gemm_sm100_tune")


def ring_model(M: int, N: int, K: int, *, block_n: int = 256, cta_group: int = 2, split_k: int = 1, max_ctas: int = 0,
               sm_count: int = 148, stages: int | None = None, skew: int = 4, seed: int = 0, group: int = 0,
               inject: int = 0):
    """Run the host-side model of the kernels' barrier protocol for one CTA group of a launch plan
    (spork_gemm_sm100_ring_model); returns (code, stats) with code 0 = every invariant held."""
    if stages is None:
        stages = 4 if block_n == 512 else 6
    stats = (ctypes.c_uint64 * 4)()
    rc = lib().spork_gemm_sm100_ring_model(M, N, K, block_n, cta_group, split_k, max_ctas, sm_count, stages, skew, seed,
                                           group, inject, stats)
    return rc, {"items": int(stats[0]), "mma_ops": int(stats[1]), "steps": int(stats[2]), "groups": int(stats[3])}


def choice(M: int, N: int, K: int, *, variant: int = 0, split_k: int = 1, sm_count: int = 148, tf32: bool = False) -> dict:
    """What a launch of this shape resolves to (tile width, CTAs per tile, column blocks per stage, K split),
    computed without a GPU (spork_gemm_sm100_choice)."""
    out = (ctypes.c_int * 4)()
    _check(lib().spork_gemm_sm100_choice(M, N, K, variant, split_k, sm_count, int(tf32), out), "spork_gemm_sm100_choice")
    return {"block_n": int(out[0]), "cta_group": int(out[1]), "k_atoms": int(out[2]), "split_k": int(out[3])}


def tmap_cache_stats() -> tuple[int, int]:
    """(hits, misses) of the per-thread cache of encoded TMA descriptors, summed over the process."""
    h, m = ctypes.c_uint64(0), ctypes.c_uint64(0)
    _check(lib().spork_gemm_sm100_tmap_cache_stats(ctypes.byref(h), ctypes.byref(m)), "spork_gemm_sm100_tmap_cache_stats")
    return int(h.value), int(m.value)


def stream_k_counters(stream=None) -> list[tuple[int, int]]:
    """The 16 counter pairs stream-K launches meet at, after ``stream`` has drained: all zero unless a launch
    gave up half way (see spork_gemm_sm100_stream_k_counters)."""
    out = (ctypes.c_uint32 * 32)()
    _check(lib().spork_gemm_sm100_stream_k_counters(out, _stream_ptr(stream)), "spork_gemm_sm100_stream_k_counters")
    return [(int(out[2 * i]), int(out[2 * i + 1])) for i in range(16)]


def trace(buffer=None) -> None:
    """Switch the tile hand-over trace of the 256 x 512 kernel on (``buffer``: an int64 CUDA tensor of
    8 * items elements that outlives the traced launches) or off (None).  See spork_gemm_sm100_trace."""
    import torch

    if buffer is None:
        _check(lib().spork_gemm_sm100_trace(None, 0), "spork_gemm_sm100_trace")
        return
    if not buffer.is_cuda or buffer.dtype != torch.int64 or not buffer.is_contiguous() or buffer.numel() < 8:
        raise TypeError("the trace buffer must be a contiguous int64 CUDA tensor of at least 8 elements")
    _check(lib().spork_gemm_sm100_trace(int(buffer.data_ptr()), buffer.numel() // 8), "spork_gemm_sm100_trace")


def tuning() -> dict:
    """The knobs as the next launch will see them (``l2_hints`` is the effective hint mask)."""
    out = (ctypes.c_int * 10)()
    _check(lib().spork_gemm_sm100_tuning(out, 10), "spork_gemm_sm100_tuning")
    keys = ("stages", "group_m", "l2_hints", "backoff_ns", "experiment", "k_atoms", "wide", "wide_skew", "wide_group_m",
            "no_early_launch")
    return dict(zip(keys, (int(v) for v in out)))


def status(stream=None, device=None) -> None:
    """Synchronise ``stream`` and raise SporkError if a kernel reported a device-side timeout."""
    import torch

    with _OnDevice(device if device is not None else torch.cuda.current_device()):
        detail = ctypes.c_uint32(0)
        rc = lib().spork_gemm_sm100_status(_stream_ptr(stream), ctypes.byref(detail))
    if rc != 0:
        # a launch that was given up may have left its counters as they were
        _workspaces.clear()
        with _lent_lock:
            for pool in _lent.values():
                for entry in pool:
                    entry.clean = False
        raise SporkError(rc, f"device status (detail 0x{detail.value:08x})")


def matmul_sm100_htod(a_host, b_host, c_host=None):
    """Host-buffer GEMM: fp16 CPU tensors in, fp32 CPU tensor out (copies inside the call)."""
    import torch

    M, K = a_host.shape
    N, _ = b_host.shape
    if c_host is None:
        c_host = torch.empty((M, N), dtype=torch.float32)
    for t, dt in ((a_host, torch.float16), (b_host, torch.float16), (c_host, torch.float32)):
        if t.is_cuda or t.dtype != dt or not t.is_contiguous():
            raise TypeError("host tensors must be contiguous CPU tensors (fp16, fp16, fp32)")
    rc = lib().spork_gemm_sm100_htod_f16f32(M, N, K, a_host.data_ptr(), b_host.data_ptr(), c_host.data_ptr())
    _check(rc, "spork_gemm_sm100_htod_f16f32")
    return c_host


def init_test_data(t, code: int, seed: int = 0, transpose_rule: bool = False, stream=None, row0: int = 0,
                   col0: int = 0):
    """Fill the 2-D fp16 CUDA tensor ``t`` with fixture ``code`` (gemm/gemm_test.cu:55-96 plus codes 3, 4).

    ``row0``/``col0`` place ``t`` inside a larger logical matrix (a rank's slab of a sharded operand)."""
    import torch

    rows, cols = t.shape
    with _OnDevice(t.device):
        rc = lib().spork_init_test_data_f16_at(_dev_ptr(t, torch.float16, "t"), rows, cols, code, seed & 0xFFFFFFFF,
                                               int(transpose_rule), row0, col0, _stream_ptr(stream))
    _check(rc, "spork_init_test_data_f16")
    return t


def gemm_baseline(a, b, c=None, stream=None):
    """The slow CUDA-core comparison GEMM (same operand layout as matmul_sm100)."""
    import torch

    M, K = a.shape
    N, _ = b.shape
    if c is None:
        c = torch.empty((M, N), dtype=torch.float32, device=a.device)
    with _OnDevice(a.device):
        rc = lib().spork_gemm_baseline_f16f32(M, N, K, _dev_ptr(a, torch.float16, "a"), _dev_ptr(b, torch.float16, "b"),
                                              _dev_ptr(c, torch.float32, "c"), _stream_ptr(stream))
    _check(rc, "spork_gemm_baseline_f16f32")
    return c


def compare_f32(x, y, stream=None):
    """On-device comparison; returns (first_failure or None, max_abs_diff) like the reference's comparator."""
    import torch

    rows, cols = x.shape
    out = torch.empty(2, dtype=torch.int64, device=x.device)
    with _OnDevice(x.device):
        rc = lib().spork_compare_f32(_dev_ptr(x, torch.float32, "x"), _dev_ptr(y, torch.float32, "y"), rows, cols,
                                     int(out.data_ptr()), _stream_ptr(stream))
    _check(rc, "spork_compare_f32")
    packed, diff_bits = (int(v) & 0xFFFFFFFFFFFFFFFF for v in out.cpu().tolist())
    first = None if packed == 0xFFFFFFFFFFFFFFFF else (packed >> 32, packed & 0xFFFFFFFF)
    max_diff = struct.unpack("<d", struct.pack("<Q", diff_bits))[0]
    return first, max_diff


def attn_fwd(q, k, v, o=None, scale: float | None = None, stream=None, causal: bool = False):
    """o = softmax(q k^T scale) v per head; q, k, v are (BH, S, D) CUDA tensors, all fp16 or all bfloat16
    (the reference interface's type)."""
    import torch

    if q.dim() != 3:
        raise ValueError(f"q must be (BH, S, D), got {tuple(q.shape)}")
    BH, S, D = q.shape
    if o is None:
        o = torch.empty_like(q)
    # every tensor map and every store is sized from q: a shorter k or v, or a smaller o, would be read or
    # written past its end
    for t, name in ((k, "k"), (v, "v"), (o, "o")):
        if tuple(t.shape) != (BH, S, D):
            raise ValueError(f"{name} must have q's shape {(BH, S, D)}, got {tuple(t.shape)}")
    _same_device(q, k, v, o)
    if scale is None:
        scale = 1.0 / (D ** 0.5)
    dt = q.dtype
    if dt not in (torch.float16, torch.bfloat16):
        raise TypeError(f"q must be float16 or bfloat16, got {dt}")
    with _OnDevice(q.device):
        rc = lib().spork_attn_sm100_fwd_ex(BH, S, D, _dev_ptr(q, dt, "q"), _dev_ptr(k, dt, "k"), _dev_ptr(v, dt, "v"),
                                           _dev_ptr(o, dt, "o"), ctypes.c_float(scale), int(dt == torch.bfloat16),
                                           int(bool(causal)), _stream_ptr(stream))
    _check(rc, "spork_attn_sm100_fwd")
    return o


# --------------------------------------------------------------------------- paged key-value cache

# The argument structures of include/spork_b200.h (spork_paged_cache inside the last two), packed by hand: a call of a
# few microseconds on the GPU should not wait for ctypes to convert thirty arguments.
_CACHE = "QQ6q6i"
_TABLES_ARGS = struct.Struct("=9Q2q4i")
_STORE_ARGS = struct.Struct("=" + _CACHE + "3Q5q2i")
_PAGED_ATTN_ARGS = struct.Struct("=" + _CACHE + "6Q4q4ifi")
# torch, its types' codes and its unwrapped calls, once a call below has needed them: these functions stand in front of
# kernels of a few microseconds, so they look each property of a tensor up once and call as little as they can
_T = None
_TYPE_CODES: dict = {}
_CACHE_TYPES: set = set()
_current_device = _raw_stream = _capturing = None
_workspace_bytes: dict = {}  # by device and what the size depends on
_workspaces: dict = {}       # by device and stream of torch's: the one that calls without a workspace of their own use
_lent: dict = {}             # by device: those that calls on other streams take turns with
_lent_lock = threading.Lock()
_LENT = 4                    # of a device, at most
_COUNTER_BYTES = 65536       # SPORK_ATTN_PAGED_COUNTERS


def _bind_torch():
    global _T, _current_device, _raw_stream, _capturing
    import torch

    _TYPE_CODES.update({torch.float16: 0, torch.bfloat16: 1, torch.float32: 2})
    _CACHE_TYPES.update((torch.float16, torch.bfloat16))
    _current_device, _raw_stream = torch._C._cuda_getDevice, torch._C._cuda_getCurrentRawStream
    _capturing = torch._C._cuda_isCurrentStreamCapturing
    _T = torch
    return torch


def _on_gpu(**tensors) -> None:
    """Raise for the tensor that is not where the first one is, on one GPU."""
    device = None
    for name, t in tensors.items():
        if not t.is_cuda:
            raise TypeError(f"{name} must be a CUDA tensor")
        if device is None:
            first, device = name, t.get_device()
        if t.get_device() != device:
            raise ValueError(f"tensors are on different devices: {first} on {device}, {name} on {t.get_device()}")


def _stream_of(stream, device: int) -> int:
    """The given stream, which must be of the tensors' device, or that device's current one."""
    if stream is None:
        return _raw_stream(device)
    if stream.device_index != device:
        raise ValueError(f"the stream is of device {stream.device_index}, the tensors of device {device}")
    return stream.cuda_stream


def _call(fn, packed: bytes, device: int, stream: int, what: str) -> None:
    if _current_device() == device:
        rc = fn(packed, stream)
    else:
        with _T.cuda.device(device):
            rc = fn(packed, stream)
    if rc:
        raise SporkError(rc, what)


def _new(like, shape, dtype, stream):
    """An output or scratch tensor that belongs to the stream of the launch."""
    if stream is None:
        return _T.empty(shape, dtype=dtype, device=like.device)
    with _T.cuda.stream(stream):
        return _T.empty(shape, dtype=dtype, device=like.device)


class _Lent:
    """A workspace with the event of its last use, and the handle of the stream that this was on."""

    __slots__ = ("workspace", "used", "handle", "clean")


def _whose_turn(pool: list, handle: int) -> _Lent:
    """The pool's workspace for a launch on the stream of that handle: the one that it had last, a new one (which has no
    memory yet), or the one that was not used for the longest time.  The pool is kept in the order of use."""
    entry = next((e for e in pool if e.handle == handle), None)
    if entry is not None:
        pool.remove(entry)
    elif len(pool) >= _LENT:
        entry = pool.pop(0)
    else:
        entry = _Lent()
        entry.workspace = entry.used = None
        entry.clean = False
    entry.handle = handle
    pool.append(entry)
    return entry


@contextlib.contextmanager
def _lent_workspace(like, device: int, stream):
    """A workspace for one launch on a stream that torch did not make.  What its handle stands for may change: one of a stream
    that was destroyed comes back, and that of the per-thread default stream means another stream in every thread.  So the
    launches that use a workspace are put in order by an event, whatever their streams, and one is large enough for all
    shapes and is never freed."""
    torch = _T
    with _lent_lock, torch.cuda.device(device):
        if stream is None:
            stream = torch.cuda.current_stream()
        with torch.cuda.stream(stream):
            entry = _whose_turn(_lent.setdefault(device, []), stream.cuda_stream)
            if entry.workspace is None:
                entry.used = torch.cuda.Event()
                entry.workspace = torch.empty((attn_paged_workspace(32, 1, 128),), dtype=torch.uint8, device=like.device)
            else:
                stream.wait_event(entry.used)
            if not entry.clean:
                entry.workspace[:_COUNTER_BYTES].zero_()
                entry.clean = True
            try:
                yield entry.workspace
            finally:
                entry.used.record(stream)


def _own_workspace(like, device: int, stream, key):
    """The workspace of one launch that was not given any; None for one on a stream that torch did not make.  Launches of one
    stream follow one another and share the stream's; a captured launch, whose graph may be replayed beside any other, gets
    one of its own, with the clearing of its counters in the graph."""
    if stream is not None:
        with _T.cuda.stream(stream):
            return _own_workspace(like, device, None, key)
    if _current_device() != device:
        with _T.cuda.device(device):
            return _own_workspace(like, device, None, key)
    need = _workspace_bytes.get(key)
    if need is None:
        need = _workspace_bytes[key] = attn_paged_workspace(*key[1:])
    if _capturing():
        workspace = _T.empty((need,), dtype=_T.uint8, device=like.device)
        workspace[:_COUNTER_BYTES].zero_()
        return workspace
    at = (device, _raw_stream(device))
    workspace = _workspaces.get(at)
    if workspace is None and at[1] and _T.cuda.current_stream(device).stream_id == at[1]:
        return None  # (torch names its own streams otherwise than by their handles, which stay theirs)
    if workspace is None or workspace.numel() < need:
        workspace = _workspaces[at] = _T.zeros((need,), dtype=_T.uint8, device=like.device)
    return workspace


def _vector(t, n, dtype, what: str):
    """Raise unless t is a contiguous 1-D tensor of n elements (any number where n is None)."""
    shape = t.shape
    if len(shape) != 1 or (n is not None and shape[0] != n):
        raise ValueError(f"{what} must be ({'n' if n is None else n},), got {tuple(shape)}")
    if t.dtype is not dtype:
        raise TypeError(f"{what} must be {dtype}, got {t.dtype}")
    if not t.is_contiguous():
        raise ValueError(f"{what} must be contiguous")
    return t


def _block_table(t, requests: int):
    """(requests, max_blocks) int32, columns contiguous; returns max_blocks and the row stride."""
    shape = t.shape
    if len(shape) != 2 or shape[0] != requests:
        raise ValueError(f"block_table must be ({requests}, max_blocks), got {tuple(shape)}")
    if t.dtype is not _T.int32:
        raise TypeError(f"block_table must be torch.int32, got {t.dtype}")
    rows, columns = t.stride()
    if columns != 1 and shape[1] > 1:
        raise ValueError("the entries of a block_table row must be contiguous")
    return shape[1], rows


def _pages(k_cache, v_cache):
    """Shape (num_pages, kv_heads, page_size, head_dim), type code, and strides of a cache's two halves."""
    shape, dtype = k_cache.shape, k_cache.dtype
    if len(shape) != 4 or v_cache.shape != shape:
        raise ValueError("k_cache and v_cache must both be (num_pages, kv_heads, page_size, head_dim), got "
                         f"{tuple(shape)} and {tuple(v_cache.shape)}")
    code = _TYPE_CODES.get(dtype, 2)
    if code == 2 or v_cache.dtype is not dtype:
        raise TypeError(f"k_cache and v_cache must both be float16 or both bfloat16, got {dtype} and {v_cache.dtype}")
    ks, vs = k_cache.stride(), v_cache.stride()
    if (ks[3] != 1 or vs[3] != 1) and shape[3] > 1:
        raise ValueError("the head dimension of a cache must be contiguous")
    return shape, code, ks, vs


def paged_tables(lengths, new_tokens, block_table, free_pages, free_used, *, page_size: int, max_tokens: int | None = None,
                 slots=None, offsets=None, lengths_after=None, info=None, stream=None):
    """Give each request the pages that its new tokens need; returns (slots, offsets, lengths_after, info).

    ``lengths`` and ``new_tokens`` (R,), ``block_table`` (R, max_blocks), ``free_pages`` (F,) and ``free_used`` (1,) are
    int32 CUDA tensors.  Request r holds ``lengths[r]`` tokens and gets ``new_tokens[r]`` more; the pages that it lacks come
    from ``free_pages`` in the order of the requests, from entry ``free_used[0]`` on, and are entered into its row of
    ``block_table`` in place.  ``slots`` (int64) names the place in the cache of every new token, request by request, -1
    where there is none: it has ``max_tokens`` entries, so that a launch of one size serves steps of any number of tokens.
    ``offsets`` (R + 1,) says where each request's tokens begin in it.  A request that does not fit (its table row, the
    slot map, the free list) is left as it was, and ``info`` counts it: [free pages used afterwards, tokens, requests
    refused, pages asked for].  The rules in full are beside spork_paged_sm100_tables in include/spork_b200.h.  To go on
    from this step, pass ``lengths_after`` as ``lengths`` and ``info[:1]`` as ``free_used`` (with other outputs: inputs and
    outputs must not overlap)."""
    torch = _T or _bind_torch()
    i32 = torch.int32
    shape = lengths.shape
    if len(shape) != 1:
        raise ValueError(f"lengths must be (R,), got {tuple(shape)}")
    n = shape[0]
    # (looked at together, and one by one only to say what is wrong)
    if not (lengths.dtype is i32 and new_tokens.dtype is i32 and free_pages.dtype is i32 and free_used.dtype is i32
            and new_tokens.shape == shape and lengths.is_contiguous() and new_tokens.is_contiguous()
            and free_pages.is_contiguous() and free_used.shape == (1,) and len(free_pages.shape) == 1):
        _vector(lengths, n, i32, "lengths")
        _vector(new_tokens, n, i32, "new_tokens")
        _vector(free_pages, None, i32, "free_pages")
        _vector(free_used, 1, i32, "free_used")
    blocks, row = _block_table(block_table, n)
    if not 1 <= page_size < 1 << 31:
        raise ValueError(f"page_size must be at least 1 and below 2^31, got {page_size}")
    if slots is None:
        if max_tokens is None or max_tokens < 0:
            raise ValueError("max_tokens (or slots) says how many new tokens there is room for")
        slots = _new(lengths, (max_tokens,), torch.int64, stream)
    else:
        _vector(slots, max_tokens, torch.int64, "slots")
    offsets = _new(lengths, (n + 1,), i32, stream) if offsets is None else _vector(offsets, n + 1, i32, "offsets")
    lengths_after = _new(lengths, (n,), i32, stream) if lengths_after is None else _vector(lengths_after, n, i32, "lengths_after")
    info = _new(lengths, (4,), i32, stream) if info is None else _vector(info, 4, i32, "info")
    device = lengths.get_device()
    if device < 0 or not (device == new_tokens.get_device() == block_table.get_device() == free_pages.get_device()
                          == free_used.get_device() == slots.get_device() == offsets.get_device()
                          == lengths_after.get_device() == info.get_device()):
        _on_gpu(lengths=lengths, new_tokens=new_tokens, block_table=block_table, free_pages=free_pages,
                free_used=free_used, slots=slots, offsets=offsets, lengths_after=lengths_after, info=info)
    packed = _TABLES_ARGS.pack(
        lengths.data_ptr(), new_tokens.data_ptr(), block_table.data_ptr(), free_pages.data_ptr(), free_used.data_ptr(),
        slots.data_ptr(), offsets.data_ptr(), lengths_after.data_ptr(), info.data_ptr(), row, slots.shape[0], n, blocks,
        page_size, free_pages.shape[0])
    _call((_lib or lib()).spork_paged_sm100_tables, packed, device, _stream_of(stream, device), "spork_paged_sm100_tables")
    return slots, offsets, lengths_after, info


def paged_store(k, v, k_cache, v_cache, slots, stream=None):
    """Write the keys and values of T tokens into their slots of the cache (in place).

    ``k`` and ``v`` are (T, kv_heads, head_dim) with the last dimension contiguous (slices of a projection's rows, say), of
    the cache's type or float32 (what the GEMMs write; rounded to nearest even).  ``k_cache`` and ``v_cache`` are (num_pages,
    kv_heads, page_size, head_dim) float16 or bfloat16, the first three dimensions in any order in memory.  ``slots`` (T,)
    int64 is page * page_size + row, as paged_tables gives it; a slot outside the cache (-1) writes nothing, and slots
    inside it must differ from each other.  ``k`` and ``v`` must not overlap the cache, nor its halves each other."""
    torch = _T or _bind_torch()
    shape, code, ks, vs = _pages(k_cache, v_cache)
    pages, kv_heads, page, dim = shape
    tokens = k.shape
    if v.shape != tokens or len(tokens) != 3 or tokens[1] != kv_heads or tokens[2] != dim:
        raise ValueError(f"k and v must both be (T, {kv_heads}, {dim}), got {tuple(tokens)} and {tuple(v.shape)}")
    src = _TYPE_CODES.get(k.dtype)
    if (src != 2 and src != code) or v.dtype is not k.dtype:
        raise TypeError(f"k and v must both be float32 or of the cache's type {k_cache.dtype}, got {k.dtype} and {v.dtype}")
    kn, vn = k.stride(), v.stride()
    if (kn[2] != 1 or vn[2] != 1) and dim > 1:
        raise ValueError("the head dimension of k and v must be contiguous")
    if slots.dtype is not torch.int64 or slots.shape != tokens[:1] or not slots.is_contiguous():
        _vector(slots, tokens[0], torch.int64, "slots")
    device = k_cache.get_device()
    if device < 0 or not (device == v_cache.get_device() == k.get_device() == v.get_device() == slots.get_device()):
        _on_gpu(k_cache=k_cache, v_cache=v_cache, k=k, v=v, slots=slots)
    packed = _STORE_ARGS.pack(
        k_cache.data_ptr(), v_cache.data_ptr(), ks[0], ks[1], ks[2], vs[0], vs[1], vs[2], code, pages, kv_heads, page, dim, 0,
        k.data_ptr(), v.data_ptr(), slots.data_ptr(), kn[0], kn[1], vn[0], vn[1], tokens[0], src, 0)
    _call((_lib or lib()).spork_paged_sm100_store, packed, device, _stream_of(stream, device), "spork_paged_sm100_store")


def attn_paged_supports(heads: int, kv_heads: int, head_dim: int, page_size: int) -> bool:
    return bool(lib().spork_attn_sm100_paged_supports(heads, kv_heads, head_dim, page_size))


def attn_paged_workspace(heads: int, kv_heads: int, head_dim: int) -> int:
    """Bytes of workspace that attn_paged needs on the current device, whatever the requests and their lengths."""
    n = int(lib().spork_attn_sm100_paged_workspace(heads, kv_heads, head_dim))
    if n < 0:
        raise SporkError(-n, "spork_attn_sm100_paged_workspace")
    return n


def attn_paged_plan(lengths, block: int, *, heads: int, kv_heads: int, head_dim: int, page_size: int, max_blocks: int,
                    sm_count: int = 148) -> list[dict]:
    """What one block of an attn_paged launch works on, for lengths known on the host (a sequence of ints); computed without
    a GPU (spork_attn_sm100_paged_plan)."""
    n = len(lengths)
    host = (ctypes.c_int * max(n, 1))(*lengths)
    args = (host, n, heads, kv_heads, head_dim, page_size, max_blocks, sm_count, block)
    count = lib().spork_attn_sm100_paged_plan(*args, None, 0)
    if count < 0:
        raise ValueError("not a launch that attn_paged makes")
    out = (ctypes.c_int * max(9 * count, 1))()
    lib().spork_attn_sm100_paged_plan(*args, out, count)
    keys = ("request", "kv_head", "head_unit", "first", "count", "units", "first_block", "blocks", "slot")
    return [dict(zip(keys, out[9 * i:9 * i + 9])) for i in range(count)]


def _refuse_attn_paged(q, k_cache, v_cache, block_table, lengths, o, lse):
    """Raise for what is wrong with the tensors of an attn_paged call."""
    q_shape = q.shape
    if len(q_shape) != 3:
        raise ValueError(f"q must be (R, heads, head_dim), got {tuple(q_shape)}")
    n, heads, dim = q_shape
    shape, code, _, _ = _pages(k_cache, v_cache)
    if shape[3] != dim:
        raise ValueError(f"q has head dimension {dim}, the cache {shape[3]}")
    if _TYPE_CODES.get(q.dtype) not in (2, code):
        raise TypeError(f"q must be float32 or of the cache's type {k_cache.dtype}, got {q.dtype}")
    if q.stride()[2] != 1:
        raise ValueError("the head dimension of q must be contiguous")
    _block_table(block_table, n)
    _vector(lengths, n, _T.int32, "lengths")
    if o is not None:
        if o.shape != q_shape:
            raise ValueError(f"o must have q's shape {(n, heads, dim)}, got {tuple(o.shape)}")
        if o.dtype is not k_cache.dtype:
            raise TypeError(f"o must be of the cache's type {k_cache.dtype}, got {o.dtype}")
        if not o.is_contiguous():
            raise ValueError("o must be contiguous")
    if lse is not None:
        if lse.shape != (n, heads) or not lse.is_contiguous():
            raise ValueError(f"lse must be a contiguous ({n}, {heads}), got {tuple(lse.shape)}")
        if lse.dtype is not _T.float32:
            raise TypeError(f"lse must be torch.float32, got {lse.dtype}")
    _on_gpu(q=q, k_cache=k_cache, v_cache=v_cache, block_table=block_table, lengths=lengths,
            **{name: t for name, t in (("o", o), ("lse", lse)) if t is not None})
    raise ValueError("q, the cache and the block table do not fit together")


def attn_paged(q, k_cache, v_cache, block_table, lengths, o=None, *, lse=None, scale: float | None = None, workspace=None,
               stream=None):
    """o[r] = softmax(scale q[r] K^T) V over the first ``lengths[r]`` keys that request r holds in the cache.

    One new token per request: ``q`` is (R, heads, head_dim) of the cache's type or float32, with the last dimension
    contiguous; ``heads`` is a multiple of kv_heads, and query head h reads key head h // (heads // kv_heads).  ``k_cache``
    and ``v_cache`` are (num_pages, kv_heads, page_size, head_dim), the first three dimensions in any order in memory;
    ``block_table`` (R, max_blocks), whose rows must not overlap, and ``lengths`` (R,) are int32.  ``o`` (contiguous) has the cache's type.  ``lse``, if
    given, is (R, heads) float32 and receives the logarithm of each softmax's sum.  A request of length 0 gets zeros (lse
    -inf); one with a length outside its table row or a page outside the cache gets NaN.  No gradient goes through it.
    Softmax weights, and ``q`` where it is float32, are taken as two parts of the cache's type each: 22 bits with float16, 16
    with bfloat16, for queries of any size (beside spork_attn_sm100_paged in include/spork_b200.h).

    ``workspace`` is a contiguous CUDA tensor of attn_paged_workspace bytes, zero when it is first used and left so by every
    call (unless status() raises: zero it again then); launches that may run at the same time (other streams, other captured
    graphs) need one each.  Without one, a stream's launches share one that is kept for the stream until the process ends (up
    to about 10 MB), and a captured launch gets its own.  Launches on streams that torch did not make
    (torch.cuda.ExternalStream) take turns with four workspaces a device, each waiting for the one before it."""
    torch = _T or _bind_torch()
    q_shape, shape, table = q.shape, k_cache.shape, block_table.shape
    if not (len(q_shape) == 3 and len(shape) == 4 and len(table) == 2):
        _refuse_attn_paged(q, k_cache, v_cache, block_table, lengths, o, lse)
    n, heads, dim = q_shape
    pages, kv_heads, page, cache_dim = shape
    rows, blocks = table
    dtype, q_dtype = k_cache.dtype, q.dtype
    if o is None:
        o = _new(q, (n, heads, dim), dtype, stream)
    qs, ks, vs, ts = q.stride(), k_cache.stride(), v_cache.stride(), block_table.stride()
    device = q.get_device()
    # (looked at together, and one by one only to say what is wrong)
    if not (v_cache.shape == shape and cache_dim == dim and rows == n and lengths.shape == (n,) and o.shape == q_shape
            and v_cache.dtype is dtype and (q_dtype is dtype or q_dtype is torch.float32) and o.dtype is dtype
            and lengths.dtype is torch.int32 and block_table.dtype is torch.int32 and dtype in _CACHE_TYPES
            and qs[2] == 1 and ks[3] == 1 and vs[3] == 1 and (ts[1] == 1 or blocks <= 1) and lengths.is_contiguous()
            and o.is_contiguous() and device == k_cache.get_device() == v_cache.get_device() == block_table.get_device()
            == lengths.get_device() == o.get_device() >= 0):
        _refuse_attn_paged(q, k_cache, v_cache, block_table, lengths, o, lse)
    lse_ptr = 0
    if lse is not None:
        if not (lse.shape == (n, heads) and lse.dtype is torch.float32 and lse.is_contiguous() and lse.get_device() == device):
            _refuse_attn_paged(q, k_cache, v_cache, block_table, lengths, o, lse)
        lse_ptr = lse.data_ptr()
    launch_stream = _stream_of(stream, device)
    if workspace is None:
        workspace = _own_workspace(q, device, stream, (device, heads, kv_heads, dim))
        if workspace is None:
            with _lent_workspace(q, device, stream) as workspace:
                return attn_paged(q, k_cache, v_cache, block_table, lengths, o, lse=lse, scale=scale, workspace=workspace,
                                  stream=stream)
    else:
        if not workspace.is_contiguous():
            raise ValueError("workspace must be contiguous")
        if workspace.get_device() != device:
            _on_gpu(q=q, workspace=workspace)
    packed = _PAGED_ATTN_ARGS.pack(
        k_cache.data_ptr(), v_cache.data_ptr(), ks[0], ks[1], ks[2], vs[0], vs[1], vs[2], _TYPE_CODES[dtype], pages, kv_heads,
        page, dim, 0, q.data_ptr(), block_table.data_ptr(), lengths.data_ptr(), o.data_ptr(), lse_ptr, workspace.data_ptr(),
        workspace.nbytes, qs[0], qs[1], ts[0], n, heads, blocks, _TYPE_CODES[q_dtype],
        1.0 / dim ** 0.5 if scale is None else scale, 0)
    _call((_lib or lib()).spork_attn_sm100_paged, packed, device, launch_stream, "spork_attn_sm100_paged")
    return o
