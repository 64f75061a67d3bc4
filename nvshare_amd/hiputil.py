"""ctypes wrapper for the gfx950 kernels (hip/hiputil.hip, hip/kvcache.hip).

GPU-only: importing is safe anywhere, calling load() requires a box
with an MI355X and the built libnvshare_hiputil.so.
"""

from __future__ import annotations

import ctypes
import struct
from dataclasses import dataclass

from nvshare_amd.paths import artifacts


class _Args(struct.Struct):
    """A C structure's members, "type: name name; type: name", which
    pack() lays out as C does.  Packed bytes cost a tenth of what filling
    a ctypes.Structure does, and these calls are made for each token."""

    CODES = {"ptr": "P", "i64": "q", "int": "i", "f32": "f"}

    def __new__(cls, spec: str) -> "_Args":
        return super().__new__(cls, "@" + cls._codes(spec) + "0P")

    def __init__(self, spec: str) -> None:
        super().__init__("@" + self._codes(spec) + "0P")
        self.names = [n for part in spec.split(";")
                      for n in part.split(":")[1].split()]

    @classmethod
    def _codes(cls, spec: str) -> str:
        return "".join(cls.CODES[kind.strip()] * len(names.split())
                       for kind, names in (part.split(":")
                                           for part in spec.split(";")))


# The structures of hip/kvcache.h.
KV_CACHE = _Args(
    "ptr: k_cache v_cache k_scale v_scale table lens starts;"
    "i64: table_row k_page k_slot k_head v_page v_slot v_head;"
    "int: type cache_type batch total heads kv_heads dim pages page_size"
    " per_seq")
KV_APPEND = _Args(
    "ptr: q k v q_out rotation;"
    "i64: q_row q_head k_row k_head v_row v_head q_out_row q_out_head"
    " rotation_row;"
    "int: rotary interleaved fill")
KV_ATTEND = _Args(
    "ptr: q out lse; i64: q_row q_head out_row out_head;"
    "f32: scale; int: window max_new fill")

KV_BF16, KV_FP16, KV_E4M3 = 0, 1, 2


@dataclass
class HipUtil:
    lib: ctypes.CDLL

    def _ck(self, rc: int, what: str) -> None:
        if rc != 0:
            raise RuntimeError(f"{what} failed with hipError_t={rc}")

    def malloc_managed(self, nbytes: int) -> int:
        p = ctypes.c_void_p()
        self._ck(self.lib.nvs_hip_malloc_managed(ctypes.byref(p),
                                                 ctypes.c_size_t(nbytes)),
                 "hipMallocManaged")
        assert p.value is not None
        return p.value

    def malloc(self, nbytes: int) -> int:
        p = ctypes.c_void_p()
        self._ck(self.lib.nvs_hip_malloc(ctypes.byref(p),
                                         ctypes.c_size_t(nbytes)),
                 "hipMalloc")
        assert p.value is not None
        return p.value

    def free(self, ptr: int) -> None:
        self._ck(self.lib.nvs_hip_free(ctypes.c_void_p(ptr)), "hipFree")

    def prefetch(self, ptr: int, nbytes: int, device: int = 0) -> None:
        self._ck(self.lib.nvs_hip_prefetch(ctypes.c_void_p(ptr),
                                           ctypes.c_size_t(nbytes),
                                           device), "hipMemPrefetchAsync")

    ADVISE_PREFERRED_LOCATION = 3
    ADVISE_ACCESSED_BY = 5
    ADVISE_COARSE_GRAIN = 100

    def prefetch_chunked(self, ptr: int, nbytes: int, device: int = 0,
                         n_streams: int = 4,
                         chunk_bytes: int = 256 << 20) -> None:
        self._ck(self.lib.nvs_hip_prefetch_chunked(
            ctypes.c_void_p(ptr), ctypes.c_size_t(nbytes), device,
            n_streams, ctypes.c_size_t(chunk_bytes)),
            "prefetch_chunked")

    def advise(self, ptr: int, nbytes: int, advice: int,
               device: int = 0) -> None:
        self._ck(self.lib.nvs_hip_advise(ctypes.c_void_p(ptr),
                                         ctypes.c_size_t(nbytes),
                                         advice, device), "hipMemAdvise")

    def touch_pages(self, ptr: int, n_floats: int, stride: int = 1,
                    val: float = 1.0) -> None:
        self._ck(self.lib.nvs_touch_pages(ctypes.c_void_p(ptr),
                                          ctypes.c_size_t(n_floats),
                                          ctypes.c_size_t(stride),
                                          ctypes.c_float(val), None),
                 "touch_pages")

    def busy(self, ms: float) -> None:
        self._ck(self.lib.nvs_busy(ctypes.c_double(ms), None), "busy")

    def stream_triad(self, a: int, b: int, c: int, s: float,
                     n_floats: int) -> None:
        self._ck(self.lib.nvs_stream_triad(
            ctypes.c_void_p(a), ctypes.c_void_p(b), ctypes.c_void_p(c),
            ctypes.c_float(s), ctypes.c_size_t(n_floats), None),
            "stream_triad")

    def kv_append(self, cache: bytes, args: bytes, stream: int) -> None:
        """KV_CACHE and KV_APPEND, packed."""
        rc = self.lib.nvs_kv_append(cache, args, stream)
        if rc:
            self._ck(rc, "kv_append")

    def kv_attend_work(self, cache: bytes, args: bytes) -> int:
        """Bytes of the workspace that kv_attend needs."""
        n = self.lib.nvs_kv_attend_work(cache, args)
        if n < 0:
            self._ck(1, "kv_attend_work")
        return n

    def kv_attend(self, cache: bytes, args: bytes, work: int,
                  stream: int) -> None:
        """KV_CACHE and KV_ATTEND, packed."""
        rc = self.lib.nvs_kv_attend(cache, args, work, stream)
        if rc:
            self._ck(rc, "kv_attend")

    def sync(self) -> None:
        self._ck(self.lib.nvs_hip_sync(), "hipDeviceSynchronize")

    def mem_get_info(self) -> tuple[int, int]:
        f = ctypes.c_size_t()
        t = ctypes.c_size_t()
        self._ck(self.lib.nvs_hip_mem_get_info(ctypes.byref(f),
                                               ctypes.byref(t)),
                 "hipMemGetInfo")
        return f.value, t.value


def load() -> HipUtil:
    path = artifacts().hiputil
    if not path.exists():
        raise FileNotFoundError(
            f"{path} missing; build with `make -C hip` (hipcc, gfx950)")
    lib = ctypes.CDLL(str(path))
    for fname in ("nvs_hip_malloc_managed", "nvs_hip_malloc",
                  "nvs_hip_free", "nvs_hip_prefetch", "nvs_hip_advise",
                  "nvs_hip_prefetch_chunked",
                  "nvs_touch_pages", "nvs_read_pages", "nvs_busy",
                  "nvs_stream_triad", "nvs_hip_sync",
                  "nvs_hip_mem_get_info", "nvs_kv_append",
                  "nvs_kv_attend"):
        getattr(lib, fname).restype = ctypes.c_int
    text, ptr = ctypes.c_char_p, ctypes.c_void_p
    lib.nvs_kv_attend_work.restype = ctypes.c_int64
    lib.nvs_kv_attend_work.argtypes = [text, text]
    lib.nvs_kv_attend.argtypes = [text, text, ptr, ptr]
    lib.nvs_kv_append.argtypes = [text, text, ptr]
    return HipUtil(lib)
