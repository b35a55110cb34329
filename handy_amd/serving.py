"""Serving operators over a paged K/V cache, for callers that run a text decoder of their own next to the transcription: the
step's block tables and slots (`plan_pages`), the new tokens' K and V (`write_kv`), attention of the new tokens over the cache
(`paged_attention`) and the draw of the next token (`sample_tokens`), through the C ABI of libwhisper_mi355.so (include/wmi.h).
No counterpart in the reference, whose engine keeps one sequence at a time.

Arguments are device arrays: anything with `data_ptr()`, `shape`, `stride()` and `dtype` -- a torch tensor on the GPU, or a
`DeviceArray` in memory of the HIP runtime the library is linked against. (In a process that uses torch, import torch before the
library is loaded, so that both use one runtime.) Calls enqueue on `stream` (a hipStream_t value; 0 = the null stream) and return
without waiting; outputs are the caller's buffers, so calls can be captured into graphs. Wrong arguments raise ValueError before
anything is enqueued."""
import ctypes as C
import math
import operator
import struct
from typing import Optional

import numpy as np

from . import whisper_rs as wr

_DTYPES = {"float16": 0, "bfloat16": 1, "float32": 2}
_SIZES = {"float16": 2, "bfloat16": 2, "float32": 4, "int32": 4, "uint8": 1}
_NUMPY = {"float16": np.float16, "bfloat16": np.uint16, "float32": np.float32, "int32": np.int32, "uint8": np.uint8}


class DeviceArray:
    """Array in device memory on the current HIP device. bfloat16 travels to and from the host as uint16 bit patterns."""

    def __init__(self, shape, dtype: str, _base=None, _strides=None, _offset: int = 0):
        self.shape = tuple(int(s) for s in (shape if isinstance(shape, (tuple, list)) else (shape,)))
        self.dtype = dtype
        self._strides = tuple(_strides) if _strides is not None else _contiguous(self.shape)
        self._base, self._offset, self._ptr = _base, _offset, None
        if _base is None:
            self._bytes = math.prod(self.shape) * _SIZES[dtype]
            self._ptr = wr.load_library().wmi_dev_alloc(max(self._bytes, 16))
            if not self._ptr:
                raise wr.WhisperError(f"device allocation of {self._bytes} bytes failed")

    @classmethod
    def from_numpy(cls, a, dtype: Optional[str] = None):
        a = np.ascontiguousarray(a)
        d = cls(a.shape, dtype or a.dtype.name)
        if a.dtype != _NUMPY[d.dtype]:
            raise ValueError(f"{a.dtype} is not the host form of {d.dtype}")
        if a.size and wr.load_library().wmi_dev_upload(d.data_ptr(), a.ctypes.data, a.nbytes) != 0:
            raise wr.WhisperError("hipMemcpy to the device failed")
        return d

    def numpy(self) -> np.ndarray:
        """The whole array on the host (waits for the null stream's work); views copy their base and pick on the host."""
        if self._base is not None:
            flat = self._base.numpy().reshape(-1)[self._offset:]
            return np.lib.stride_tricks.as_strided(flat, self.shape, [s * flat.itemsize for s in self._strides]).copy()
        out = np.empty(self.shape, _NUMPY[self.dtype])
        if out.size and wr.load_library().wmi_dev_download(out.ctypes.data, self._ptr, out.nbytes) != 0:
            raise wr.WhisperError("hipMemcpy from the device failed")
        return out

    def view(self, shape, strides, offset: int = 0):
        """Another shape over the same memory; strides and offset in elements."""
        root = self._base or self
        last = self._offset + offset + sum((s - 1) * t for s, t in zip(shape, strides))
        if min(strides, default=0) < 0 or self._offset + offset < 0 or (0 not in shape and last >= math.prod(root.shape)):
            raise ValueError("view outside the array")
        return DeviceArray(shape, self.dtype, root, strides, self._offset + offset)

    def permute(self, *order):
        return self.view([self.shape[i] for i in order], [self._strides[i] for i in order])

    def data_ptr(self): return self._ptr if self._base is None else self._base.data_ptr() + self._offset * _SIZES[self.dtype]
    def stride(self): return self._strides
    def numel(self): return math.prod(self.shape)

    def free(self):
        if self._ptr:
            wr.load_library().wmi_dev_free(self._ptr)
            self._ptr = None

    def __del__(self):
        try:
            self.free()
        except Exception:
            pass


def _contiguous(shape):
    out, n = [], 1
    for s in reversed(shape):
        out.append(n)
        n *= s
    return tuple(reversed(out))


_ATTN = struct.Struct("@5P5q7if")         # wmi_paged_attn (packing bytes takes half the time of filling the ctypes structure)
assert _ATTN.size == C.sizeof(wr.wmi_paged_attn)
_NAMES = {}         # dtype object -> name ("float16" and torch.float16 alike)


def _dtype(x) -> str:
    d = x.dtype
    n = _NAMES.get(d)
    if n is None:
        n = _NAMES[d] = str(d).replace("torch.", "")
    return n


def _i32(v, name: str):
    """v where it fits the C ABI's int (ctypes would pass its low bits on)"""
    try:
        if -0x80000000 <= operator.index(v) <= 0x7fffffff:
            return v
    except TypeError:
        pass
    raise ValueError(f"{name}: {v} is no 32-bit whole number")


def _flat(x, dtype: str, n: int, name: str):
    """pointer of a contiguous 1-d array of at least n elements (none of no elements)"""
    s = x.shape
    if len(s) != 1 or s[0] < n or _dtype(x) != dtype or (n > 1 and x.stride()[0] != 1):
        raise ValueError(f"{name}: expected a contiguous {dtype} array of {n}")
    return x.data_ptr() if n else None


def _rows(x, shape, dtype: str, name: str):
    """pointer and the two outer strides of a [rows][heads][dim] array with contiguous heads"""
    st = x.stride()
    if x.shape != shape or _dtype(x) != dtype or (st[2] != 1 and shape[2] > 1):
        raise ValueError(f"{name}: expected {dtype} {tuple(shape)} with contiguous last axis")
    return x.data_ptr(), st[0], st[1]


def _table(x, n_seq: int):
    """pointer, row stride and columns of an int32 [n_seq][cols] array with contiguous rows"""
    s, st = x.shape, x.stride()
    if len(s) != 2 or s[0] != n_seq or _dtype(x) != "int32" or (st[1] != 1 and s[1] > 1):
        raise ValueError("block_table: expected int32 [n_seq, cols] with contiguous rows")
    cols = s[1]
    if n_seq > 1 and st[0] < cols:
        raise ValueError("block_table: its rows share memory (an expanded row, or overlapping ones)")
    return x.data_ptr() if n_seq and cols else None, max(st[0], cols), cols


def _lib():
    return wr._lib or wr.load_library()


def _check(rc: int, what: str):
    if rc in (-1, -2, -3):
        raise ValueError(what + {-1: ": bad arguments (sizes, alignment, outputs that share memory, or memory that is not the call's GPU's)", -2: ": workspace too small",
                                 -3: ": sizes not supported"}[rc])
    if rc != 0:
        raise wr.WhisperError(f"{what} failed", rc)


class PagedCache:
    """One layer's K and V in pages: two arrays of shape [n_pages, page_tokens, n_kv_heads, head_dim], any strides with a contiguous last
    axis and the same for both (a head-major cache is passed as its permuted view). Keeps the arrays."""

    def __init__(self, k, v):
        dt = _dtype(k)
        if dt not in ("float16", "bfloat16") or _dtype(v) != dt:
            raise ValueError("K and V: float16 or bfloat16, both the same")
        if len(k.shape) != 4 or tuple(k.shape) != tuple(v.shape) or tuple(k.stride()) != tuple(v.stride()) or (k.shape[3] > 1 and k.stride()[3] != 1):
            raise ValueError("K and V: [n_pages, page_tokens, n_kv_heads, head_dim] with the same strides and a contiguous last axis")
        self.k, self.v, self.dtype = k, v, dt
        self.n_pages, self.page_tokens, self.n_kv_heads, self.head_dim = (int(_i32(n, "K and V")) for n in k.shape)
        st = k.stride()
        self.c = wr.wmi_paged_cache(k.data_ptr(), v.data_ptr(), _DTYPES[dt], self.n_pages, self.page_tokens, self.n_kv_heads, self.head_dim, st[0], st[1], st[2])
        self.ref = C.byref(self.c)


class PagePlan:
    """Buffers of one step's plan, int32: cu_q[n_seq + 1], kv_lens[n_seq], slots[rows], positions[rows], counts[4]. Keeps the arrays."""
    __slots__ = ("cu_q", "kv_lens", "slots", "positions", "counts", "n_seq", "n_rows", "_p")

    def __init__(self, cu_q, kv_lens, slots, positions, counts):
        self.cu_q, self.kv_lens, self.slots, self.positions, self.counts = cu_q, kv_lens, slots, positions, counts
        self.n_seq, self.n_rows = int(_i32(kv_lens.shape[0], "kv_lens")), int(_i32(slots.shape[0], "slots"))
        self._p = (_flat(cu_q, "int32", self.n_seq + 1, "cu_q"), _flat(kv_lens, "int32", self.n_seq, "kv_lens"), _flat(slots, "int32", self.n_rows, "slots"),
                   _flat(positions, "int32", self.n_rows, "positions"), self.n_rows, _flat(counts, "int32", 4, "counts"))

    def __iter__(self):
        return iter((self.cu_q, self.kv_lens, self.slots, self.positions, self.counts))

    @classmethod
    def allocate(cls, n_seq: int, n_rows: int):
        return cls(*(DeviceArray(n, "int32") for n in (n_seq + 1, n_seq, n_rows, n_rows, 4)))


def plan_pages(ctx_lens, new_lens, free_pages, block_table, page_tokens: int, out: PagePlan, stream: int = 0) -> PagePlan:
    """Admit requests in order, give them fresh pages from the front of free_pages (entered in block_table[n_seq, cols]) and number
    their rows: see wmi_paged_plan in include/wmi.h. The number of rows planned for is the length of out.slots. The plan's arrays and
    block_table share no memory with each other or the inputs (copy out.kv_lens for the next step's ctx_lens)."""
    n_seq, n_free = out.n_seq, free_pages.shape[0]
    tp, stride, cols = _table(block_table, n_seq)
    if ctx_lens.shape[0] != n_seq or new_lens.shape[0] != n_seq:
        raise ValueError(f"ctx_lens, new_lens: expected the plan's {n_seq} requests")
    rc = _lib().wmi_paged_plan(_flat(ctx_lens, "int32", n_seq, "ctx_lens"), _flat(new_lens, "int32", n_seq, "new_lens"), n_seq,
                               _flat(free_pages, "int32", n_free, "free_pages"), _i32(n_free, "free_pages"), _i32(page_tokens, "page_tokens"), tp, cols, stride, *out._p, stream)
    if rc:
        _check(rc, "plan_pages")
    return out


def write_kv(cache: PagedCache, k_new, v_new, slots, stream: int = 0) -> None:
    """cache[slots[r]] = k_new[r], v_new[r] (rows [n_kv_heads, head_dim], any row and head strides); rows with a slot outside the cache
    are skipped. The slots of one call must be distinct."""
    n = _i32(k_new.shape[0], "k_new")
    shape = (n, cache.n_kv_heads, cache.head_dim)
    kp, kr, kh = _rows(k_new, shape, cache.dtype, "k_new")
    vp, vr, vh = _rows(v_new, shape, cache.dtype, "v_new")
    rc = _lib().wmi_paged_write(cache.ref, kp if n else None, kr, kh, vp if n else None, vr, vh, _flat(slots, "int32", n, "slots"), n, stream)
    if rc:
        _check(rc, "write_kv")


def paged_attention_workspace(cache: PagedCache, n_rows: int, n_q_heads: int, n_seq: int, max_new: int = 0, max_kv: int = 0) -> int:
    """Bytes of device memory `paged_attention` needs for these sizes (0: none)."""
    try:
        a = _ATTN.pack(0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, n_rows, n_seq, n_q_heads, 0, max_new, max_kv, 1.0)
    except struct.error as e:
        raise ValueError(f"paged_attention_workspace: {e}") from None
    need = _lib().wmi_paged_attention_workspace(cache.ref, a)
    if need < 0:
        _check(int(need), "paged_attention_workspace")
    return int(need)


def paged_attention(q, cache: PagedCache, block_table, cu_q, kv_lens, max_new: int, max_kv: int, out, scale: Optional[float] = None, window: int = 0,
                    workspace=None, stream: int = 0):
    """softmax(scale q K^T) V of the requests' new tokens (q and out: [n_rows, n_q_heads, head_dim]) over the cache, causal, with window
    > 0 over the last `window` keys only: see wmi_paged_attention in include/wmi.h. max_new / max_kv: the longest request's new and
    total tokens (0: not known; they steer the split of the work). workspace: uint8 device array of `paged_attention_workspace`
    bytes, one for each call that may run at the same time. Returns out."""
    shape, dim = q.shape, cache.head_dim
    if len(shape) != 3 or shape[2] != dim:
        raise ValueError("q: expected [n_rows, n_q_heads, head_dim]")
    qp, qr, qh = _rows(q, shape, cache.dtype, "q")
    op, orow, oh = _rows(out, shape, cache.dtype, "out")
    n_seq = kv_lens.shape[0]
    tp, stride, cols = _table(block_table, n_seq)
    try:
        a = _ATTN.pack(qp or 0, op or 0, tp or 0, _flat(cu_q, "int32", n_seq + 1, "cu_q") or 0, _flat(kv_lens, "int32", n_seq, "kv_lens") or 0, qr, qh, orow, oh, stride, cols,
                       shape[0], n_seq, shape[1], window, max_new, max_kv, dim ** -0.5 if scale is None else scale)
    except (struct.error, OverflowError) as e:
        raise ValueError(f"paged_attention: {e}") from None
    ws, ws_bytes = None, 0
    if workspace is not None:
        ws_bytes = workspace.shape[0]
        ws = _flat(workspace, "uint8", ws_bytes, "workspace")
    rc = _lib().wmi_paged_attention(cache.ref, a, ws, ws_bytes, stream)
    if rc:
        _check(rc, "paged_attention")
    return out


def sample_tokens(logits, uniform, token, logprob=None, temperature=None, top_k=None, top_p=None, min_p=None, stream: int = 0):
    """One token a row of logits [n_rows, n_vocab] (float32, float16 or bfloat16) into token (int32), from uniform numbers in [0, 1) (float32,
    one a row): see wmi_sample_tokens in include/wmi.h. temperature, top_p, min_p (float32) and top_k (int32) are per row or None.
    logprob (float32, may be None): the token's log-probability before the filters. Returns token."""
    dt, shape, st = _DTYPES.get(_dtype(logits), -1), logits.shape, logits.stride()
    if dt < 0 or len(shape) != 2 or (st[1] != 1 and shape[1] > 1):
        raise ValueError("logits: expected float32, float16 or bfloat16 [n_rows, n_vocab] with contiguous rows")
    n, v = _i32(shape[0], "logits"), _i32(shape[1], "logits")
    rc = _lib().wmi_sample_tokens(
        logits.data_ptr() if n else None, dt, st[0], n, v, _flat(uniform, "float32", n, "uniform"),
        None if temperature is None else _flat(temperature, "float32", n, "temperature"), None if top_k is None else _flat(top_k, "int32", n, "top_k"),
        None if top_p is None else _flat(top_p, "float32", n, "top_p"), None if min_p is None else _flat(min_p, "float32", n, "min_p"),
        _flat(token, "int32", n, "token"), None if logprob is None else _flat(logprob, "float32", n, "logprob"), stream)
    if rc:
        _check(rc, "sample_tokens")
    return token
