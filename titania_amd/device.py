"""The hip device, as the reference's `Device` trait (model/device.rs:9-89)
presents it: weights are uploaded once, activations live in buffers allocated
on the device, and every operation runs there.

Method names, argument order and meaning follow the trait. Misuse that the
reference answers with a panic (its length asserts) raises InvalidArgument.
"""

from __future__ import annotations

import ctypes as C
from dataclasses import dataclass

import numpy as np

from . import _lib
from ._lib import HipError, InvalidArgument, check, lib


@dataclass
class Tensor:
    """A bf16 tensor as raw bits, row-major (model/weights.rs:13-17)."""

    shape: tuple
    data: np.ndarray  # uint16

    def __post_init__(self):
        self.shape = tuple(int(s) for s in self.shape)
        self.data = np.ascontiguousarray(self.data, dtype=np.uint16).reshape(-1)
        if self.data.size != int(np.prod(self.shape)):
            raise ValueError(f"{self.data.size} values for shape {self.shape}")


class Weight:
    """`Device::Weight` (model/device.rs:14-15): a bf16 tensor in device memory."""

    def __init__(self, dev: "Hip", handle: int, shape: tuple):
        self._dev = dev
        self.handle = handle
        self.shape = shape

    def free(self) -> None:
        if self.handle:
            self._dev._refuse_while_capturing("free a weight")
            lib().th_weight_free(self._dev.handle, self.handle)
            self.handle = None

    def __del__(self):
        try:
            if self._dev.handle:
                self.free()
        except Exception:
            pass


class Graph:
    """A captured sequence of device calls (th_graph_end): each launch() queues
    one replay on the device's stream over the buffers named at capture time."""

    def __init__(self, dev: "Hip", handle: int):
        self._dev = dev
        self.handle = handle

    def launch(self) -> None:
        check(lib().th_graph_launch(self._dev.handle, self.handle))

    def free(self) -> None:
        if self.handle:
            self._dev._refuse_while_capturing("free a graph")
            lib().th_graph_free(self._dev.handle, self.handle)
            self.handle = None

    def __del__(self):
        try:
            if self._dev.handle and not self._dev._capturing:
                self.free()
        except Exception:
            pass


class Buffer:
    """`Device::Buffer` (model/device.rs:10-13): f32 activations in device memory."""

    def __init__(self, dev: "Hip", handle: int):
        self._dev = dev
        self.handle = handle

    def __len__(self) -> int:
        return int(lib().th_buffer_len(self.handle))

    def free(self) -> None:
        if self.handle:
            self._dev._refuse_while_capturing("free a buffer")
            lib().th_buffer_free(self._dev.handle, self.handle)
            self.handle = None

    def __del__(self):
        try:
            if self._dev.handle:
                self.free()
        except Exception:
            pass


class Q8:
    """A matrix of 8-bit rows in device memory (th_q8), weights or activations:
    integers and an f32 scale for each row, whose product is the value."""

    def __init__(self, dev: "Hip", handle: int):
        self._dev = dev
        self.handle = handle

    @property
    def shape(self) -> tuple:
        rows, cols = C.c_size_t(), C.c_size_t()
        check(lib().th_q8_shape(self.handle, C.byref(rows), C.byref(cols)))
        return int(rows.value), int(cols.value)

    def free(self) -> None:
        if self.handle:
            self._dev._refuse_while_capturing("free 8-bit rows")
            lib().th_q8_free(self._dev.handle, self.handle)
            self.handle = None

    def __del__(self):
        try:
            if self._dev.handle:
                self.free()
        except Exception:
            pass


class Paged:
    """One layer's keys and values in pages in device memory (th_paged)."""

    def __init__(self, dev: "Hip", handle: int):
        self._dev = dev
        self.handle = handle

    @property
    def shape(self) -> tuple:
        """(pages, page_len, n_kv_heads, head_dim, kv_dtype)"""
        n, kv = [C.c_size_t() for _ in range(4)], C.c_int()
        check(lib().th_paged_shape(self.handle, *map(C.byref, n), C.byref(kv)))
        return (*(int(x.value) for x in n), int(kv.value))

    def free(self) -> None:
        if self.handle:
            self._dev._refuse_while_capturing("free a paged cache")
            lib().th_paged_free(self._dev.handle, self.handle)
            self.handle = None

    def __del__(self):
        try:
            if self._dev.handle:
                self.free()
        except Exception:
            pass


class Batch:
    """A step's sequences and their new tokens (th_batch): n_seqs and n_tokens of what is set."""

    def __init__(self, dev: "Hip", handle: int):
        self._dev = dev
        self.handle = handle
        self.n_seqs = self.n_tokens = 0

    def free(self) -> None:
        if self.handle:
            self._dev._refuse_while_capturing("free a batch")
            lib().th_batch_free(self._dev.handle, self.handle)
            self.handle = None

    def __del__(self):
        try:
            if self._dev.handle:
                self.free()
        except Exception:
            pass


def _ints(a, dtype) -> np.ndarray:
    """Whole numbers as `dtype`, those that it does not hold refused."""
    if type(a) is np.ndarray and a.dtype == dtype and a.ndim == 1 and a.flags.c_contiguous:
        return a
    a = np.asarray(a)
    if a.size and not np.issubdtype(a.dtype, np.integer):
        raise TypeError(f"whole numbers, not {a.dtype}")
    info = np.iinfo(dtype)
    if a.size and (int(a.min()) < info.min or int(a.max()) > info.max):
        raise ValueError(f"numbers past {np.dtype(dtype).name}")
    return np.ascontiguousarray(a, dtype=dtype).reshape(-1)


def _f32(a) -> np.ndarray:
    return np.ascontiguousarray(a, dtype=np.float32).reshape(-1)


class Hip:
    """A GPU running the model's operations (the `hip` device)."""

    def __init__(self, ordinal: int = 0):
        self._capturing = False
        h = C.c_void_p()
        check(lib().th_device_create(ordinal, C.byref(h)))
        self.handle = h.value

    def close(self) -> None:
        if self.handle:
            lib().th_device_destroy(self.handle)
            self.handle = None

    def synchronize(self) -> None:
        check(lib().th_device_synchronize(self.handle))

    # ---- HIP graphs of the device's stream (th_graph_*) ----

    def graph_begin(self) -> None:
        """Starts capturing: the compute calls that follow are recorded, not run,
        until graph_end (calls that allocate, copy to or from the host or wait
        raise meanwhile)."""
        check(lib().th_graph_begin(self.handle))
        self._capturing = True

    def graph_end(self) -> Graph:
        self._capturing = False
        out = C.c_void_p()
        check(lib().th_graph_end(self.handle, C.byref(out)))
        return Graph(self, out.value)

    def _refuse_while_capturing(self, what: str) -> None:
        if self._capturing:
            raise RuntimeError(f"cannot {what} while the device's stream is being captured (graph_begin)")

    def timer_begin(self) -> None:
        check(lib().th_timer_begin(self.handle))

    def timer_end(self) -> float:
        """Milliseconds of GPU time since timer_begin (waits for the queued work)."""
        ms = C.c_float()
        check(lib().th_timer_end(self.handle, C.byref(ms)))
        return float(ms.value)

    # ---- memory (model/device.rs:17-42) ----

    def upload(self, tensor: Tensor) -> Weight:
        shape = (C.c_size_t * len(tensor.shape))(*tensor.shape)
        out = C.c_void_p()
        check(lib().th_upload(self.handle, tensor.data.ctypes.data, shape, len(tensor.shape), C.byref(out)))
        return Weight(self, out.value, tensor.shape)

    def alloc(self, length: int) -> Buffer:
        out = C.c_void_p()
        check(lib().th_alloc(self.handle, int(length), C.byref(out)))
        return Buffer(self, out.value)

    def resize(self, buf: Buffer, length: int) -> None:
        check(lib().th_resize(self.handle, buf.handle, int(length)))

    def read(self, buf: Buffer) -> np.ndarray:
        n = len(buf)
        out = np.empty(n, dtype=np.float32)
        check(lib().th_read(self.handle, buf.handle, out.ctypes.data, n))
        return out

    def write(self, buf: Buffer, data) -> None:
        d = _f32(data)
        check(lib().th_write(self.handle, buf.handle, d.ctypes.data, d.size))

    def copy(self, dst: Buffer, dst_offset: int, src: Buffer, src_offset: int, length: int) -> None:
        check(lib().th_copy(self.handle, dst.handle, int(dst_offset), src.handle, int(src_offset), int(length)))

    # ---- compute (model/device.rs:44-88) ----

    def embed(self, out: Buffer, table: Weight, tokens) -> None:
        t = np.ascontiguousarray(tokens, dtype=np.uint32).reshape(-1)
        check(lib().th_embed(self.handle, out.handle, table.handle, t.ctypes.data, t.size))

    def matmul(self, out: Buffer, w: Weight, x: Buffer) -> None:
        check(lib().th_matmul(self.handle, out.handle, w.handle, x.handle))

    def add(self, x: Buffer, y: Buffer) -> None:
        check(lib().th_add(self.handle, x.handle, y.handle))

    def rmsnorm(self, x: Buffer, weight: Weight, eps: float) -> None:
        check(lib().th_rmsnorm(self.handle, x.handle, weight.handle, float(eps)))

    def rope(self, x: Buffer, table: Buffer, pos: int, n_heads: int, head_dim: int) -> None:
        check(lib().th_rope(self.handle, x.handle, table.handle, int(pos), int(n_heads), int(head_dim)))

    def attention(self, out: Buffer, q: Buffer, k_cache: Buffer, v_cache: Buffer, pos: int, n_heads: int,
                  head_dim: int, n_kv_heads: int) -> None:
        check(lib().th_attention(self.handle, out.handle, q.handle, k_cache.handle, v_cache.handle, int(pos),
                                 int(n_heads), int(head_dim), int(n_kv_heads)))

    def attention_noalloc(self, out: Buffer, q: Buffer, k_cache: Buffer, v_cache: Buffer, pos: int, n_heads: int,
                          head_dim: int, n_kv_heads: int) -> None:
        """attention() with its split partials in the library's fixed per-GPU
        array (no allocation); calls whose partials exceed it raise."""
        check(lib().th_attention_noalloc(self.handle, out.handle, q.handle, k_cache.handle, v_cache.handle,
                                         int(pos), int(n_heads), int(head_dim), int(n_kv_heads)))

    def silu_mul(self, gate: Buffer, up: Buffer) -> None:
        check(lib().th_silu_mul(self.handle, gate.handle, up.handle))

    # ---- fused extensions ----

    def add_rmsnorm(self, x: Buffer, y: Buffer | None, xb: Buffer, weight: Weight, eps: float) -> None:
        check(lib().th_add_rmsnorm(self.handle, x.handle, y.handle if y is not None else None, xb.handle,
                                   weight.handle, float(eps)))

    def qkv_rope_append(self, q: Buffer, k: Buffer, v: Buffer, wq: Weight, wk: Weight, wv: Weight,
                        q_norm: Weight | None, k_norm: Weight | None, xb: Buffer, rope: Buffer, k_cache: Buffer,
                        v_cache: Buffer, pos: int, n_heads: int, n_kv_heads: int, head_dim: int, eps: float) -> None:
        """model.rs:108-120 in one call: the q/k/v projections of xb, the
        per-head norms, the rotations and the appends to position-major
        caches (k and v are left holding the raw projections)."""
        check(lib().th_qkv_rope_append(self.handle, q.handle, k.handle, v.handle, wq.handle, wk.handle, wv.handle,
                                       q_norm.handle if q_norm is not None else None,
                                       k_norm.handle if k_norm is not None else None, xb.handle, rope.handle,
                                       k_cache.handle, v_cache.handle, int(pos), int(n_heads), int(n_kv_heads),
                                       int(head_dim), float(eps)))

    def gate_up_silu(self, gate: Buffer, up: Buffer, w_gate: Weight, w_up: Weight, xb: Buffer) -> None:
        """gate = silu(w_gate . xb) * (w_up . xb) (model.rs:137-139); up is scratch."""
        check(lib().th_gate_up_silu(self.handle, gate.handle, up.handle, w_gate.handle, w_up.handle, xb.handle))

    # ---- 8-bit rows ----

    def alloc_q8(self, rows: int, cols: int) -> Q8:
        out = C.c_void_p()
        check(lib().th_q8_alloc(self.handle, int(rows), int(cols), C.byref(out)))
        return Q8(self, out.value)

    def resize_q8(self, q: Q8, rows: int) -> None:
        check(lib().th_q8_resize(self.handle, q.handle, int(rows)))

    def read_q8(self, q: Q8) -> tuple[np.ndarray, np.ndarray]:
        """The integers [rows, cols] and the scales [rows]."""
        rows, cols = q.shape
        values, scales = np.empty((rows, cols), dtype=np.int8), np.empty(rows, dtype=np.float32)
        check(lib().th_q8_read(self.handle, q.handle, values.ctypes.data, scales.ctypes.data))
        return values, scales

    def write_q8(self, q: Q8, values, scales) -> None:
        v, s = np.asarray(values), _f32(scales)
        if v.dtype != np.int8:
            raise TypeError(f"8-bit rows are int8, not {v.dtype}")
        if v.size != q.shape[0] * q.shape[1] or s.size != q.shape[0]:
            raise ValueError(f"{v.size} integers and {s.size} scales for 8-bit rows of shape {q.shape}")
        v = np.ascontiguousarray(v)
        check(lib().th_q8_write(self.handle, q.handle, v.ctypes.data, s.ctypes.data))

    def quantize_q8(self, q: Q8, x: Buffer) -> None:
        """q = the rows of x."""
        check(lib().th_quantize_q8(self.handle, q.handle, x.handle))

    def quantize_weight_q8(self, q: Q8, w: Weight) -> None:
        """q = the rows of w, each output channel with its scale."""
        check(lib().th_quantize_weight_q8(self.handle, q.handle, w.handle))

    def dequantize_q8(self, out: Buffer, q: Q8) -> None:
        """out = the values that q stands for."""
        check(lib().th_dequantize_q8(self.handle, out.handle, q.handle))

    def add_rmsnorm_q8(self, x: Buffer, y: Buffer | None, q: Q8, weight: Weight, eps: float) -> None:
        """x += y (unless y is None), then q = the rows of rmsnorm(x)."""
        check(lib().th_add_rmsnorm_q8(self.handle, x.handle, y.handle if y is not None else None, q.handle,
                                      weight.handle, float(eps)))

    def silu_mul_q8(self, q: Q8, gate: Buffer, up: Buffer) -> None:
        """q = the rows of silu(gate) * up."""
        check(lib().th_silu_mul_q8(self.handle, q.handle, gate.handle, up.handle))

    def matmul_q8(self, out: Buffer, w: Q8, x: Q8) -> None:
        """matmul() over 8-bit rows: sums of integer products, times both scales."""
        check(lib().th_matmul_q8(self.handle, out.handle, w.handle, x.handle))

    # ---- paged caches ----

    def alloc_paged(self, pages: int, page_len: int, n_kv_heads: int, head_dim: int,
                    kv_dtype: int = _lib.TH_KV_F32) -> Paged:
        """A layer's cache of zeroed pages of page_len positions."""
        out = C.c_void_p()
        check(lib().th_paged_alloc(self.handle, int(pages), int(page_len), int(n_kv_heads), int(head_dim), int(kv_dtype),
                                   C.byref(out)))
        return Paged(self, out.value)

    def read_paged(self, cache: Paged, page: int) -> tuple[np.ndarray, np.ndarray]:
        """A page's keys and values [page_len, n_kv_heads, head_dim]."""
        k, v = (np.empty(cache.shape[1:4], dtype=np.float32) for _ in range(2))
        check(lib().th_paged_read(self.handle, cache.handle, int(page), k.ctypes.data, v.ctypes.data))
        return k, v

    def write_paged(self, cache: Paged, page: int, k, v) -> None:
        k, v = _f32(k), _f32(v)
        if not k.size == v.size == int(np.prod(cache.shape[1:4])):
            raise ValueError(f"{k.size} keys and {v.size} values for a page of shape {cache.shape[1:4]}")
        check(lib().th_paged_write(self.handle, cache.handle, int(page), k.ctypes.data, v.ctypes.data))

    def alloc_batch(self, cache: Paged, n_heads: int, max_seqs: int, max_tokens: int, max_pages: int) -> Batch:
        """Room for a step's sequences, new tokens and pages, over caches of this one's shape."""
        out = C.c_void_p()
        check(lib().th_batch_alloc(self.handle, cache.handle, int(n_heads), int(max_seqs), int(max_tokens),
                                   int(max_pages), C.byref(out)))
        return Batch(self, out.value)

    def set_batch(self, batch: Batch, context, new, pages, parents=None) -> None:
        """Once a step: sequence s has context[s] positions in the caches and
        new[s] tokens behind them, in its pages (those of all sequences one
        after another); parents: of each token the one of its sequence that it
        follows, -1 for the context (None: each follows the one before)."""
        c, n, p = _ints(context, np.uint32), _ints(new, np.uint32), _ints(pages, np.uint32)
        if c.size != n.size:
            raise ValueError(f"{c.size} contexts of {n.size} sequences")
        t = None if parents is None else _ints(parents, np.int32)
        tokens = int(n.sum(dtype=np.int64))
        if t is not None and t.size != tokens:
            raise ValueError(f"{t.size} parents of {tokens} tokens")
        try:
            check(lib().th_batch_set(self.handle, batch.handle, n.size, c.ctypes.data, n.ctypes.data, p.ctypes.data, p.size,
                                     None if t is None else t.ctypes.data))
        except HipError as e:
            if not isinstance(e, InvalidArgument):  # nothing is set
                batch.n_seqs = batch.n_tokens = 0
            raise
        batch.n_seqs, batch.n_tokens = n.size, tokens

    def paged_append(self, q_out: Buffer, q: Buffer, k: Buffer, v: Buffer, q_norm: Weight | None, k_norm: Weight | None,
                     rope: Buffer, cache: Paged, batch: Batch, eps: float) -> None:
        """q_out = q, normed and rotated; k, normed and rotated, and v to the batch's rows of the cache."""
        check(lib().th_paged_append(self.handle, q_out.handle, q.handle, k.handle, v.handle,
                                    q_norm.handle if q_norm is not None else None,
                                    k_norm.handle if k_norm is not None else None, rope.handle, cache.handle,
                                    batch.handle, float(eps)))

    def paged_attention(self, out: Buffer, q: Buffer, cache: Paged, batch: Batch) -> None:
        """attention() of the batch's tokens over what each of them sees."""
        check(lib().th_paged_attention(self.handle, out.handle, q.handle, cache.handle, batch.handle))

    def accept(self, batch: Batch, logits: Buffer, tokens) -> tuple[np.ndarray, np.ndarray, np.ndarray]:
        """The greedy verification of the batch's drafted tokens: each row's
        largest logit, how many tokens of each sequence are kept, and their
        places in it, from its first token's element on (-1 behind them)."""
        t = _ints(tokens, np.uint32)
        if t.size != batch.n_tokens:
            raise ValueError(f"{t.size} tokens of a batch of {batch.n_tokens}")
        picks, n_kept, kept = np.empty(t.size, np.uint32), np.empty(batch.n_seqs, np.uint32), np.empty(t.size, np.int32)
        check(lib().th_batch_accept(self.handle, batch.handle, logits.handle, t.ctypes.data, picks.ctypes.data,
                                    n_kept.ctypes.data, kept.ctypes.data))
        return picks, n_kept, kept

    def paged_keep(self, caches, batch: Batch, n_kept, kept) -> None:
        """The rows of the tokens kept (as accept() gives them), moved up behind the context in each cache."""
        n, k = _ints(n_kept, np.uint32), _ints(kept, np.int32)
        if n.size != batch.n_seqs or k.size != batch.n_tokens:
            raise ValueError(f"{n.size} counts and {k.size} places for {batch.n_seqs} sequences of {batch.n_tokens} tokens")
        handles = (C.c_void_p * len(caches))(*[c.handle for c in caches])
        check(lib().th_paged_keep(self.handle, handles, len(caches), batch.handle, n.ctypes.data, k.ctypes.data))

    # ---- the next token ----

    def argmax(self, logits: Buffer) -> int:
        tok = C.c_uint32()
        check(lib().th_argmax(self.handle, logits.handle, C.byref(tok)))
        return int(tok.value)

    def sample(self, logits: Buffer, sampler) -> int:
        """A draw of `sampler` (titania_amd.sampler.Sampler) from the buffer's
        values (th_sample); advances sampler.rng."""
        tok = C.c_uint32()
        st = C.c_uint64(sampler.rng)
        check(lib().th_sample(self.handle, logits.handle, sampler.temperature, max(sampler.top_k, 0),
                              sampler.top_p, C.byref(st), C.byref(tok)))
        sampler.rng = st.value
        return int(tok.value)


__all__ = ["Hip", "Tensor", "Weight", "Buffer", "Q8", "Paged", "Batch", "_lib"]
