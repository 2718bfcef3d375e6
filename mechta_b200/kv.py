"""Host-side mirror of the reference's KV operators above the C ABI.

Names follow the reference (engine/crates/mechta/src/engine.rs, quad.rs): KvFormat, check_ctx, rope_table,
Root, read_root / write_root, need_bytes; step4-style helpers take `pos` exactly as the reference does (token t of
a call sits at pos + t). PyTorch is used only for device memory and streams; every computation is a call into
libmechta_kv through ctypes with raw pointers.
"""
from __future__ import annotations

import array
import ctypes as C
import enum
import itertools
from dataclasses import dataclass

import numpy as np
import torch

from . import _lib
from ._lib import MkvError, check

CTX_DEFAULT, CTX_MIN, CTX_MAX = 65536, 4096, 262144  # engine.rs:23-25
HQ, HKV, D, ROW = 16, 2, 256, 512
K_VERIFY = 4  # quad.rs K


class KvFormat(enum.IntEnum):
    """engine.rs:49-68"""
    F16 = _lib.F16
    F32 = _lib.F32

    @property
    def elem_bytes(self) -> int:
        return 2 if self is KvFormat.F16 else 4

    def data_words(self, n: int) -> int:
        return n if self is KvFormat.F32 else n // 2

    def buffer_bytes_for(self, ctx: int) -> int:
        return 4 * self.data_words(ctx * 512)

    @property
    def torch_dtype(self):
        return torch.float16 if self is KvFormat.F16 else torch.float32


def check_ctx(n: int) -> int:
    """engine.rs:28-33: a multiple of 1024 in [CTX_MIN, CTX_MAX]."""
    if n % 1024 != 0 or not (CTX_MIN <= n <= CTX_MAX):
        raise ValueError(f"context {n}: must be a multiple of 1024 between {CTX_MIN} and {CTX_MAX}")
    return n


def rope_table(pos: int, ntok: int = 1) -> np.ndarray:
    """engine.rs:108-114 for positions pos..pos+ntok-1: [ntok][64] = [cos 0..31 | sin 0..31]."""
    out = np.empty((ntok, 64), np.float32)
    _lib.lib().mkv_rope_table(int(pos), int(ntok), out.ctypes.data_as(C.c_void_p))
    return out


def need_bytes(ctx: int, fmt: KvFormat, n_layers: int = 11) -> int:
    """memcheck.rs:14-20 without BASE_BYTES (10 attention layers + the MTP layer by default)."""
    return int(_lib.lib().mkv_need_bytes(ctx, int(fmt), n_layers))


def root_key(tokens) -> str:
    """session.rs:61-66"""
    t = np.ascontiguousarray(tokens, np.uint32)
    return f"{int(_lib.lib().mkv_root_key(t.ctypes.data_as(C.c_void_p), t.size)):016x}"


@dataclass
class Root:
    """engine.rs:194-195 Root, KV part: rows [0, p) of every attention layer, K then V, raw cache bytes."""
    p: int
    fmt: KvFormat
    n_layers: int
    payload: torch.Tensor  # uint8, pinned host memory


def _ptr(t) -> int:
    if t is None:
        return 0
    assert t.is_contiguous(), "tensors passed to the KV operators must be contiguous"
    return t.data_ptr()


class KvContext:
    """One device + the stream the KV operators run on (mkv_ctx)."""

    def __init__(self, device: int = 0, stream: torch.cuda.Stream | None = None):
        self._h = C.c_void_p()
        self.device = int(device)
        self.stream = stream
        sp = C.c_void_p(stream.cuda_stream) if stream is not None else None
        check(_lib.lib().mkv_ctx_create(self.device, sp, C.byref(self._h)))

    def sync(self) -> None:
        check(_lib.lib().mkv_sync(self._h))

    @property
    def launches(self) -> int:
        return int(_lib.lib().mkv_launch_count(self._h))

    def prof_enable(self, on: int) -> None:
        """0 = off; n > 0 = on, with n event pairs created ahead of time."""
        check(_lib.lib().mkv_prof_enable(self._h, int(on)))

    def prof_read(self) -> tuple[float, int]:
        ms, n = C.c_double(), C.c_uint64()
        check(_lib.lib().mkv_prof_read(self._h, C.byref(ms), C.byref(n)))
        return ms.value, int(n.value)

    def combine_shards(self, recs: torch.Tensor, ntok: int, out: torch.Tensor) -> None:
        """recs [n_shards][64][258] f32 -> out [ntok][16][256] (ops.wgsl:529-537 over shards)."""
        check(_lib.lib().mkv_combine_shards(self._h, _ptr(recs), recs.shape[0], ntok, _ptr(out)))

    def attn_verify_batch(self, items) -> None:
        """items: iterable of (cache, layer, first_pos, pos, q, out); one launch pair for all of them."""
        items = list(items)
        arr = (_lib.VerifyItem * len(items))()
        for i, (cache, layer, first_pos, pos, q, out) in enumerate(items):
            arr[i] = _lib.VerifyItem(cache._h.value, layer, first_pos, pos, q.shape[0], _ptr(q), _ptr(out))
        check(_lib.lib().mkv_attn_verify_batch(self._h, arr, len(items)))

    def close(self) -> None:
        if self._h:
            _lib.lib().mkv_ctx_destroy(self._h)
            self._h = C.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class KvCache:
    """The per-layer K and V buffers of the attention layers and the operators that touch them (mkv_cache)."""

    def __init__(self, ctx: KvContext, fmt: KvFormat, n_layers: int, context: int, shard_first: int = 0,
                 shard_tokens: int = 0, ring: int = 0):
        """context: the sequence's context (check_ctx rule). shard_tokens = 0: the whole context lives here;
        otherwise only rows [shard_first, shard_first + shard_tokens). ring > 0: a ring cache of that many rows,
        position p in row p % ring (flint.rs:24-26)."""
        self.ctx, self.fmt, self.n_layers = ctx, KvFormat(fmt), n_layers
        self.context, self.ring = context, ring
        self.capacity, self.shard_first = (ring or shard_tokens or context), shard_first
        self._h = C.c_void_p()
        if ring:
            check(_lib.lib().mkv_cache_create_ring(ctx._h, int(fmt), n_layers, context, ring, C.byref(self._h)))
        else:
            check(_lib.lib().mkv_cache_create(ctx._h, int(fmt), n_layers, context, shard_first, shard_tokens,
                                              C.byref(self._h)))

    # -- bookkeeping
    def __len__(self) -> int:
        return int(_lib.lib().mkv_cache_len(self._h))

    def set_len(self, n: int) -> None:
        check(_lib.lib().mkv_cache_set_len(self._h, n))

    @property
    def device_bytes(self) -> int:
        return int(_lib.lib().mkv_cache_device_bytes(self._h))

    def buffers(self, layer: int) -> tuple[int, int]:
        k, v = C.c_void_p(), C.c_void_p()
        check(_lib.lib().mkv_cache_buffers(self._h, layer, C.byref(k), C.byref(v)))
        return k.value, v.value

    def buffer_tensors(self, layer: int) -> tuple[torch.Tensor, torch.Tensor]:
        """Zero-copy torch views [capacity][2][256] of a layer's K and V (for tests and synthetic fills)."""
        kp, vp = self.buffers(layer)
        return tuple(_as_tensor(p, self.capacity * ROW, self.fmt.torch_dtype, self.ctx.device).view(self.capacity, HKV, D)
                     for p in (kp, vp))

    # -- operators
    def append(self, layer: int, pos: int, k: torch.Tensor, v: torch.Tensor, tab: torch.Tensor | None) -> None:
        """kv_rope2 + kv_copy (kv.wgsl:19-42): k, v f32 [ntok][2][256]; tab f32 [ntok][64] or None."""
        check(_lib.lib().mkv_append(self._h, layer, pos, k.shape[0], _ptr(k), _ptr(v), _ptr(tab)))

    def append_layers(self, pos: int, k: torch.Tensor, v: torch.Tensor, tab: torch.Tensor | None) -> None:
        """All layers in one launch: k, v f32 [n_layers][ntok][2][256]."""
        check(_lib.lib().mkv_append_layers(self._h, pos, k.shape[1], _ptr(k), _ptr(v), _ptr(tab)))

    def truncate(self, new_len: int, scrub: bool = False) -> None:
        """Rollback of refused drafts: the next step continues at new_len (session.rs:385-411)."""
        check(_lib.lib().mkv_truncate(self._h, new_len, int(scrub)))

    def attn_verify(self, layer: int, first_pos: int, pos: int, q: torch.Tensor, out: torch.Tensor) -> None:
        """q_dmx + attn_dmx2 + attn_fd_combine (dmx.rs) / attn_fd (+combine): q, out f32 [ntok][16][256]."""
        check(_lib.lib().mkv_attn_verify(self._h, layer, first_pos, pos, q.shape[0], _ptr(q), _ptr(out)))

    def attn_verify_window(self, layer: int, window: int, sinks: torch.Tensor | None, pos: int, q: torch.Tensor,
                           out: torch.Tensor) -> None:
        """Verify attention with a sliding window (0 = none) and per-head sinks [16] (None = none), on a ring or an
        ordinary cache (flint.rs:22-26, flint_attn.wgsl:79-82,243-255)."""
        check(_lib.lib().mkv_attn_verify_window(self._h, layer, window, _ptr(sinks), pos, q.shape[0], _ptr(q), _ptr(out)))

    def attn_step(self, layer: int, first_pos: int, pos: int, qf: torch.Tensor, kb: torch.Tensor, vb: torch.Tensor,
                  q_norm: torch.Tensor, k_norm: torch.Tensor, tab: torch.Tensor, out: torch.Tensor | None = None,
                  out16: torch.Tensor | None = None, eps: float = 1e-6) -> None:
        """The layer's step around the KV path in two launches (quad.rs:113-125): rmsnorm of q and k heads, rope2,
        kv_rope2 + kv_copy of rows [pos, pos + ntok), the attention, attn_gate (out, f32) / attn_gate16 (out16, f16).
        qf [ntok][16][512] (query | gate per head), kb [ntok][2][256], vb [ntok][512], norms [256], tab [ntok][64]."""
        inp = _lib.StepIn(_ptr(qf), _ptr(kb), _ptr(vb), _ptr(q_norm), _ptr(k_norm), _ptr(tab), eps)
        check(_lib.lib().mkv_attn_step(self._h, layer, first_pos, pos, qf.shape[0], C.byref(inp),
                                       _ptr(out) if out is not None else None, _ptr(out16) if out16 is not None else None))

    def attn_verify_partial(self, layer: int, first_pos: int, pos: int, q: torch.Tensor, rec: torch.Tensor) -> None:
        """This shard's un-normalised record [64][258] for the step."""
        check(_lib.lib().mkv_attn_verify_partial(self._h, layer, first_pos, pos, q.shape[0], _ptr(q), _ptr(rec)))

    def attn_prefill(self, layer: int, first_pos: int, pos0: int, q: torch.Tensor, out: torch.Tensor) -> None:
        """q_f16 + attn_fa_mx / attn_fa / attn_fd4 (+combine): q [ntok][16][256] f32 (`qr`) or f16 (`qh`, f16 cache only),
        out f32 [ntok][16][256]; the block's K/V appended before."""
        assert q.dtype in (torch.float32, torch.float16)
        check(_lib.lib().mkv_attn_prefill(self._h, layer, first_pos, pos0, q.shape[0], _ptr(q), int(q.dtype == torch.float16),
                                          _ptr(out)))

    def dispatch(self, layer: int, op: str, uniform, in0=None, in1=None, out=None) -> None:
        """The reference's own form: WGSL entry point name + its 8-word uniform (ops.wgsl:4)."""
        u = (C.c_uint32 * 8)(*[int(x) & 0xFFFFFFFF for x in uniform])
        check(_lib.lib().mkv_dispatch(self._h, layer, op.encode(), u, _ptr(in0), _ptr(in1), _ptr(out)))

    # -- prefix cache
    def snapshot_bytes(self, p: int) -> int:
        return int(_lib.lib().mkv_snapshot_bytes(self._h, p))

    def read_root(self, p: int, payload: torch.Tensor | None = None, wait: bool = True) -> Root:
        """Engine::read_root, KV part (engine.rs:784-802): rows [0, p) to pinned host memory."""
        n = self.snapshot_bytes(p)
        if payload is None:
            payload = torch.empty(n, dtype=torch.uint8, pin_memory=True)
        w = C.c_size_t()
        check(_lib.lib().mkv_snapshot(self._h, p, payload.data_ptr(), payload.numel(), C.byref(w)))
        if wait:
            self.snapshot_wait()
        return Root(p, self.fmt, self.n_layers, payload[: w.value])

    def snapshot_wait(self) -> None:
        check(_lib.lib().mkv_snapshot_wait(self._h))

    def write_root(self, root: Root) -> None:
        """Engine::write_root, KV part (engine.rs:804-823)."""
        if root.fmt != self.fmt or root.n_layers != self.n_layers:
            raise MkvError(_lib.ERR_FORMAT, "root of another format or layer count")
        check(_lib.lib().mkv_restore(self._h, root.p, root.payload.data_ptr(), root.payload.numel()))

    def check_guards(self) -> int:
        """Canary bytes around this cache's buffers that were overwritten (always 0 with the shipped library, which has no
        guards; the checked build is `make -C mechta_b200/csrc checks`, selected with MKV_LIB_PATH)."""
        bad = C.c_uint64(0)
        check(_lib.lib().mkv_cache_check_guards(self._h, C.byref(bad)))
        return int(bad.value)

    def close(self) -> None:
        if self._h:
            bad = self.check_guards() if _lib.lib().mkv_checks_enabled() else 0
            _lib.lib().mkv_cache_destroy(self._h)
            self._h = C.c_void_p()
            if bad:
                raise _lib.MkvError(-1, f"{bad} guard bytes around the cache's buffers were overwritten")

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


def _need(ok, text: str) -> None:
    if not ok:
        raise MkvError(_lib.ERR_INVALID, text)


def _u32(*numbers: int) -> None:
    """Refuses what ctypes would cut to 32 bits."""
    if min(numbers) < 0 or max(numbers) >= 2**32:
        _need(False, f"{numbers}: must lie between 0 and 2^32 - 1")


def _u32_array(numbers) -> np.ndarray:
    """Whole numbers as uint32; refuses those that a cast would cut or round."""
    a = np.ascontiguousarray(numbers)
    if a.dtype.kind not in "iu" and a.size:
        _need(False, f"{a.dtype}: must be whole numbers from 0 to 2^32 - 1")
    words = a.astype(np.int64, copy=False).view(np.uint32)  # the low half of each number, then the high half
    if words[..., 1::2].any():
        _need(False, "numbers must lie between 0 and 2^32 - 1")
    return words[..., ::2]


def _fmt_of(t: torch.Tensor) -> int:
    if t.dtype is torch.float32:
        return _lib.F32
    if t.dtype is not torch.float16:
        _need(False, f"{t.dtype}: must be float16 or float32")
    return _lib.F16


def _block(t: torch.Tensor, device: int, what: str) -> tuple[tuple, int, int]:
    """Shape, token and head stride (0 where they are dense, or where there is one token or head) of a [tokens][heads][dims] tensor on
    `device` whose dims are contiguous and whose tokens and heads are not broadcast."""
    shape = t.shape
    if len(shape) == 3 and t.is_contiguous() and (device < 0 or t.get_device() == device):
        return shape, 0, 0
    stride = t.stride()
    if len(shape) != 3 or (stride[2] != 1 and shape[2] > 1 and 0 not in shape):
        _need(False, f"{what} must be [tokens][heads][dims] with contiguous dims")
    ts, hs = (stride[0] if shape[0] > 1 else 0), (stride[1] if shape[1] > 1 else 0)
    if (shape[0] > 1 and ts <= 0) or (shape[1] > 1 and hs <= 0):
        _need(False, f"{what} may not be broadcast")
    if device >= 0 and t.get_device() != device:
        _need(False, f"{what} must be on cuda:{device}")
    return shape, ts, hs


class Rope:
    """Rotary positions (mkv_rope): which dims turn, how they pair, how the frequencies are scaled for long contexts. The defaults
    are the reference's (engine.rs:108-114); without `ctx` only `freqs` can be asked for."""

    LAYOUTS = {"half": 0, "interleaved": 1}
    SCALINGS = {"none": 0, "linear": 1, "ntk": 2, "yarn": 3}

    def __init__(self, ctx: KvContext | None, dims: int = 64, base: float = 1e7, layout: str = "half", scaling: str = "none",
                 factor: float = 1.0, original: float = 0.0, slow: float = 0.0, fast: float = 0.0):
        self._h = C.c_void_p()
        _need(layout in self.LAYOUTS, f"layout {layout!r}: one of {sorted(self.LAYOUTS)}")
        _need(scaling in self.SCALINGS, f"scaling {scaling!r}: one of {sorted(self.SCALINGS)}")
        self.ctx, self.dims = ctx, int(dims)
        _need(0 <= self.dims < 2**31, f"{dims} rotated dims")
        d = _lib.RopeDesc(self.dims, self.LAYOUTS[layout], self.SCALINGS[scaling], base, factor, original, slow, fast)
        check(_lib.lib().mkv_rope_create(C.byref(d), C.byref(self._h)))
        self._apply = _lib.lib().mkv_rope_apply

    def freqs(self) -> tuple[np.ndarray, float]:
        """Radians per position of each pair, and the factor on cosine and sine."""
        f, m = np.empty(self.dims // 2), C.c_double()
        check(_lib.lib().mkv_rope_freqs(self._h, f.ctypes.data_as(C.c_void_p), C.byref(m)))
        return f, m.value

    def apply(self, x: torch.Tensor, positions: torch.Tensor, out: torch.Tensor, backward: bool = False) -> None:
        """out = x rotated at `positions` (int32 [tokens]); x, out [tokens][heads][dims], f16 or f32 each, any token and head
        strides, the same memory allowed. backward: the transposed map, for gradients."""
        ctx = self.ctx
        _need(ctx is not None, "a Rope without a context does not run")
        shape, xt, xh = _block(x, ctx.device, "x")
        out_shape, yt, yh = _block(out, ctx.device, "out")
        if shape != out_shape:
            _need(False, f"x is {tuple(shape)}, out {tuple(out_shape)}")
        n, heads, dim = shape
        if max(shape) >= 2**31:
            _need(False, f"x is {tuple(shape)}: at most 2^31 - 1 of each")
        if positions.dtype is not torch.int32 or positions.shape != (n,) or not positions.is_contiguous() or positions.get_device() != ctx.device:
            _need(False, f"positions must be contiguous int32 [tokens] on cuda:{ctx.device}")
        r = _lib.RopeRows(x.data_ptr(), out.data_ptr(), _fmt_of(x), _fmt_of(out), n, heads, dim, xt, xh, yt, yh, positions.data_ptr(), backward)
        check(self._apply(ctx._h, self._h, C.byref(r)))

    def close(self) -> None:
        if self._h:
            _lib.lib().mkv_rope_destroy(self._h)
            self._h = C.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class KvPool:
    """Pages for the K and V rows of many sequences (mkv_pool). `items` of write() and attn() are rows of (sequence, first_pos, pos,
    ntok): a [n][4] uint32 array, or a list of such tuples. Without a context the bookkeeping alone works."""

    def __init__(self, ctx: KvContext | None, fmt: KvFormat, n_layers: int, n_pages: int, page_tokens: int, max_seqs: int, max_tokens: int,
                 q_heads: int = HQ, kv_heads: int = HKV, head_dim: int = D):
        self._h = C.c_void_p()
        self.ctx, self.fmt, self.n_layers, self.n_pages, self.page_tokens = ctx, KvFormat(fmt), n_layers, n_pages, page_tokens
        self.q_heads, self.kv_heads, self.head_dim, self.max_seqs = q_heads, kv_heads, head_dim, max_seqs
        _u32(n_pages, page_tokens, max_seqs, max_tokens)
        for v in (n_layers, q_heads, kv_heads, head_dim):
            _need(0 <= v < 2**31, f"{v} is no size")
        _need(ctx is None or ctx._h, "the context is closed")  # (a null handle would make a pool of the bookkeeping alone)
        d = _lib.PoolDesc(int(fmt), n_layers, n_pages, page_tokens, max_seqs, max_tokens, q_heads, kv_heads, head_dim)
        L = _lib.lib()
        check(L.mkv_pool_create(ctx._h if ctx is not None else None, C.byref(d), C.byref(self._h)))
        self._dtype, self._device = self.fmt.torch_dtype, ctx.device if ctx is not None else -1
        self._write, self._attn, self._lib = L.mkv_pool_write, L.mkv_attn_pool, L
        self._out = C.c_uint32()  # where calls put a number
        self._out_ref = C.byref(self._out)

    # -- bookkeeping
    @property
    def free_pages(self) -> int:
        return self._lib.mkv_pool_free_pages(self._h)

    def create(self) -> int:
        """An empty sequence."""
        check(self._lib.mkv_seq_create(self._h, self._out_ref))
        return self._out.value

    def fork(self, seq: int, length: int | None = None, n: int = 1, copy: bool = False) -> list[int]:
        """n sequences that begin with the first `length` rows of `seq` (all of them by default), on the same pages or on copies."""
        _need(0 < n <= self.max_seqs, f"fork of {n} sequences: 1 to {self.max_seqs}")
        if length is None:
            length = self.length(seq)
        if not (0 <= seq < 2**32 and 0 <= length < 2**32):
            _u32(seq, length)
        if n == 1:
            check(self._lib.mkv_seq_fork(self._h, seq, length, copy, 1, self._out_ref))
            return [self._out.value]
        kids = (C.c_uint32 * n)()
        check(self._lib.mkv_seq_fork(self._h, seq, length, copy, n, kids))
        return kids[:]

    def free(self, seqs) -> None:
        if type(seqs) is list and {*map(type, seqs)} <= {int}:
            if seqs:
                _u32(*seqs)
            a, n = (C.c_uint32 * len(seqs))(*seqs), len(seqs)
        else:
            held = np.ascontiguousarray(_u32_array(seqs)).reshape(-1)
            a, n = held.ctypes.data, held.size
        check(self._lib.mkv_seq_free(self._h, a, n))

    def truncate(self, seq: int, length: int) -> None:
        if not (0 <= seq < 2**32 and 0 <= length < 2**32):
            _u32(seq, length)
        check(self._lib.mkv_seq_truncate(self._h, seq, length))

    def set_len(self, seq: int, length: int) -> None:
        """Declares rows valid that the host fills itself (buffer_tensors), in all layers."""
        _u32(seq, length)
        check(self._lib.mkv_seq_set_len(self._h, seq, length))

    def length(self, seq: int) -> int:
        if not 0 <= seq < 2**32:
            _u32(seq, seq)
        return self._lib.mkv_seq_len(self._h, seq)

    def pages(self, seq: int) -> np.ndarray:
        _u32(seq, seq)
        n = C.c_uint32()
        check(_lib.lib().mkv_seq_pages(self._h, seq, None, 0, C.byref(n)))
        a = np.empty(n.value, np.uint32)
        check(_lib.lib().mkv_seq_pages(self._h, seq, a.ctypes.data, a.size, C.byref(n)))
        return a

    def compact(self) -> int:
        """Moves the pages in use together; returns how many moved."""
        check(self._lib.mkv_pool_compact(self._h, self._out_ref))
        return self._out.value

    # -- rows
    def _layer(self, layer: int) -> None:
        if not 0 <= layer < self.n_layers:
            _need(False, f"layer {layer} outside [0, {self.n_layers})")

    def buffers(self, layer: int) -> tuple[int, int]:
        self._layer(layer)
        k, v = C.c_void_p(), C.c_void_p()
        check(_lib.lib().mkv_pool_buffers(self._h, layer, C.byref(k), C.byref(v)))
        return k.value, v.value

    def buffer_tensors(self, layer: int) -> tuple[torch.Tensor, torch.Tensor]:
        """Zero-copy torch views [n_pages][page_tokens][kv_heads][head_dim] of a layer's K and V pages; a view keeps the pool alive."""
        shape = (self.n_pages, self.page_tokens, self.kv_heads, self.head_dim)
        return tuple(_as_tensor(p, self.n_pages * self.page_tokens * self.kv_heads * self.head_dim, self.fmt.torch_dtype, self.ctx.device, self).view(shape)
                     for p in self.buffers(layer))

    def _rows(self, t: torch.Tensor, heads: int, rows: int, what: str) -> int:
        """Checks [rows][heads][head_dim] with dense heads; the token stride (0 for one token)."""
        shape, ts, hs = _block(t, self._device, what)
        if shape != (rows, heads, self.head_dim):
            _need(False, f"{what} is {tuple(shape)}, the items want {(rows, heads, self.head_dim)}")
        if heads > 1 and rows > 0 and hs not in (0, self.head_dim):
            _need(False, f"{what}: a token's heads must be contiguous")
        return ts

    @staticmethod
    def _items(items) -> tuple[bytes, int, int]:
        """The items as the library takes them, their number, their tokens."""
        a = items
        if type(a) is list and a:
            try:
                if {*map(len, a)} != {4}:
                    _need(False, "items are rows of (sequence, first_pos, pos, ntok)")
                a = array.array("I", itertools.chain.from_iterable(a))
            except (TypeError, OverflowError):
                _need(False, "items must be whole numbers from 0 to 2^32 - 1")
            return a.tobytes(), len(items), sum(a[3::4])
        if not (type(a) is np.ndarray and a.dtype == np.uint32):
            a = _u32_array(items)
        if a.ndim != 2 or a.shape[1] != 4:
            _need(a.size == 0, "items are rows of (sequence, first_pos, pos, ntok)")
            a = a.reshape(0, 4)
        n = len(a)
        rows = sum(a[:, 3].tolist()) if n <= 64 else int(a[:, 3].sum(dtype=np.int64))
        return a.tobytes(), n, rows  # (a copy in rows' order, sooner made than an array's address is asked for)

    def write(self, layer: int, items, k: torch.Tensor, v: torch.Tensor, rope: Rope | None = None) -> None:
        """New rows of the items' sequences in one layer; k, v f32 or f16 [tokens of all items][kv_heads][head_dim]. rope rotates k at
        the rows' positions."""
        self._layer(layer)
        a, n, rows = self._items(items)
        if k.dtype is not v.dtype:
            _need(False, "k and v must have one type")
        if rope is not None and not rope._h:
            _need(False, "rope is closed")  # (a null handle would mean: k is rotated already)
        r = _lib.PoolRows(k.data_ptr(), v.data_ptr(), _fmt_of(k), self._rows(k, self.kv_heads, rows, "k"), self._rows(v, self.kv_heads, rows, "v"),
                          rope._h if rope is not None else None)
        check(self._write(self._h, layer, a, n, C.byref(r)))

    def attn(self, layer: int, items, q: torch.Tensor, out: torch.Tensor, window: int = 0, sinks: torch.Tensor | None = None,
             scale: float = 0.0) -> None:
        """Attention of the items' tokens over their sequences; q, out in the pool's type, [tokens of all items][q_heads][head_dim].
        scale 0 = 1 / sqrt(head_dim); sinks f32 [q_heads]."""
        self._layer(layer)
        a, n, rows = self._items(items)
        if q.dtype is not self._dtype or out.dtype is not self._dtype:
            _need(False, f"q and out must be {self._dtype}")
        if not 0 <= window < 2**32:
            _need(False, f"window {window}")
        if sinks is not None:
            _need(sinks.dtype is torch.float32 and sinks.is_contiguous() and sinks.shape == (self.q_heads,), "sinks must be f32 [q_heads]")
            _need(sinks.get_device() == self._device, "sinks must be where the pool is")
        r = _lib.PoolAttn(q.data_ptr(), out.data_ptr(), self._rows(q, self.q_heads, rows, "q"), self._rows(out, self.q_heads, rows, "out"), scale,
                          window, sinks.data_ptr() if sinks is not None else None)
        check(self._attn(self._h, layer, a, n, C.byref(r)))

    def close(self) -> None:
        if self._h:
            _lib.lib().mkv_pool_destroy(self._h)
            self._h = C.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class KvExchange:
    """Mailboxes for the peer exchange of shard records (mkv_exchange): every rank's attention kernel stores its
    record into every rank's mailbox over NVLink, no collective call. `gather_handles(my_handle) -> [bytes] * world`
    is how the 64-byte IPC handles travel between the processes (e.g. torch.distributed.all_gather_object)."""

    def __init__(self, ctx: KvContext, rank: int, world: int, gather_handles=None):
        self.ctx, self.rank, self.world = ctx, rank, world
        self._h = C.c_void_p()
        check(_lib.lib().mkv_exchange_create(ctx._h, rank, world, C.byref(self._h)))
        mine = C.create_string_buffer(64)
        check(_lib.lib().mkv_exchange_handle(self._h, mine))
        handles = [mine.raw] if world == 1 else gather_handles(mine.raw)
        handles = [h if h is not None else bytes(64) for h in handles]  # None = a rank that never joined
        assert len(handles) == world and all(len(h) == 64 for h in handles)
        check(_lib.lib().mkv_exchange_connect(self._h, b"".join(handles)))

    def attn_verify(self, cache: "KvCache", layer: int, first_pos: int, pos: int, q: torch.Tensor, out: torch.Tensor) -> None:
        """Local record -> peer stores into all mailboxes -> merge; `out` is final on every rank."""
        check(_lib.lib().mkv_attn_verify_exchange(cache._h, self._h, layer, first_pos, pos, q.shape[0], _ptr(q), _ptr(out)))

    def close(self) -> None:
        if self._h:
            _lib.lib().mkv_exchange_destroy(self._h)
            self._h = C.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


def write_root_file(path: str, tokens, root: Root) -> None:
    """session.rs:92-111 (KV section; n_ssm = 0)."""
    t = np.ascontiguousarray(tokens, np.uint32)
    assert t.size == root.p
    check(_lib.lib().mkv_root_write(path.encode(), int(root.fmt), root.n_layers, root.p, t.ctypes.data_as(C.c_void_p),
                                    root.payload.data_ptr(), root.payload.numel()))


def read_root_file(path: str, fmt: KvFormat, n_layers: int, pin: bool = True) -> tuple[np.ndarray, Root]:
    """session.rs:113-129: returns (tokens, Root)."""
    L = _lib.lib()
    p, nbytes = C.c_uint32(), C.c_size_t()
    check(L.mkv_root_read(path.encode(), int(fmt), n_layers, C.byref(p), None, 0, None, 0, C.byref(nbytes)))
    toks = np.empty(p.value, np.uint32)
    payload = torch.empty(nbytes.value, dtype=torch.uint8, pin_memory=pin)
    check(L.mkv_root_read(path.encode(), int(fmt), n_layers, C.byref(p), toks.ctypes.data_as(C.c_void_p), toks.size,
                          payload.data_ptr(), payload.numel(), C.byref(nbytes)))
    return toks, Root(p.value, KvFormat(fmt), n_layers, payload)


def _as_tensor(ptr: int, numel: int, dtype, device: int, owner=None) -> torch.Tensor:
    """A torch view over device memory owned by the library (no copy); the view keeps `owner` alive."""
    itemsize = torch.empty((), dtype=dtype).element_size()

    class _Mem:
        pass

    m = _Mem()
    m.owner = owner
    typestr = {torch.float16: "<f2", torch.float32: "<f4", torch.uint8: "|u1"}[dtype]
    m.__cuda_array_interface__ = {"shape": (numel,), "typestr": typestr, "data": (ptr, False), "version": 3,
                                  "strides": (itemsize,)}
    return torch.as_tensor(m, device=f"cuda:{device}")
