"""Queries and keys between their projections and the attention, and the paged 8-bit key/value cache.

`HeadOps` is the part of `dfdx_b200.Cuda` that norms and rotates query / key heads (training: forward and backward),
appends keys and values to a `KvCache`, reads the cache back, and attends over it (serving).  Like the rest of the
device, the methods take torch tensors as buffers, enqueue on torch's current stream and do no arithmetic of their own.
"""
from __future__ import annotations

import ctypes as C
import functools
import struct
from typing import NamedTuple

import torch

from . import _lib
from ._lib import B200Error, check


class ShapeMismatch(AssertionError):
    """Raised where the reference panics with `assertion left == right failed` before any launch."""


class Rotary(NamedTuple):
    """A position rotation: `frequencies` (f64, on the device) in radians per position of every rotated pair,
    `axis_pairs` how many pairs, in order, turn with each position axis (one axis: `(pairs,)`; up to three), and whether
    a pair's elements are adjacent (`interleaved`) or `pairs` apart."""
    frequencies: torch.Tensor
    axis_pairs: tuple
    interleaved: bool = False


class KvCache(NamedTuple):
    """`b200_kv_cache`: e4m3 codes `k`, `v` (pages, heads, page_size, d) and f32 block scales (pages, heads)."""
    k: torch.Tensor
    v: torch.Tensor
    k_scale: torch.Tensor
    v_scale: torch.Tensor


# These calls are short: a decoding step's kernels take a few microseconds each, and so does every ctypes object that
# is made for their arguments.  All structs and strides of a call therefore go into one block of words, laid out as
# `b200_head_op`, `b200_kv_cache`, `b200_kv_batch` and the stride arrays are, and are passed by address.
_entry = functools.lru_cache(None)(_lib.by_address)
_packer = functools.lru_cache(None)(lambda n: struct.Struct(f"={n}Q").pack)
_double_bits = functools.lru_cache(64)(lambda x: struct.unpack("<Q", struct.pack("<d", x))[0])


def _block(*words):
    """(the block, which has to outlive the call; its address)"""
    blk = C.c_char.from_buffer(bytearray(_packer(len(words))(*words)))
    return blk, C.addressof(blk)


def _data(t):
    return 0 if t is None else t.data_ptr()


class HeadOps:
    # -- plumbing ---------------------------------------------------------------------------------
    def _here(self, *tensors) -> None:
        """Every operand on this device; the C ABI would read another device's memory, or the host's, as its own."""
        for t in tensors:
            if t is not None and t.get_device() != self.ordinal:
                raise ValueError(f"a tensor on {t.device}, the device is {self.device}")

    def _index(self, t: torch.Tensor, what: str, shape) -> torch.Tensor:
        if t.dtype is not torch.int32:
            raise TypeError(f"{what}: int32 is required, got {t.dtype}")
        if t.shape != shape:
            raise ShapeMismatch(f"{what}: shape {tuple(t.shape)}, {tuple(shape)} is required")
        if not t.is_contiguous():
            raise ValueError(f"{what}: a contiguous tensor is required")
        return t

    def _under_device(self, fn, *args):
        """fn(*args) with this device current, whichever one torch has made so."""
        if torch._C._cuda_getDevice() == self.ordinal:
            return fn(*args)
        with torch.cuda.device(self.ordinal):
            return fn(*args)

    def _raw_stream(self) -> int:
        """`_stream` without the Stream object around it."""
        return torch._C._cuda_getCurrentRawStream(self.ordinal)

    def _head_op(self, d: int, dtype, rotary, norm: bool, q_gain, k_gain, eps: float):
        """The words of a `b200_head_op`, and the number of position axes it reads."""
        f, axes, n0, n1, n2, inter = 0, 0, 0, 0, 0, 0
        if rotary is not None:
            freq, axis_pairs, inter = rotary
            if freq.dtype is not torch.float64 or not freq.is_contiguous():
                raise TypeError("Rotary.frequencies: a contiguous f64 tensor is required")
            if not 1 <= len(axis_pairs) <= 3 or min(axis_pairs) < 0:
                raise ShapeMismatch(f"Rotary.axis_pairs: one to three counts are required, got {axis_pairs}")
            n0, n1, n2 = (*axis_pairs, 0, 0)[:3]
            if freq.numel() != n0 + n1 + n2 or 2 * (n0 + n1 + n2) > d:
                raise ShapeMismatch(f"Rotary: {freq.numel()} frequencies for pairs {axis_pairs} of heads of {d}")
            axes = 3 if n2 else 2 if n1 else 1 if n0 else 0
            self._here(freq)
            f = freq.data_ptr()
        for g in (q_gain, k_gain):
            if g is None:
                continue
            if not norm:
                raise ValueError("a gain belongs to the norm")
            if g.dim() != 1 or g.shape[0] != d or g.dtype is not dtype or not g.is_contiguous():
                raise ShapeMismatch(f"gain: {d} contiguous elements of {dtype} are required")
            self._here(g)
        return (f, n0, n1, n2, bool(inter) | bool(norm) << 32, _double_bits(float(eps)), _data(q_gain), _data(k_gain)), axes

    def _float(self, t: torch.Tensor, *others) -> int:
        """The dtype code of operands that are all f16 or all f32."""
        dt = t.dtype
        for o in others:
            if o is not None and o.dtype is not dt:
                raise TypeError(f"{dt} and {o.dtype}: one type is required")
        if dt is torch.float16:
            return _lib.AMP_F16 if self.amp else _lib.F16
        if dt is torch.float32:
            return _lib.F32
        raise TypeError(f"unsupported dtype {dt}: f16 or f32 is required")

    def _qk(self, q, k):
        qs, ks = q.shape, k.shape
        if len(qs) == 4 and len(ks) == 4:
            (b, s, hq, d), (b2, s2, hk, d2) = qs, ks
            if (b, s, d) == (b2, s2, d2):
                return b, s, hq, hk, d
        raise ShapeMismatch(f"q {tuple(qs)}, k {tuple(ks)}: (batch, tokens, heads, d) each are required")

    @staticmethod
    def _like(what: str, given, t):
        """`given`, a view shaped and typed like t, or a fresh contiguous tensor of that kind."""
        if given is None:
            return torch.empty_like(t, memory_format=torch.contiguous_format)
        if given.shape != t.shape or given.dtype is not t.dtype:
            raise ShapeMismatch(f"{what}: {tuple(given.shape)} {given.dtype}, {tuple(t.shape)} {t.dtype} is required")
        return given

    # -- norm and rotation of queries and keys ------------------------------------------------------
    def rotary_frequencies(self, axis_pairs, base: float = 10000.0) -> torch.Tensor:
        """`Rotary.frequencies` of the usual schedule, base^(-i / n) for the n pairs of each axis."""
        parts = [torch.arange(n, dtype=torch.float64) / max(n, 1) for n in axis_pairs]
        return torch.pow(torch.tensor(base, dtype=torch.float64), -torch.cat(parts)).to(self.device)

    def qk_norm_rotary_forward(self, q, k, rotary=None, positions=None, norm: bool = True, q_gain=None, k_gain=None,
                               eps: float = 1e-6, out=None):
        """RMS norm over each head (`norm`; times the gains) and rotation by position (`rotary`) of q (B, S, Hq, D) and
        k (B, S, Hk, D), views with a unit last stride, in one pass.  `positions`: int32 (axes, B, S), or None for the
        index in the sequence.  Returns (q, k) as contiguous tensors, or `out`, two views, which may be q and k."""
        b, s, hq, hk, d = self._qk(q, k)
        dt = self._float(q, k)
        op, axes = self._head_op(d, q.dtype, rotary, norm, q_gain, k_gain, eps)
        if positions is not None:
            self._index(positions, "positions", (max(axes, 1), b, s))
        qo, ko = (None, None) if out is None else out
        qo, ko = self._like("out", qo, q), self._like("out", ko, k)
        self._here(q, k, positions, qo, ko)
        blk, at = _block(*op, *q.stride(), *k.stride(), *qo.stride(), *ko.stride())
        check(self._under_device(_entry("b200_qk_norm_rotary_forward"), dt, at, b, s, hq, hk, d, q.data_ptr(), at + 64, k.data_ptr(),
                                 at + 96, _data(positions), qo.data_ptr(), at + 128, ko.data_ptr(), at + 160, self._raw_stream()),
              "b200_qk_norm_rotary_forward")
        return qo, ko

    def qk_norm_rotary_backward(self, q, k, grad_q_out, grad_k_out, rotary=None, positions=None, norm: bool = True, q_gain=None,
                                k_gain=None, eps: float = 1e-6, out=None, gain_grads=None):
        """Gradients of `qk_norm_rotary_forward` from its inputs (nothing else is saved): (grad_q, grad_k, grad_q_gain,
        grad_k_gain), the first two contiguous or `out`, two views, which may be the upstream gradients; the last two f32,
        fresh, or `gain_grads`, two f32 tensors that are added to; None without `norm`.  The gradient of a broadcast view
        comes for each of its elements."""
        b, s, hq, hk, d = self._qk(q, k)
        if grad_q_out.shape != q.shape or grad_k_out.shape != k.shape:
            raise ShapeMismatch("upstream gradients shaped like q and k are required")
        dt = self._float(q, k, grad_q_out, grad_k_out)
        op, axes = self._head_op(d, q.dtype, rotary, norm, q_gain, k_gain, eps)
        if positions is not None:
            self._index(positions, "positions", (max(axes, 1), b, s))
        gq, gk = (None, None) if out is None else out
        gq, gk = self._like("out", gq, q), self._like("out", gk, k)
        go_q = grad_q_out if grad_q_out.stride(3) == 1 else grad_q_out.contiguous()
        go_k = grad_k_out if grad_k_out.stride(3) == 1 else grad_k_out.contiguous()
        ggq = ggk = ws = None
        need = 0
        if norm:
            if gain_grads is None:
                ggq, ggk = torch.empty((2, d), dtype=torch.float32, device=q.device).unbind(0)
            else:
                ggq, ggk = gain_grads
                for g in (ggq, ggk):
                    if g.dtype is not torch.float32 or g.shape != (d,) or not g.is_contiguous():
                        raise ShapeMismatch(f"gain_grads: two f32 tensors of {d} elements are required")
            need = _entry("b200_qk_norm_rotary_backward_workspace_bytes")(d)
            # from torch's allocator rather than `get_workspace`: calls on several streams, and graphs, each have their own
            ws = torch.empty(need, dtype=torch.uint8, device=q.device)
        self._here(q, k, positions, go_q, go_k, gq, gk, ggq, ggk)
        blk, at = _block(*op, *q.stride(), *k.stride(), *go_q.stride(), *go_k.stride(), *gq.stride(), *gk.stride())
        check(self._under_device(_entry("b200_qk_norm_rotary_backward"), dt, at, b, s, hq, hk, d, q.data_ptr(), at + 64, k.data_ptr(),
                                 at + 96, _data(positions), go_q.data_ptr(), at + 128, go_k.data_ptr(), at + 160, gq.data_ptr(),
                                 at + 192, gk.data_ptr(), at + 224, _data(ggq), _data(ggk), gain_grads is not None, _data(ws), need,
                                 self._raw_stream()), "b200_qk_norm_rotary_backward")
        return gq, gk, ggq, ggk

    # -- the paged cache ----------------------------------------------------------------------------
    def kv_cache(self, pages: int, page_size: int, heads: int, d: int) -> KvCache:
        """An empty cache.  It is not filled with anything: only slots that an append has written are read."""
        shape = (pages, heads, page_size, d)
        k, v = (torch.empty(shape, dtype=torch.float8_e4m3fn, device=self.device) for _ in range(2))
        ks, vs = (torch.empty((pages, heads), dtype=torch.float32, device=self.device) for _ in range(2))
        return KvCache(k, v, ks, vs)

    def _cache_words(self, c: KvCache):
        """The words of a `b200_kv_cache`."""
        ck, cv, sk, sv = c
        shape = tuple(ck.shape)
        two = shape[:2]
        if len(shape) != 4 or cv.shape != shape or sk.shape != two or sv.shape != two:
            raise ShapeMismatch(f"cache: codes {tuple(ck.shape)}, {tuple(cv.shape)}, scales {tuple(sk.shape)}, {tuple(sv.shape)}")
        if ck.dtype is not torch.float8_e4m3fn or cv.dtype is not torch.float8_e4m3fn or sk.dtype is not torch.float32 \
                or sv.dtype is not torch.float32:
            raise TypeError("cache: float8_e4m3fn codes and f32 scales are required")
        if not (ck.is_contiguous() and cv.is_contiguous() and sk.is_contiguous() and sv.is_contiguous()):
            raise ValueError("cache: contiguous tensors are required")
        self._here(ck, cv, sk, sv)
        return ck.data_ptr(), cv.data_ptr(), sk.data_ptr(), sv.data_ptr(), *shape

    def _batch_words(self, tokens: int, cu_tokens, seq_lens, page_table, max_new: int):
        """The words of a `b200_kv_batch`."""
        n = seq_lens.shape[0]
        self._index(seq_lens, "seq_lens", (n,))
        self._index(cu_tokens, "cu_tokens", (n + 1,))
        if page_table.dtype is not torch.int32 or page_table.dim() != 2 or page_table.shape[0] != n:
            raise ShapeMismatch(f"page_table: int32 ({n}, pages) is required, got {page_table.dtype} {tuple(page_table.shape)}")
        width = page_table.shape[1]
        if width > 1 and page_table.stride(1) != 1:
            raise ValueError("page_table: a unit last stride is required")
        if max_new < 0:
            raise ShapeMismatch(f"max_new: {max_new}")
        self._here(cu_tokens, seq_lens, page_table)
        return (n, tokens, min(max_new, tokens), cu_tokens.data_ptr(), seq_lens.data_ptr(), page_table.data_ptr(),
                page_table.stride(0) if n > 1 else width, width)

    def kv_cache_append(self, cache: KvCache, k, v, cu_tokens, seq_lens, page_table, max_new: int, q=None, rotary=None,
                        positions=None, norm: bool = False, q_gain=None, k_gain=None, eps: float = 1e-6, q_out=None):
        """Writes the keys and values of the new tokens, k and v (T, heads, D), into the cache, the keys normed and rotated
        on the way, and returns their queries q (T, Hq, D), treated likewise (None without q).  Sequence s has the tokens
        [cu_tokens[s], cu_tokens[s + 1]) and, with them, seq_lens[s] slots in use, the pages of which page_table[s] names
        (all int32, on the device); at most `max_new` of them are new.  `positions`: int32 (axes, T), or None for the
        tokens' slots.  See `b200_kv_cache_append` for the scales."""
        words = self._cache_words(cache)
        heads, d = words[5], words[7]
        t = k.shape[0]
        if v.shape != k.shape or k.shape != (t, heads, d) or (q is not None and (q.dim() != 3 or q.shape[0] != t or q.shape[2] != d)):
            raise ShapeMismatch(f"k {tuple(k.shape)}, v {tuple(v.shape)}, q {None if q is None else tuple(q.shape)}: "
                                f"(tokens, heads, {d}) with the cache's {heads} key heads are required")
        dt = self._float(k, v, q)
        op, axes = self._head_op(d, k.dtype, rotary, norm, q_gain, k_gain, eps)
        if positions is not None:
            self._index(positions, "positions", (max(axes, 1), t))
        batch = self._batch_words(t, cu_tokens, seq_lens, page_table, max_new)
        q_out = None if q is None else self._like("q_out", q_out, q)
        self._here(k, v, q, q_out, positions)
        none = (0, 0, 0)
        blk, at = _block(*words, *batch, *op, *k.stride(), *v.stride(), *(none if q is None else q.stride()),
                         *(none if q is None else q_out.stride()))
        check(self._under_device(_entry("b200_kv_cache_append"), dt, at, at + 64, at + 128, 0 if q is None else q.shape[1], _data(q),
                                 at + 240, k.data_ptr(), at + 192, v.data_ptr(), at + 216, _data(positions), _data(q_out), at + 264,
                                 self._raw_stream()), "b200_kv_cache_append")
        return q_out

    def kv_cache_read(self, cache: KvCache, pages, dtype=torch.float16):
        """The values of the given pages (int32): k, v (n, heads, page_size, D) in f16 or f32.  For moving sequences between
        caches, or keys and values into the dense attention.  Slots that no append has written hold anything."""
        words = self._cache_words(cache)
        n = pages.shape[0]
        self._index(pages, "pages", (n,))
        if dtype is not torch.float16 and dtype is not torch.float32:
            raise TypeError(f"unsupported dtype {dtype}")
        self._here(pages)
        shape = (n, *cache.k.shape[1:])
        k, v = (torch.empty(shape, dtype=dtype, device=self.device) for _ in range(2))
        blk, at = _block(*words)
        check(self._under_device(_entry("b200_kv_cache_read"), _lib.F32 if dtype is torch.float32 else _lib.F16, at, n, pages.data_ptr(),
                                 k.data_ptr(), v.data_ptr(), self._raw_stream()), "b200_kv_cache_read")
        return k, v

    def kv_cache_attention(self, cache: KvCache, q, cu_tokens, seq_lens, page_table, max_new: int, alpha: float,
                           causal: bool = True, window: int = 0, out=None, want_lse: bool = False):
        """softmax(alpha * q K^T) V of the new tokens' queries q (T, Hq, D) over the cache; Hq is a multiple of the cache's
        heads.  A token sees the slots up to its own, the last `window` of these if that is not 0; with `causal` false
        all of its sequence's slots.  Returns (out (T, Hq, D), lse (T, Hq) or None); tokens of no sequence are not written.
        The page table's width bounds the lengths and with them the work that is laid out: pass the columns that the
        longest sequence needs."""
        words = self._cache_words(cache)
        heads, d = words[5], words[7]
        if q.dim() != 3 or q.shape[2] != d or heads == 0 or q.shape[1] % heads:
            raise ShapeMismatch(f"q {tuple(q.shape)}: (tokens, a multiple of {heads} heads, {d}) is required")
        t, hq = q.shape[0], q.shape[1]
        dt = self._float(q)
        if window < 0:
            raise ShapeMismatch(f"window: {window}")
        batch = self._batch_words(t, cu_tokens, seq_lens, page_table, max_new)
        out = self._like("out", out, q)
        lse = torch.empty((t, hq), dtype=torch.float32, device=q.device) if want_lse else None
        self._here(q, out)
        blk, at = _block(*words, *batch, *q.stride(), *out.stride())
        need = self._under_device(_entry("b200_kv_cache_attention_workspace_bytes"), at, at + 64, hq, causal, window)
        # from torch's allocator rather than `get_workspace`: calls on several streams, and graphs, each have their own
        ws = torch.empty(need, dtype=torch.uint8, device=q.device) if need else None
        check(self._under_device(_entry("b200_kv_cache_attention"), dt, at, at + 64, hq, q.data_ptr(), at + 128, alpha, causal, window,
                                 out.data_ptr(), at + 152, _data(lse), _data(ws), need, self._raw_stream()), "b200_kv_cache_attention")
        return out, lse
