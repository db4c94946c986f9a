"""Queries and keys between their projections and the attention, and the paged 8-bit key/value cache.

`HeadOps` is the part of `dfdx_b200.Cuda` that norms and rotates query / key heads (training: forward and backward),
appends keys and values to a `KvCache`, reads the cache back, and attends over it (serving).  Like the rest of the
device, the methods take torch tensors as buffers, enqueue on torch's current stream and do no arithmetic of their own.
"""
from __future__ import annotations

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


_IN_CALL = (torch.float32, torch.float16)


def _strides(t: torch.Tensor):
    return _lib.strides(t.stride())


def _data(t):
    return None if t is None else t.data_ptr()


class HeadOps:
    # -- plumbing ---------------------------------------------------------------------------------
    def _here(self, *tensors) -> None:
        """Every operand on this device; the C ABI would read another device's memory, or the host's, as its own."""
        for t in tensors:
            if t is not None and t.device != self.device:
                raise ValueError(f"a tensor on {t.device}, the device is {self.device}")

    def _index(self, t: torch.Tensor, what: str, shape) -> torch.Tensor:
        if t.dtype != torch.int32:
            raise TypeError(f"{what}: int32 is required, got {t.dtype}")
        if tuple(t.shape) != tuple(shape):
            raise ShapeMismatch(f"{what}: shape {tuple(t.shape)}, {tuple(shape)} is required")
        if not t.is_contiguous():
            raise ValueError(f"{what}: a contiguous tensor is required")
        return t

    def _under_device(self, fn, *args):
        """fn(*args) with this device current, whichever one torch has made so."""
        if torch.cuda.current_device() == self.ordinal:
            return fn(*args)
        with torch.cuda.device(self.ordinal):
            return fn(*args)

    def _call(self, name: str, *args) -> None:
        check(self._under_device(getattr(self.lib, name), *args), name)

    def _head_op(self, d: int, dtype, rotary, norm: bool, q_gain, k_gain, eps: float):
        op = _lib.HeadOp()
        axes = 0
        if rotary is not None:
            f, axis_pairs = rotary.frequencies, tuple(rotary.axis_pairs)
            if f.dtype != torch.float64 or not f.is_contiguous():
                raise TypeError("Rotary.frequencies: a contiguous f64 tensor is required")
            if not 1 <= len(axis_pairs) <= 3 or min(axis_pairs) < 0:
                raise ShapeMismatch(f"Rotary.axis_pairs: one to three counts are required, got {axis_pairs}")
            if f.numel() != sum(axis_pairs) or 2 * sum(axis_pairs) > d:
                raise ShapeMismatch(f"Rotary: {f.numel()} frequencies for pairs {axis_pairs} of heads of {d}")
            self._here(f)
            op.frequencies = f.data_ptr()
            for a, n in enumerate(axis_pairs):
                op.axis_pairs[a] = n
                axes = a + 1 if n else axes
            op.interleaved = int(rotary.interleaved)
        for g in (q_gain, k_gain):
            if g is None:
                continue
            if not norm:
                raise ValueError("a gain belongs to the norm")
            if tuple(g.shape) != (d,) or g.dtype != dtype or not g.is_contiguous():
                raise ShapeMismatch(f"gain: {d} contiguous elements of {dtype} are required")
            self._here(g)
        op.normalize, op.epsilon = int(norm), eps
        op.q_gain, op.k_gain = _data(q_gain), _data(k_gain)
        return op, axes

    def _qk(self, q, k):
        if q.dim() != 4 or k.dim() != 4 or q.shape[:2] != k.shape[:2] or q.shape[3] != k.shape[3]:
            raise ShapeMismatch(f"q {tuple(q.shape)}, k {tuple(k.shape)}: (batch, tokens, heads, d) each are required")
        if q.dtype != k.dtype or q.dtype not in _IN_CALL:
            raise TypeError(f"q {q.dtype}, k {k.dtype}: both f16 or both f32 are required")
        self._here(q, k)

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
        self._qk(q, k)
        b, s, hq, d = q.shape
        hk = k.shape[2]
        op, axes = self._head_op(d, q.dtype, rotary, norm, q_gain, k_gain, eps)
        if positions is not None:
            self._index(positions, "positions", (max(axes, 1), b, s))
            self._here(positions)
        qo, ko = (torch.empty(q.shape, dtype=q.dtype, device=q.device), torch.empty(k.shape, dtype=k.dtype, device=k.device)) \
            if out is None else out
        if out is not None and (qo.shape != q.shape or ko.shape != k.shape or qo.dtype != q.dtype or ko.dtype != k.dtype):
            raise ShapeMismatch("out: views shaped and typed like q and k are required")
        self._here(qo, ko)
        self._call("b200_qk_norm_rotary_forward", self._dtype(q), op, b, s, hq, hk, d, q.data_ptr(),
                   _strides(q), k.data_ptr(), _strides(k), _data(positions), qo.data_ptr(), _strides(qo), ko.data_ptr(),
                   _strides(ko), self._stream())
        return qo, ko

    def qk_norm_rotary_backward(self, q, k, grad_q_out, grad_k_out, rotary=None, positions=None, norm: bool = True, q_gain=None,
                                k_gain=None, eps: float = 1e-6, out=None, gain_grads=None):
        """Gradients of `qk_norm_rotary_forward` from its inputs (nothing else is saved): (grad_q, grad_k, grad_q_gain,
        grad_k_gain), the first two contiguous or `out`, two views, which may be the upstream gradients; the last two f32,
        fresh, or `gain_grads`, two f32 tensors that are added to; None without `norm`.  The gradient of a broadcast view
        comes for each of its elements."""
        self._qk(q, k)
        b, s, hq, d = q.shape
        hk = k.shape[2]
        op, axes = self._head_op(d, q.dtype, rotary, norm, q_gain, k_gain, eps)
        if positions is not None:
            self._index(positions, "positions", (max(axes, 1), b, s))
            self._here(positions)
        if grad_q_out.shape != q.shape or grad_k_out.shape != k.shape or grad_q_out.dtype != q.dtype or grad_k_out.dtype != k.dtype:
            raise ShapeMismatch("upstream gradients shaped and typed like q and k are required")
        gq, gk = (torch.empty(q.shape, dtype=q.dtype, device=q.device), torch.empty(k.shape, dtype=k.dtype, device=k.device)) \
            if out is None else out
        if out is not None and (gq.shape != q.shape or gk.shape != k.shape or gq.dtype != q.dtype or gk.dtype != k.dtype):
            raise ShapeMismatch("out: views shaped and typed like q and k are required")
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
                    if g.dtype != torch.float32 or tuple(g.shape) != (d,) or not g.is_contiguous():
                        raise ShapeMismatch(f"gain_grads: two f32 tensors of {d} elements are required")
            need = self.lib.b200_qk_norm_rotary_backward_workspace_bytes(d)
            # from torch's allocator rather than `get_workspace`: calls on several streams, and graphs, each have their own
            ws = torch.empty(need, dtype=torch.uint8, device=q.device)
        self._here(go_q, go_k, gq, gk, ggq, ggk)
        self._call("b200_qk_norm_rotary_backward", self._dtype(q), op, b, s, hq, hk, d,
                   q.data_ptr(), _strides(q), k.data_ptr(), _strides(k), _data(positions), go_q.data_ptr(), _strides(go_q),
                   go_k.data_ptr(), _strides(go_k), gq.data_ptr(), _strides(gq), gk.data_ptr(), _strides(gk), _data(ggq),
                   _data(ggk), int(gain_grads is not None), _data(ws), need, self._stream())
        return gq, gk, ggq, ggk

    # -- the paged cache ----------------------------------------------------------------------------
    def kv_cache(self, pages: int, page_size: int, heads: int, d: int) -> KvCache:
        """An empty cache.  It is not filled with anything: only slots that an append has written are read."""
        shape = (pages, heads, page_size, d)
        k, v = (torch.empty(shape, dtype=torch.float8_e4m3fn, device=self.device) for _ in range(2))
        ks, vs = (torch.empty((pages, heads), dtype=torch.float32, device=self.device) for _ in range(2))
        return KvCache(k, v, ks, vs)

    def _cache_view(self, c: KvCache):
        pages, heads, page, d = c.k.shape
        if c.v.shape != c.k.shape or c.k_scale.shape != (pages, heads) or c.v_scale.shape != (pages, heads):
            raise ShapeMismatch(f"cache: codes {tuple(c.k.shape)}, {tuple(c.v.shape)}, scales {tuple(c.k_scale.shape)}, {tuple(c.v_scale.shape)}")
        if c.k.dtype != torch.float8_e4m3fn or c.v.dtype != torch.float8_e4m3fn or c.k_scale.dtype != torch.float32 \
                or c.v_scale.dtype != torch.float32:
            raise TypeError("cache: float8_e4m3fn codes and f32 scales are required")
        if not (c.k.is_contiguous() and c.v.is_contiguous() and c.k_scale.is_contiguous() and c.v_scale.is_contiguous()):
            raise ValueError("cache: contiguous tensors are required")
        self._here(*c)
        return _lib.KvCacheView(c.k.data_ptr(), c.v.data_ptr(), c.k_scale.data_ptr(), c.v_scale.data_ptr(), pages, heads, page, d)

    def _kv_batch(self, tokens: int, cu_tokens, seq_lens, page_table, max_new: int):
        n = seq_lens.shape[0]
        self._index(seq_lens, "seq_lens", (n,))
        self._index(cu_tokens, "cu_tokens", (n + 1,))
        if page_table.dtype != torch.int32 or page_table.dim() != 2 or page_table.shape[0] != n:
            raise ShapeMismatch(f"page_table: int32 ({n}, pages) is required, got {page_table.dtype} {tuple(page_table.shape)}")
        if page_table.shape[1] > 1 and page_table.stride(1) != 1:
            raise ValueError("page_table: a unit last stride is required")
        if max_new < 0:
            raise ShapeMismatch(f"max_new: {max_new}")
        self._here(cu_tokens, seq_lens, page_table)
        return _lib.KvBatch(n, tokens, min(max_new, tokens), cu_tokens.data_ptr(), seq_lens.data_ptr(), page_table.data_ptr(),
                            page_table.stride(0) if n > 1 else page_table.shape[1], page_table.shape[1])

    def kv_cache_append(self, cache: KvCache, k, v, cu_tokens, seq_lens, page_table, max_new: int, q=None, rotary=None,
                        positions=None, norm: bool = False, q_gain=None, k_gain=None, eps: float = 1e-6, q_out=None):
        """Writes the keys and values of the new tokens, k and v (T, heads, D), into the cache, the keys normed and rotated
        on the way, and returns their queries q (T, Hq, D), treated likewise (None without q).  Sequence s has the tokens
        [cu_tokens[s], cu_tokens[s + 1]) and, with them, seq_lens[s] slots in use, the pages of which page_table[s] names
        (all int32, on the device); at most `max_new` of them are new.  `positions`: int32 (axes, T), or None for the
        tokens' slots.  See `b200_kv_cache_append` for the scales."""
        view = self._cache_view(cache)
        t, hk, d = k.shape
        if v.shape != k.shape or (hk, d) != (view.heads, view.d) or (q is not None and (q.dim() != 3 or q.shape[0] != t or q.shape[2] != d)):
            raise ShapeMismatch(f"k {tuple(k.shape)}, v {tuple(v.shape)}, q {None if q is None else tuple(q.shape)}: "
                                f"(tokens, heads, {view.d}) with the cache's {view.heads} key heads are required")
        if k.dtype not in _IN_CALL or v.dtype != k.dtype or (q is not None and q.dtype != k.dtype):
            raise TypeError("q, k, v: all f16 or all f32 are required")
        op, axes = self._head_op(d, k.dtype, rotary, norm, q_gain, k_gain, eps)
        if positions is not None:
            self._index(positions, "positions", (max(axes, 1), t))
        batch = self._kv_batch(t, cu_tokens, seq_lens, page_table, max_new)
        if q is not None:
            if q_out is None:
                q_out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
            elif q_out.shape != q.shape or q_out.dtype != q.dtype:
                raise ShapeMismatch("q_out: a view shaped and typed like q is required")
        else:
            q_out = None
        self._here(k, v, q, q_out, positions)
        self._call("b200_kv_cache_append", self._dtype(k), view, batch, op, 0 if q is None else q.shape[1],
                   _data(q), None if q is None else _strides(q), k.data_ptr(), _strides(k), v.data_ptr(), _strides(v),
                   _data(positions), _data(q_out), None if q is None else _strides(q_out), self._stream())
        return q_out

    def kv_cache_read(self, cache: KvCache, pages, dtype=torch.float16):
        """The values of the given pages (int32): k, v (n, heads, page_size, D) in f16 or f32.  For moving sequences between
        caches, or keys and values into the dense attention.  Slots that no append has written hold anything."""
        view = self._cache_view(cache)
        n = pages.shape[0]
        self._index(pages, "pages", (n,))
        if dtype not in _IN_CALL:
            raise TypeError(f"unsupported dtype {dtype}")
        self._here(pages)
        k, v = (torch.empty((n, view.heads, view.page_size, view.d), dtype=dtype, device=self.device) for _ in range(2))
        self._call("b200_kv_cache_read", _lib.F32 if dtype == torch.float32 else _lib.F16, view, n,
                   pages.data_ptr(), k.data_ptr(), v.data_ptr(), self._stream())
        return k, v

    def kv_cache_attention(self, cache: KvCache, q, cu_tokens, seq_lens, page_table, max_new: int, alpha: float,
                           causal: bool = True, window: int = 0, out=None, want_lse: bool = False):
        """softmax(alpha * q K^T) V of the new tokens' queries q (T, Hq, D) over the cache; Hq is a multiple of the cache's
        heads.  A token sees the slots up to its own, the last `window` of these if that is not 0; with `causal` false
        all of its sequence's slots.  Returns (out (T, Hq, D), lse (T, Hq) or None); tokens of no sequence are not written.
        The page table's width bounds the lengths and with them the work that is laid out: pass the columns that the
        longest sequence needs."""
        view = self._cache_view(cache)
        if q.dim() != 3 or q.shape[2] != view.d or q.shape[1] % view.heads:
            raise ShapeMismatch(f"q {tuple(q.shape)}: (tokens, a multiple of {view.heads} heads, {view.d}) is required")
        t, hq, _ = q.shape
        if q.dtype != torch.float16:
            raise B200Error(_lib.ERR_UNSUPPORTED, "b200_kv_cache_attention (f16 queries only)")
        if window < 0:
            raise ShapeMismatch(f"window: {window}")
        batch = self._kv_batch(t, cu_tokens, seq_lens, page_table, max_new)
        if out is None:
            out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        elif out.shape != q.shape or out.dtype != q.dtype:
            raise ShapeMismatch("out: a view shaped and typed like q is required")
        lse = torch.empty((t, hq), dtype=torch.float32, device=q.device) if want_lse else None
        self._here(q, out)
        need = self._under_device(self.lib.b200_kv_cache_attention_workspace_bytes, view, batch, hq, int(causal), window)
        # from torch's allocator rather than `get_workspace`: calls on several streams, and graphs, each have their own
        ws = torch.empty(need, dtype=torch.uint8, device=q.device) if need else None
        self._call("b200_kv_cache_attention", self._dtype(q), view, batch, hq, q.data_ptr(), _strides(q),
                   alpha, int(causal), window, out.data_ptr(), _strides(out), _data(lse), _data(ws), need, self._stream())
        return out, lse
