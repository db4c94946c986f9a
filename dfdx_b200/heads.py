"""Queries and keys between their projections and the attention, and the paged 8-bit key/value cache.

`HeadOps` is the part of `dfdx_b200.Cuda` that norms and rotates query / key heads (training: forward and backward),
appends keys and values to a `KvCache`, reads the cache back, and attends over it (serving).  Like the rest of the
device, the methods take torch tensors as buffers, enqueue on torch's current stream and do no arithmetic of their own.
"""
from __future__ import annotations

import ctypes as C
import importlib.machinery
import importlib.util
from typing import NamedTuple

import torch

from . import _lib


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


_ENTRIES = ("b200_qk_norm_rotary_forward", "b200_qk_norm_rotary_backward", "b200_qk_norm_rotary_backward_workspace_bytes",
            "b200_kv_cache_append", "b200_kv_cache_read", "b200_kv_cache_attention", "b200_kv_cache_attention_workspace_bytes")
_module = None


def _host():
    """The compiled host side (csrc/py_heads.cpp), bound to the library's entry points.  Raises if it is missing, also where
    there is one for another torch or Python."""
    global _module
    if _module is None:
        from .build import module_path
        path = module_path()
        if not path.exists():
            raise RuntimeError(f"{path} is missing: build it with `python -m dfdx_b200.build`")
        loader = importlib.machinery.ExtensionFileLoader("_heads", str(path))
        m = importlib.util.module_from_spec(importlib.util.spec_from_loader("_heads", loader))
        loader.exec_module(m)
        lib = _lib.load()
        m.bind(ShapeMismatch, _lib.check, *(C.cast(getattr(lib, n), C.c_void_p).value for n in _ENTRIES))
        _module = m
    return _module


class HeadOps:
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
        qo, ko = (None, None) if out is None else out
        return _host().qk_forward(self.ordinal, self.amp, q, k, rotary, positions, norm, q_gain, k_gain, eps, qo, ko)

    def qk_norm_rotary_backward(self, q, k, grad_q_out, grad_k_out, rotary=None, positions=None, norm: bool = True, q_gain=None,
                                k_gain=None, eps: float = 1e-6, out=None, gain_grads=None):
        """Gradients of `qk_norm_rotary_forward` from its inputs (nothing else is saved): (grad_q, grad_k, grad_q_gain,
        grad_k_gain), the first two contiguous or `out`, two views, which may be the upstream gradients; the last two f32,
        fresh, or `gain_grads`, two f32 tensors that are added to; None without `norm`.  The gradient of a broadcast view
        comes for each of its elements."""
        gq, gk = (None, None) if out is None else out
        ggq, ggk = (None, None) if gain_grads is None else gain_grads
        return _host().qk_backward(self.ordinal, self.amp, q, k, grad_q_out, grad_k_out, rotary, positions, norm, q_gain, k_gain, eps,
                                   gq, gk, ggq, ggk)

    # -- the paged cache ----------------------------------------------------------------------------
    def kv_cache(self, pages: int, page_size: int, heads: int, d: int) -> KvCache:
        """An empty cache.  It is not filled with anything: only slots that an append has written are read."""
        shape = (pages, heads, page_size, d)
        k, v = (torch.empty(shape, dtype=torch.float8_e4m3fn, device=self.device) for _ in range(2))
        ks, vs = (torch.empty((pages, heads), dtype=torch.float32, device=self.device) for _ in range(2))
        return KvCache(k, v, ks, vs)

    def kv_cache_append(self, cache: KvCache, k, v, cu_tokens, seq_lens, page_table, max_new: int, q=None, rotary=None,
                        positions=None, norm: bool = False, q_gain=None, k_gain=None, eps: float = 1e-6, q_out=None):
        """Writes the keys and values of the new tokens, k and v (T, heads, D), into the cache, the keys normed and rotated
        on the way, and returns their queries q (T, Hq, D), treated likewise (None without q).  Sequence s has the tokens
        [cu_tokens[s], cu_tokens[s + 1]) and, with them, seq_lens[s] slots in use, the pages of which page_table[s] names
        (all int32, on the device); at most `max_new` of them are new.  `positions`: int32 (axes, T), or None for the
        tokens' slots.  See `b200_kv_cache_append` for the scales."""
        return _host().kv_append(self.ordinal, self.amp, cache, k, v, cu_tokens, seq_lens, page_table, max_new, q, rotary, positions,
                                 norm, q_gain, k_gain, eps, q_out)

    def kv_cache_read(self, cache: KvCache, pages, dtype=torch.float16):
        """The values of the given pages (int32): k, v (n, heads, page_size, D) in f16 or f32.  For moving sequences between
        caches, or keys and values into the dense attention.  Slots that no append has written hold anything."""
        if dtype is not torch.float16 and dtype is not torch.float32:
            raise TypeError(f"unsupported dtype {dtype}")
        return _host().kv_read(self.ordinal, cache, pages, dtype is torch.float16)

    def kv_cache_attention(self, cache: KvCache, q, cu_tokens, seq_lens, page_table, max_new: int, alpha: float,
                           causal: bool = True, window: int = 0, out=None, want_lse: bool = False):
        """softmax(alpha * q K^T) V of the new tokens' queries q (T, Hq, D) over the cache; Hq is a multiple of the cache's
        heads.  A token sees the slots up to its own, the last `window` of these if that is not 0; with `causal` false
        all of its sequence's slots.  Returns (out (T, Hq, D), lse (T, Hq) or None); tokens of no sequence are not written.
        The page table's width bounds the lengths and with them the work that is laid out: pass the columns that the
        longest sequence needs."""
        return _host().kv_attention(self.ordinal, self.amp, cache, q, cu_tokens, seq_lens, page_table, max_new, alpha, causal, window,
                                    out, want_lse)
