"""Decode attention of a batch of sequences that share a prefix (rb_prefix_attn).

Beams, or several samples of one prompt, attend to the same prompt rows: the prefix is kept once and read once for the
whole batch, and each sequence adds the rows it wrote itself. Both are kv_cache.KVCache objects of one format:

    attn = PrefixAttention(q, out, prefix=prompt_cache, prefix_len=n_prompt, own=beam_cache, own_len=lens)   # built once
    attn()                                                                                                 # every step

q and out are [B, n_q_heads, head_dim] (strided in their first dimension: a view into a fused projection's output
works), prefix_len an int64 [1] and own_len an int64 [B] tensor on the device, so one CUDA graph serves every step.
A sequence without any row gets zeros. With prefix=None this is batched decode attention over own caches. The
single-sequence counterpart is attention.DecodeAttention; the reference has no batched one.
"""
import ctypes

import torch

from . import _lib, config
from .cuda_gemv import _on_device, _require


class PrefixAttention:
    """Owns its workspace; calls sharing one object must be issued on one stream. scale: head_dim ** -0.5 by default.
    kernel: which kernel streams the prefix, "tc" (tcgen05, 128 query rows a key-value head at a time) or "mma" (warp
    level); None: by the number of rows and the prefix's capacity."""

    def __init__(self, q, out, prefix=None, prefix_len=None, own=None, own_len=None, scale=None, kernel=None):
        _require(kernel in _lib.KERNEL_FLAGS, f"kernel must be None, 'tc' or 'mma', got {kernel!r}")
        _require(prefix is not None or own is not None, "a prefix or own rows are needed")
        c = prefix if prefix is not None else own
        B, nq, hd = q.shape if q.dim() == 3 else (0, 0, 0)
        _require(q.dim() == 3 and hd == c.head_dim, f"q must be [B, n_q_heads, {c.head_dim}], got {tuple(q.shape)}")
        _require(nq >= 1 and nq % c.n_kv_heads == 0 and nq // c.n_kv_heads <= 16,
                 f"{nq} query heads over {c.n_kv_heads} key-value heads: 1 to 16 each are supported")
        for t, nm in ((q, "q"), (out, "out")):
            _require(t.shape == q.shape and t.dtype == c.dtype and t.device == c.device,
                     f"{nm} must be a {c.dtype} {tuple(q.shape)} tensor on {c.device}")
            _require(t.stride(2) == 1 and t.stride(1) == hd, f"{nm}'s heads must be contiguous")
        for cache, n, lens, nm in ((prefix, 1, prefix_len, "prefix"), (own, B, own_len, "own")):
            if cache is None:
                _require(lens is None, f"{nm}_len without {nm}")
                continue
            _require(cache.n_seqs == n, f"{nm} must hold {n} sequence(s), not {cache.n_seqs}")
            _require((cache.fmt, cache.dtype, cache.n_kv_heads, cache.head_dim, cache.device) ==
                     (c.fmt, c.dtype, c.n_kv_heads, c.head_dim, c.device), "prefix and own must be alike")
            _require(lens is not None and lens.dtype == torch.int64 and lens.device == c.device and lens.numel() == n
                     and lens.is_contiguous(), f"{nm}_len must be a contiguous int64 [{n}] tensor on {c.device}")
        self.device = c.device
        self._keep = (q, out, prefix, prefix_len, own, own_len)
        a = _lib.PrefixAttnArgs()
        a.q, a.ldq, a.out, a.ldo = q.data_ptr(), q.stride(0), out.data_ptr(), out.stride(0)
        a.n_seqs, a.n_q_heads = B, nq
        if prefix is not None:
            a.prefix, a.prefix_len = ctypes.pointer(prefix.desc), prefix_len.data_ptr()
        if own is not None:
            a.own, a.own_len = ctypes.pointer(own.desc), own_len.data_ptr()
        a.scale = float(hd ** -0.5 if scale is None else scale)
        with _on_device(self.device):
            need = _lib.lib().rb_prefix_attn_workspace(ctypes.byref(a))
        if need < 0:
            _lib.check("rb_prefix_attn_workspace", -need)
        self.ws = torch.empty(need, dtype=torch.uint8, device=self.device)
        a.ws, a.ws_bytes = self.ws.data_ptr(), need
        self._args, self._ref, self._flags = a, ctypes.byref(a), _lib.KERNEL_FLAGS[kernel]

    def __call__(self):
        with _on_device(self.device):
            st = _lib.lib().rb_prefix_attn(self._ref, config.flags() | self._flags, _lib.stream_ptr(self.device))
        _lib.check("rb_prefix_attn", st)
