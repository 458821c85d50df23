"""Key-value caches of a batch of sequences, quantised as they are written and read back (rb_kv_write, rb_kv_read).

The decode attention of one sequence reads a 16-bit cache that the layer's input launch writes (attention.py); this
cache holds a batch, in 16 bits ("plain"), 8 ("int8": 0.51 of the bytes) or 4 ("int4": 0.27), one scale a row of
head_dim values - the granularity of the library's int4 groups:

    cache = KVCache(n_seqs=16, n_kv_heads=8, cache_len=4096, fmt="int8")       # one layer's K and V
    cache.write(k, v, pos)             # k, v [16, n_tokens, 8, 128] (strided views welcome), pos int64 [16] on the device
    k, v = cache.read(0, 512)          # what slots 0..511 stand for, [16, 8, 512, 128]

prefix_attention.PrefixAttention reads these caches in place, beams.BeamReorder permutes them.
The formats (include/rumik_b200.h, rb_kv_format): int8 value = code * s with s = bf16(max|x| / 127); int4 value =
code * s + m with s = bf16((max x - min x) (1 / 15)), in fp32, and m = min x. No reference counterpart (its engine keeps a 16-bit
cache of one sequence, engine/rumik_int4.py:118-130).
"""
import ctypes

import torch

from . import _lib, config
from .cuda_gemv import _on_device, _require

_Strides = ctypes.c_int64 * 3
FORMATS = {"plain": _lib.KV_PLAIN, "int8": _lib.KV_INT8, "int4": _lib.KV_INT4}


class KVCache:
    """k, v [n_seqs, n_kv_heads, cache_len, row]: `dtype` values (plain), uint8 codes + 128 (int8), or uint8 pairs of
    4-bit codes (int4, row = head_dim / 2); k_par, v_par [n_seqs, n_kv_heads, cache_len]: bf16 scales (int8), int32
    words of scale and minimum (int4), None (plain). Calls run on the current stream and are graph-capture safe
    (read allocates its result unless it is given one)."""

    def __init__(self, n_seqs, n_kv_heads, cache_len, head_dim=128, fmt="int8", dtype=torch.float16, device="cuda"):
        _require(fmt in FORMATS, f"fmt must be one of {sorted(FORMATS)}, got {fmt!r}")
        _require(min(n_seqs, n_kv_heads, cache_len) >= 1, "n_seqs, n_kv_heads and cache_len must be at least 1")
        lead = (n_seqs, n_kv_heads, cache_len)

        def pair():
            if fmt == "plain":
                return torch.zeros(lead + (head_dim,), dtype=dtype, device=device), None
            if fmt == "int8":
                return (torch.full(lead + (head_dim,), 128, dtype=torch.uint8, device=device),
                        torch.zeros(lead, dtype=torch.bfloat16, device=device))
            return (torch.zeros(lead + (head_dim // 2,), dtype=torch.uint8, device=device),
                    torch.zeros(lead, dtype=torch.int32, device=device))
        k, k_par = pair()
        v, v_par = pair()
        self._adopt(k, v, k_par, v_par, dtype)

    @classmethod
    def wrap(cls, k, v, k_par=None, v_par=None, dtype=None):
        """A cache over tensors that exist already; the format follows from their types. `dtype`: the values' type of a
        quantised cache."""
        c = cls.__new__(cls)
        c._adopt(k, v, k_par, v_par, dtype)
        return c

    def _adopt(self, k, v, k_par, v_par, dtype):
        if k_par is None:
            self.fmt = "plain"
            _require(dtype is None or dtype == k.dtype, f"a plain cache holds its dtype: {k.dtype}, not {dtype}")
            dtype = k.dtype
        else:
            _require(k.dtype == torch.uint8 and k_par.dtype in (torch.bfloat16, torch.int32),
                     "a quantised cache holds uint8 codes with bfloat16 (int8) or int32 (int4) row parameters")
            self.fmt = "int8" if k_par.dtype == torch.bfloat16 else "int4"
        _require(dtype in (torch.float16, torch.bfloat16), f"values must be fp16 or bf16, got {dtype}")
        _require(k.dim() == 4 and v.shape == k.shape and v.dtype == k.dtype, "k and v must be alike, [n_seqs, n_kv_heads, S, row]")
        for t, nm in ((k, "k"), (v, "v"), (k_par, "k_par"), (v_par, "v_par")):
            if t is None:
                _require(k_par is None and v_par is None, "k_par and v_par go together")
                continue
            _require(t.is_cuda and t.device == k.device and t.is_contiguous(), f"{nm} must be a contiguous CUDA tensor on {k.device}")
        if k_par is not None:
            _require(k_par.shape == k.shape[:3] and v_par.shape == k.shape[:3] and v_par.dtype == k_par.dtype,
                     f"row parameters must be {tuple(k.shape[:3])}")
        self.k, self.v, self.k_par, self.v_par, self.dtype, self.device = k, v, k_par, v_par, dtype, k.device
        self.n_seqs, self.n_kv_heads, self.cache_len = k.shape[:3]
        self.head_dim = k.shape[3] * (2 if self.fmt == "int4" else 1)
        _require(self.head_dim in (64, 128), f"head_dim must be 64 or 128, got {self.head_dim}")
        self.desc = _lib.KvCache(k.data_ptr(), v.data_ptr(), None if k_par is None else k_par.data_ptr(),
                                 None if v_par is None else v_par.data_ptr(), FORMATS[self.fmt], _lib.dtype_code(dtype),
                                 self.n_seqs, self.n_kv_heads, self.head_dim, self.cache_len)
        self._ref = ctypes.byref(self.desc)
        self._empty = torch.empty(0, dtype=dtype, device=k.device)

    def tensors(self):
        """The cache's tensors, for beams.BeamReorder."""
        return [t for t in (self.k, self.v, self.k_par, self.v_par) if t is not None]

    def _rows(self, x, nm):
        shape = x.shape
        if len(shape) == 3:   # one token: [n_seqs, n_kv_heads, head_dim]
            x = x.unsqueeze(1)
            shape = x.shape
        if x.dtype != self.dtype or x.device != self.device:
            _require(False, f"{nm} must be a {self.dtype} tensor on {self.device}")
        if len(shape) != 4 or shape[0] != self.n_seqs or shape[2] != self.n_kv_heads or shape[3] != self.head_dim:
            _require(False, f"{nm} must be [{self.n_seqs}, T, {self.n_kv_heads}, {self.head_dim}] (or without T), got {tuple(shape)}")
        s0, s1, s2, s3 = x.stride()
        _require(s3 == 1, "k and v must have unit stride in their last dimension")
        return x, shape[1], _Strides(s0, s1, s2)

    def write(self, k, v, pos):
        """Rows k, v [n_seqs, T, n_kv_heads, head_dim] (or [n_seqs, n_kv_heads, head_dim]: one token) into the slots
        pos[b] .. pos[b] + T - 1 (pos: int64 [n_seqs] on the device). A slot outside the cache is not written and sets
        the RB_DEVERR_ARG bit of device_error()."""
        k, T, ks = self._rows(k, "k")
        v, Tv, vs = self._rows(v, "v")
        _require(Tv == T, "k and v must hold the same number of tokens")
        if pos.dtype != torch.int64 or pos.device != self.device or pos.numel() != self.n_seqs or not pos.is_contiguous():
            _require(False, f"pos must be a contiguous int64 [{self.n_seqs}] tensor on {self.device}")
        with _on_device(self.device):
            st = _lib.lib().rb_kv_write(self._ref, k.data_ptr(), v.data_ptr(), ks, vs, T, pos.data_ptr(), config.flags(),
                                        _lib.stream_ptr(self.device))
        _lib.check("rb_kv_write", st)

    def read(self, start, count, out=None):
        """(k, v) of the slots start .. start + count - 1, [n_seqs, n_kv_heads, count, head_dim] in the cache's dtype."""
        if not (0 <= start and 0 <= count and start + count <= self.cache_len):
            _require(False, f"slots {start} .. {start + count - 1} are not in a cache of {self.cache_len}")
        shape = (self.n_seqs, self.n_kv_heads, count, self.head_dim)
        if out is None:
            out = (self._empty.new_empty(shape), self._empty.new_empty(shape))
        else:
            for t in out:
                _require(t.shape == shape and t.dtype == self.dtype and t.device == self.device and t.is_contiguous(),
                         f"out must hold two contiguous {self.dtype} {shape} tensors on {self.device}")
        with _on_device(self.device):
            st = _lib.lib().rb_kv_read(self._ref, out[0].data_ptr(), out[1].data_ptr(), start, count, config.flags(),
                                       _lib.stream_ptr(self.device))
        _lib.check("rb_kv_read", st)
        return out
