"""A beam search's step on the device (rb_beam_select, rb_beam_reorder).

    select = BeamSelect(logits, scores, done, end_idx=16384, step=step, min_new=8)      # built once
    reorder = BeamReorder([t for c in caches for t in c.tensors()], select.parents, lens)
    best = select()          # {"scores", "parents", "tokens", "done"}: the n_beams best of each request, best first
    reorder()                # every cache: beam b takes over its parent's rows, in place

The search's state stays on the device, so a step can be captured in a CUDA graph. The reference decodes one sequence
with a sampler (engine/sample.py; here sample.FusedSampler) and has no beam search.
"""
import ctypes
import math

import torch

from . import _lib, config
from .cuda_gemv import _on_device, _require


class BeamSelect:
    """logits [R, n_beams, V] (fp16, bf16 or fp32; strided in the first two dimensions as one row stride), scores
    fp32 [R, n_beams] (the beams' summed log-probabilities), done bool [R, n_beams]. A finished beam keeps its score and
    proposes end_idx only. step (int64 [1] on the device) and min_new: end_idx is masked while step < min_new. ids
    (int64 [V]): the token ids of the logits' rows (tokens then holds ids, as FusedSampler's does). The outputs are this
    object's own buffers: scores, parents (the index within the request), tokens, done; a program copies them into its
    inputs before the next call. Exact rules of ties and masked rows: include/rumik_b200.h, rb_beam_select."""

    def __init__(self, logits, scores, done, end_idx, step=None, min_new=0, ids=None):
        _require(logits.is_cuda and logits.dim() == 3, "logits must be a CUDA [R, n_beams, V] tensor")
        R, nb, V = logits.shape
        _require(logits.dtype in (torch.float16, torch.bfloat16, torch.float32), f"logits must be fp16, bf16 or fp32, got {logits.dtype}")
        _require(V == 1 or logits.stride(2) == 1, "logits must have unit stride in their last dimension")
        ld = logits.stride(1) if nb > 1 else (logits.stride(0) if R > 1 else V)
        _require(R <= 1 or logits.stride(0) == nb * ld, "the rows of logits must be evenly spaced")
        dev = logits.device
        for t, nm, dt in ((scores, "scores", torch.float32), (done, "done", torch.bool)):
            _require(t.dtype == dt and t.device == dev and tuple(t.shape) == (R, nb) and t.is_contiguous(),
                     f"{nm} must be a contiguous {dt} [{R}, {nb}] tensor on {dev}")
        for t, nm, n in ((step, "step", 1), (ids, "ids", V)):
            _require(t is None or (t.dtype == torch.int64 and t.device == dev and t.numel() == n and t.is_contiguous()),
                     f"{nm} must be a contiguous int64 [{n}] tensor on {dev}")
        _require(1 <= nb <= 32, f"1 to 32 beams are supported, got {nb}")
        _require(0 <= end_idx < V, f"end_idx {end_idx} is no row of {V}")
        self.device = dev
        self.scores = torch.empty(R, nb, dtype=torch.float32, device=dev)
        self.parents = torch.empty(R, nb, dtype=torch.int64, device=dev)
        self.tokens = torch.empty(R, nb, dtype=torch.int64, device=dev)
        self.done = torch.empty(R, nb, dtype=torch.bool, device=dev)
        self._keep = (logits, scores, done, step, ids)
        with _on_device(dev):
            need = _lib.lib().rb_beam_select_workspace(R, nb, V)
        if need < 0:
            _lib.check("rb_beam_select_workspace", -need)
        self.ws = torch.zeros(need, dtype=torch.uint8, device=dev)
        self._args = _lib.BeamSelectArgs(
            logits.data_ptr(), _lib.dtype_code(logits.dtype), ld, R, nb, V, end_idx, scores.data_ptr(), done.data_ptr(),
            None if ids is None else ids.data_ptr(), None if step is None else step.data_ptr(), min_new,
            self.scores.data_ptr(), self.parents.data_ptr(), self.tokens.data_ptr(), self.done.data_ptr(),
            self.ws.data_ptr(), need)
        self._ref = ctypes.byref(self._args)

    def __call__(self):
        with _on_device(self.device):
            st = _lib.lib().rb_beam_select(self._ref, config.flags(), _lib.stream_ptr(self.device))
        _lib.check("rb_beam_select", st)
        return {"scores": self.scores, "parents": self.parents, "tokens": self.tokens, "done": self.done}


class BeamReorder:
    """tensors: contiguous CUDA tensors [R * n_beams, n_heads, cache_len, ...] that share cache_len (caches, their row
    parameters; KVCache.tensors()); parents int64 [R, n_beams] and slots int64 [R * n_beams] on the device, slots the
    beams' lengths before the reordering. Beam b's slots [0, slots[parent]) become its parent's, in place, one launch a
    hundred tensors. Slots beyond that keep what they hold."""

    def __init__(self, tensors, parents, slots):
        _require(len(tensors) > 0, "empty tensor list")
        dev = tensors[0].device
        _require(parents.dim() == 2 and parents.dtype == torch.int64 and parents.device == dev and parents.is_contiguous(),
                 f"parents must be a contiguous int64 [R, n_beams] tensor on {dev}")
        R, nb = parents.shape
        _require(1 <= nb <= 32, f"1 to 32 beams are supported, got {nb}")
        _require(slots.dtype == torch.int64 and slots.device == dev and slots.numel() == R * nb and slots.is_contiguous(),
                 f"slots must be a contiguous int64 [{R * nb}] tensor on {dev}")
        arr = (_lib.BeamTensor * len(tensors))()
        S = tensors[0].shape[2] if tensors[0].dim() >= 3 else 0
        for i, t in enumerate(tensors):
            _require(t.is_cuda and t.device == dev and t.is_contiguous() and t.dim() >= 3 and t.shape[0] == R * nb
                     and t.shape[2] == S, f"tensor {i} must be a contiguous [{R * nb}, n_heads, {S}, ...] tensor on {dev}")
            row = t.element_size() * math.prod(t.shape[3:])
            _require(row % 2 == 0, f"tensor {i}: rows of {row} bytes (an even number is needed)")
            arr[i] = _lib.BeamTensor(t.data_ptr(), t.shape[1], row)
        self.device, self._keep = dev, (list(tensors), parents, slots)
        self._call = (arr, len(tensors), R, nb, S, parents.data_ptr(), slots.data_ptr())

    def __call__(self):
        with _on_device(self.device):
            st = _lib.lib().rb_beam_reorder(*self._call, config.flags(), _lib.stream_ptr(self.device))
        _lib.check("rb_beam_reorder", st)
