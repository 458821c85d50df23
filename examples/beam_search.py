"""Beam search over one prompt with an int4 decoder: the prompt's rows are cached once, the beams share them.

    python examples/beam_search.py --fmt int8 --beams 8 --new 32

A small decoder of random int4 weights (RMS norm, rotary positions, grouped-query attention, gated MLP, int8 head)
decodes `--new` tokens for a batch of beams. One step is captured in a CUDA graph:

    BeamSelect       the beams' best continuations over beams x vocabulary
    BeamReorder      every layer's rows of the beams, in place
    gemv_int4_cuda   the projections, one launch for all beams
    KVCache.write    the new token's rows, quantised on the way
    PrefixAttention  the prompt's rows once for the whole batch, and each beam's own

Norms, rotary positions, the MLP's gate and the residual sums are plain torch operations here.
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import rumik_fast_b200 as rb  # noqa: E402
from rumik_fast_b200 import synthetic  # noqa: E402
from rumik_fast_b200.beams import BeamReorder, BeamSelect  # noqa: E402
from rumik_fast_b200.kv_cache import KVCache  # noqa: E402
from rumik_fast_b200.prefix_attention import PrefixAttention  # noqa: E402


def rms_norm(x):
    f = x.float()
    return (f * torch.rsqrt(f.square().mean(-1, keepdim=True) + 1e-6)).to(x.dtype)


class BeamDecoder:
    def __init__(self, layers=4, width=1024, ff=2048, q_heads=8, kv_heads=2, head_dim=128, vocab=16385, beams=8, max_prompt=2048,
                 max_new=64, fmt="int8", end=0, min_new=4, seed=0, device="cuda"):
        device = torch.device(device, torch.cuda.current_device())
        g = synthetic.generator(seed, device)
        self.nq, self.nkv, self.hd, self.nb, self.device = q_heads, kv_heads, head_dim, beams, device
        qkv = (q_heads + 2 * kv_heads) * head_dim
        shapes = {"qkv": (qkv, width), "o": (width, q_heads * head_dim), "gate_up": (2 * ff, width), "down": (width, ff)}
        self.layers = [{n: synthetic.int4_weights(*shape, g, device) for n, shape in shapes.items()} for _ in range(layers)]
        self.embed = torch.randn(vocab, width, generator=g, device=device).half()
        self.head = rb.quantize_int8_rows(torch.randn(vocab, width, generator=g, device=device) * (2 / width ** 0.5), pad_to=1)
        angle = torch.arange(max_prompt + max_new, device=device)[:, None] * 10000.0 ** (-torch.arange(0, head_dim, 2, device=device) / head_dim)
        self.cos, self.sin = angle.cos()[:, None], angle.sin()[:, None]

        # the prompt's rows, once, and the beams' own
        self.prompts = [KVCache(1, kv_heads, max_prompt, head_dim, fmt, device=device) for _ in range(layers)]
        self.own = [KVCache(beams, kv_heads, max_new, head_dim, fmt, device=device) for _ in range(layers)]
        long = dict(dtype=torch.int64, device=device)
        self.n_prompt, self.lens, self.step = torch.zeros(1, **long), torch.zeros(beams, **long), torch.zeros(1, **long)
        self.tokens = torch.zeros(beams, max_new, **long)
        self.scores = torch.zeros(beams, dtype=torch.float32, device=device).view(1, beams)
        self.done = torch.zeros(1, beams, dtype=torch.bool, device=device)
        self.logits = torch.zeros(1, beams, vocab, dtype=torch.float16, device=device)
        self.qkv = torch.empty(beams, qkv, dtype=torch.float16, device=device)
        self.ctx = torch.empty(beams, q_heads * head_dim, dtype=torch.float16, device=device)
        q = self.qkv[:, :q_heads * head_dim].unflatten(1, (q_heads, head_dim))
        self.attend = [PrefixAttention(q, self.ctx.unflatten(1, (q_heads, head_dim)), prefix=p, prefix_len=self.n_prompt, own=o,
                                       own_len=self.lens) for p, o in zip(self.prompts, self.own)]
        self.select = BeamSelect(self.logits, self.scores, self.done, end_idx=end, step=self.step, min_new=min_new)
        self.reorder = BeamReorder([t for c in self.own for t in c.tensors()], self.select.parents, self.lens)
        self.graph = None

    def rotate(self, x, pos):
        """x [T, heads, head_dim], in place, at the positions pos."""
        a, b = x[..., 0::2].float(), x[..., 1::2].float()
        c, s = self.cos[pos], self.sin[pos]
        x[..., 0::2], x[..., 1::2] = (a * c - b * s).to(x.dtype), (a * s + b * c).to(x.dtype)

    def split(self, qkv):
        return qkv.unflatten(-1, (-1, self.hd)).split([self.nq, self.nkv, self.nkv], dim=-2)

    def mlp(self, x, w, product):
        gate, up = product(rms_norm(x), *w["gate_up"]).chunk(2, dim=-1)
        return x + product((torch.nn.functional.silu(gate.float()) * up.float()).to(x.dtype), *w["down"])

    def prefill(self, prompt):
        """Caches the prompt's rows and leaves the last token's logits for the first selection."""
        n = len(prompt)
        at = torch.arange(n, device=self.device)
        later = at[None] > at[:, None]
        x = self.embed[prompt]
        for w, cache in zip(self.layers, self.prompts):
            q, k, v = self.split(rb.mm_int4.mm_int4(rms_norm(x), *w["qkv"]))
            self.rotate(q, at)
            self.rotate(k, at)
            cache.write(k[None], v[None], torch.zeros(1, dtype=torch.int64, device=self.device))
            kk, vv = (t.float().repeat_interleave(self.nq // self.nkv, 1) for t in (k, v))
            s = torch.einsum("ihd,jhd->hij", q.float(), kk) * self.hd ** -0.5
            ctx = torch.einsum("hij,jhd->ihd", s.masked_fill(later, -torch.inf).softmax(-1), vv)
            x = x + rb.mm_int4.mm_int4(ctx.flatten(1).half(), *w["o"])
            x = self.mlp(x, w, rb.mm_int4.mm_int4)
        self.logits.copy_(rb.gemv_int8_cuda(rms_norm(x[-1]), *self.head).expand_as(self.logits))
        self.n_prompt.fill_(n)
        for t in (self.lens, self.step, self.tokens, self.done):
            t.zero_()
        self.scores.fill_(-torch.inf)   # one live beam: the others are its continuations from the first step on
        self.scores[0, 0] = 0

    def decode_step(self):
        best = self.select()
        self.scores.copy_(best["scores"])
        self.done.copy_(best["done"])
        self.reorder()
        new = best["tokens"].view(-1, 1)
        self.tokens.copy_(self.tokens[best["parents"].view(-1)].scatter(1, self.step.expand(self.nb, 1), new))
        x = self.embed[new.view(-1)]
        pos = self.lens.clone()
        self.lens += 1
        for w, own, attend in zip(self.layers, self.own, self.attend):
            rb.gemv_int4_cuda(rms_norm(x), *w["qkv"], out=self.qkv)
            q, k, v = self.split(self.qkv)
            self.rotate(q, self.n_prompt + pos)
            self.rotate(k, self.n_prompt + pos)
            own.write(k, v, pos)
            attend()
            x = x + rb.gemv_int4_cuda(self.ctx, *w["o"])
            x = self.mlp(x, w, rb.gemv_int4_cuda)
        rb.gemv_int8_cuda(rms_norm(x), *self.head, out=self.logits[0])
        self.step += 1

    def generate(self, prompt, new, graph=True):
        """The beams' tokens [beams, new] (a finished beam's go on with the end token) and scores, best first."""
        assert 1 <= new <= self.tokens.shape[1] and 1 <= len(prompt) <= self.prompts[0].cache_len
        if graph and self.graph is None:
            self.prefill(prompt)
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                self.decode_step()      # everything that a first call sets up
            torch.cuda.current_stream().wait_stream(side)
            self.graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(self.graph):
                self.decode_step()
        self.prefill(prompt)
        for _ in range(new):
            self.graph.replay() if graph else self.decode_step()
        return self.tokens[:, :new].clone(), self.scores[0].clone()


def main():
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    ap.add_argument("--fmt", default="int8", choices=["plain", "int8", "int4"])
    ap.add_argument("--beams", type=int, default=8)
    ap.add_argument("--prompt", type=int, default=500)
    ap.add_argument("--new", type=int, default=32)
    a = ap.parse_args()
    decoder = BeamDecoder(beams=a.beams, fmt=a.fmt, max_new=a.new)
    prompt = torch.randint(1, 16385, (a.prompt,), generator=torch.Generator().manual_seed(1)).to(decoder.device)
    decoder.generate(prompt, a.new)
    decoder.prefill(prompt)
    t0, t1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    t0.record()
    for _ in range(a.new):
        decoder.graph.replay()
    t1.record()
    t1.synchronize()
    for tokens, score in zip(decoder.tokens.tolist(), decoder.scores[0].tolist()):
        print(f"{score:9.3f}  {tokens[:12]} ...")
    print(f"{t0.elapsed_time(t1) * 1000 / a.new:.0f} us a step of {a.beams} beams on {a.prompt} prompt rows ({a.fmt} cache)")


if __name__ == "__main__":
    main()
