"""examples/beam_search.py against a plain 64-bit forward of the same weights: every beam's score is the sum of its own
tokens' log-probabilities, which holds only if caches, attention, selection and reordering follow one another.

Tolerance of a score: the example rounds about a dozen values a layer to fp16, each 2^-12 of itself in the mean, so the
hidden state of two layers is off by some sqrt(24) 2^-12 = 1.2e-3, a logit of size 8 by 1e-2, and the sum of six
log-probabilities by 0.06 if all went one way; 0.1."""
import pytest
import torch

from examples.beam_search import BeamDecoder
from oracle import oracle as O
from tests import continuations_ref as ref

pytestmark = pytest.mark.gpu
F64 = torch.float64
END, NEW = 3, 6


def weights(w):
    return torch.from_numpy(O.dequantize_int4(*(t.cpu().numpy() for t in w))).to(F64)


def norm(x):
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6)


def log_probs(d, prompt, tokens, fmt):
    """Log-probabilities of the tokens after the prompt, one sequence, in 64 bits."""
    ids = torch.cat([prompt.cpu(), tokens[:-1]])
    n, P = len(ids), len(prompt)
    x = d.embed.cpu()[ids].to(F64)
    cos, sin = d.cos.cpu()[:n].to(F64), d.sin.cpu()[:n].to(F64)
    rep = d.nq // d.nkv
    for w in d.layers:
        y = (norm(x) @ weights(w["qkv"]).T).unflatten(1, (-1, d.hd))
        a, b = y[..., 0::2], y[..., 1::2]
        turned = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(2)
        q, k, v = turned[:, :d.nq], turned[:, d.nq:d.nq + d.nkv], y[:, d.nq + d.nkv:]
        held = [ref.values(t.half(), fmt).repeat_interleave(rep, 1) for t in (k, v)]
        plain = [t.repeat_interleave(rep, 1) for t in (k, v)]
        ctx = []
        for i in range(n):   # the prompt's rows attend to unquantised ones, the beams' to the cached
            kk, vv = plain if i < P else held
            s = torch.einsum("hd,jhd->hj", q[i], kk[:i + 1]) * d.hd ** -0.5
            ctx.append(torch.einsum("hj,jhd->hd", s.softmax(-1), vv[:i + 1]).flatten())
        x = x + torch.stack(ctx) @ weights(w["o"]).T
        gate, up = (norm(x) @ weights(w["gate_up"]).T).chunk(2, -1)
        x = x + (torch.nn.functional.silu(gate) * up) @ weights(w["down"]).T
    codes, s = (t.cpu() for t in d.head)
    logits = norm(x[P - 1:]) @ ((codes.to(F64) - 128) * s.to(F64)[:, None]).T
    return logits.log_softmax(-1).gather(1, tokens[:, None])[:, 0]


@pytest.mark.parametrize("fmt", ["plain", "int8", "int4"])
def test_scores_are_those_of_the_tokens(native_lib, fmt):
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    import rumik_fast_b200 as rb
    d = BeamDecoder(layers=2, width=256, ff=512, q_heads=4, kv_heads=2, head_dim=64, vocab=509, beams=5, max_prompt=64, max_new=8,
                    fmt=fmt, end=END, min_new=2, seed=4)
    prompt = torch.randint(4, 509, (41,), generator=torch.Generator().manual_seed(2)).to(d.device)
    tokens, scores = d.generate(prompt, NEW, graph=False)
    again, scores_again = d.generate(prompt, NEW)
    assert torch.equal(tokens, again) and torch.equal(scores, scores_again), "the graph's steps differ"
    assert rb.device_error() == 0
    tokens, scores = tokens.cpu(), scores.cpu().to(F64)
    assert (scores[:-1] >= scores[1:]).all() and len({tuple(t) for t in tokens.tolist()}) == 5
    for t, score in zip(tokens, scores):
        ended = (t == END).nonzero()
        n = int(ended[0]) + 1 if len(ended) else NEW
        assert n > 2 and (t[n:] == END).all()
        assert abs(float(log_probs(d, prompt, t[:n], fmt).sum() - score)) < 0.1
