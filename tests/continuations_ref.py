"""Plain 64-bit restatements of the operators that decode several continuations of one prompt, for their tests."""
import numpy as np
import torch

F64 = torch.float64


def bf16_of(x):
    """float64 tensor -> the nearest bf16 values (through fp32: a second rounding only matters 2^-15 from a tie)."""
    return x.to(torch.float32).to(torch.bfloat16)


def quantise(x, fmt):
    """Rows x [..., hd] (fp16 or bf16, on the CPU) -> (codes [..., hd] int64, s, m): value = code * s + m, in 64 bits.
    The int4 difference x - m and its product with 1 / 15 are taken in fp32, as the format says (the quotient of the
    codes is then exact enough)."""
    f = x.to(F64)
    if fmt == "int8":
        top = f.abs().amax(-1)
        s = bf16_of(top / 127).to(F64)
        s = torch.where(torch.isfinite(f).all(-1), s, torch.nan)
        c = torch.where((s > 0)[..., None], torch.round(f / torch.where(s > 0, s, 1.0)[..., None]).clamp(-127, 127), 0.0)
        return c.to(torch.int64), s, torch.zeros_like(s)
    lo, hi = f.amin(-1), f.amax(-1)
    rng = (x.float().amax(-1) - x.float().amin(-1))
    s = bf16_of(rng * torch.tensor(1 / 15, dtype=torch.float32)).to(F64)
    s = torch.where(torch.isfinite(f).all(-1) & torch.isfinite(rng), s, torch.nan)
    d = (x.float() - x.float().amin(-1, keepdim=True)).to(F64)
    c = torch.where((s > 0)[..., None], torch.round(d / torch.where(s > 0, s, 1.0)[..., None]).clamp(0, 15), 0.0)
    return c.to(torch.int64), s, lo


def values(x, fmt):
    """What a cache that x was written to stands for, in 64 bits."""
    if fmt == "plain":
        return x.to(F64)
    c, s, m = quantise(x, fmt)
    return c.to(F64) * s[..., None] + m[..., None]


def read_back(x, fmt):
    """The values as rb_kv_read returns them: fp32, clamped to the finite range of x's dtype, rounded once."""
    top = torch.finfo(x.dtype).max
    return values(x, fmt).to(torch.float32).clamp(-top, top).to(x.dtype)


def attention(q, pre, own, own_len, scale, u_p):
    """q [B, nq, hd]; pre (k, v) [nkv, P, hd] or None; own (k, v) [B, nkv, S, hd] or None, values in 64 bits.
    Returns (out, bound): the attention, and the error that a kernel may make before it rounds its output, from
      * 16-bit probabilities (relative rounding u_p, and 2^-25 of the largest one where they are subnormal),
      * fp32 scores: 2 hd 2^-24 of scale * sum |q k| (each score's relative effect on its probability),
      * fp32 sums and the exponential: 2^-19."""
    q = q.to(F64)
    B, nq, hd = q.shape
    nkv = (pre[0] if pre is not None else own[0][0]).shape[0]
    rep = nq // nkv
    out, bound = torch.zeros(B, nq, hd, dtype=F64), torch.zeros(B, nq, hd, dtype=F64)
    for b in range(B):
        for h in range(nq):
            ks, vs = [], []
            if pre is not None:
                ks.append(pre[0][h // rep])
                vs.append(pre[1][h // rep])
            if own is not None:
                ks.append(own[0][b, h // rep, :own_len[b]])
                vs.append(own[1][b, h // rep, :own_len[b]])
            k, v = torch.cat(ks), torch.cat(vs)
            if len(k) == 0:
                continue
            s = (k @ q[b, h]) * scale
            size = float((k.abs() @ q[b, h].abs()).max() * abs(scale)) if len(k) else 0.0
            p = torch.exp(s - s.max())
            l = p.sum()
            out[b, h] = (p @ v) / l
            e_s = 2 * hd * 2.0 ** -24 * size
            bound[b, h] = (p @ v.abs()) / l * (2 * u_p + 2 * e_s + 2.0 ** -19) + len(k) * 2.0 ** -25 * v.abs().amax() / l
    return out, bound


def select(logits, scores, done, end_idx, masked_end=False):
    """(scores, parents, tokens, done, margin): the nb best candidates of each request in 64 bits, ties to the lowest
    (beam, row); margin: the smallest gap between two different neighbours of the order that are not of one beam."""
    x = logits.to(F64).clone()
    R, nb, V = x.shape
    if masked_end:
        x[..., end_idx] = -torch.inf
    bad = torch.isnan(x).any(-1) | (x == torch.inf).any(-1)
    s = scores.to(F64)
    dead = ~torch.isfinite(s)
    lse = torch.logsumexp(torch.where(bad[..., None], 0.0, x), -1, keepdim=True)
    cand = (x - lse) + s[..., None]
    cand = torch.where((bad | dead)[..., None] | torch.isnan(cand), -torch.inf, cand)
    only = torch.full_like(cand, -torch.inf)
    only[..., end_idx] = torch.where(dead, -torch.inf, s)
    cand = torch.where(done[..., None], only, cand).reshape(R, nb * V)
    out = [np.empty((R, nb), dtype=d) for d in (np.float64, np.int64, np.int64, bool)]
    margin = np.inf
    for r in range(R):
        c = cand[r].numpy()
        order = np.lexsort((np.arange(nb * V), -c))[:nb + 1]
        for a, b in zip(order[:-1], order[1:]):
            if c[b] > -np.inf and a // V != b // V:
                margin = min(margin, c[a] - c[b])
        order = order[:nb]
        out[0][r], out[1][r], out[2][r] = c[order], order // V, order % V
        out[3][r] = done[r].numpy()[order // V] | (order % V == end_idx)
    return (*out, margin)


def reorder(t, parents, slots):
    """t [R nb, heads, S, ...] on the CPU -> reordered copy."""
    out = t.clone()
    R, nb = parents.shape
    for r in range(R):
        for c in range(nb):
            b = int(parents[r, c])
            n = int(slots[r * nb + b])
            out[r * nb + c, :, :n] = t[r * nb + b, :, :n]
    return out


def attention_by_weight(q, rows, scale, u_p):
    """attention() over one set of quantised rows (k, v) [nkv, S, hd] for every sequence, with an error bound that a slot
    enters by its weight: 16-bit products p s round by u_p of themselves, and by 2^-25 where they are subnormal - 2^-31 of
    the row's largest product, which is at least 2^6. A product stands for codes whose values, codes times s, are at most the
    size (the largest value plus the range) of its slot's values: 2^-31 of the largest p * size.
    fp32 scores, 2 hd 2^-24 of scale * sum |q k| for each slot; fp32 sums and the exponential, 2^-19."""
    q = q.to(F64)
    B, nq, hd = q.shape
    k, v = rows
    rep = nq // k.shape[0]
    out, bound = torch.zeros(B, nq, hd, dtype=F64), torch.zeros(B, nq, hd, dtype=F64)
    for h in range(nq):
        kh, vh = k[h // rep], v[h // rep]
        s = (q[:, h] @ kh.T) * scale
        e_s = 2 * hd * 2.0 ** -24 * abs(scale) * (q[:, h].abs() @ kh.abs().T)
        p = torch.exp(s - s.amax(-1, keepdim=True))
        l = p.sum(-1, keepdim=True)
        span = vh.abs().amax(-1) + (vh.amax(-1) - vh.amin(-1))
        out[:, h] = (p @ vh) / l
        bound[:, h] = (p @ vh.abs()) / l * (2 * u_p + 2.0 ** -19) + ((p * e_s) @ vh.abs() + (p * e_s).sum(-1, keepdim=True) * out[:, h].abs()) / l
        bound[:, h] += len(kh) * 2.0 ** -31 * (p * span).amax(-1, keepdim=True) / l
    return out, bound
