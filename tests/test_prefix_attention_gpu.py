"""Attention of a batch over a shared prefix and rows of its own (rb_prefix_attn) against softmax(q k) v in 64 bits on
the values that the caches stand for. The bound of each output is derived from the inputs (continuations_ref.attention:
16-bit probabilities, fp32 scores and sums) plus half a unit of the output's own rounding."""
import pytest
import torch

import rumik_fast_b200 as rb
from rumik_fast_b200.kv_cache import KVCache
from rumik_fast_b200.prefix_attention import PrefixAttention
from tests import continuations_ref as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module", autouse=True)
def _gpu(native_lib):
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    rb.device_error()
    yield
    assert rb.device_error() == 0


def rows(shape, dtype, seed, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g) * spread
    x[..., ::16] *= 3
    return x.to(dtype)


class Setup:
    """Caches of a random prefix and random own rows (with NaN rows beyond every length), and the attention over them."""

    def __init__(self, B, nq, nkv, hd, P, lens, fmt, dtype, seed=0, spread=1.0, slack=3, kernel=None):
        dt = DTYPES[dtype]
        self.B, self.fmt, self.dt, self.lens, self.scale = B, fmt, dt, lens, hd ** -0.5
        self.q = rows((B, nq, hd), dt, seed, spread)
        self.out = torch.full((B, nq, hd), float("nan"), dtype=dt, device=DEV)
        self.pre = self.own = self.pre_vals = self.own_vals = None
        nan = float("nan")
        kw = {}
        if P is not None:
            k, v = rows((1, P, nkv, hd), dt, seed + 1, spread), rows((1, P, nkv, hd), dt, seed + 2)
            self.pre = KVCache(1, nkv, P + slack, hd, fmt, dt)
            self.fill(self.pre, nan)
            self.pre.write(k.to(DEV), v.to(DEV), torch.zeros(1, dtype=torch.int64, device=DEV))
            self.pre_vals = tuple(ref.values(x[0], fmt).transpose(0, 1) for x in (k, v))
            self.prefix_len = torch.tensor([P], device=DEV)
            kw.update(prefix=self.pre, prefix_len=self.prefix_len)
        if lens is not None:
            S = max(lens) + slack
            k, v = rows((B, S, nkv, hd), dt, seed + 3, spread), rows((B, S, nkv, hd), dt, seed + 4)
            for b, n in enumerate(lens):
                k[b, n:], v[b, n:] = nan, nan
            self.own = KVCache(B, nkv, S, hd, fmt, dt)
            self.own.write(k.to(DEV), v.to(DEV), torch.zeros(B, dtype=torch.int64, device=DEV))
            self.own_vals = tuple(ref.values(x, fmt).transpose(1, 2) for x in (k, v))
            self.own_len = torch.tensor(lens, device=DEV)
            kw.update(own=self.own, own_len=self.own_len)
        self.attn = PrefixAttention(self.q.to(DEV), self.out, kernel=kernel, **kw)

    @staticmethod
    def fill(cache, value):
        x = torch.full((cache.n_seqs, cache.cache_len, cache.n_kv_heads, cache.head_dim), value, dtype=cache.dtype, device=DEV)
        cache.write(x, x, torch.zeros(cache.n_seqs, dtype=torch.int64, device=DEV))

    def check(self, got=None, P=None, lens=None):
        got = (self.out if got is None else got).cpu()
        lens = self.lens if lens is None else lens
        pre = self.pre_vals if P is None or self.pre_vals is None else tuple(x[:, :P] for x in self.pre_vals)
        # bf16 rows kept as they are multiply with bf16 probabilities, everything else with fp16 ones
        u_p = 2.0 ** -8 if self.fmt == "plain" and self.dt == torch.bfloat16 else 2.0 ** -11
        want, bound = ref.attention(self.q, pre, self.own_vals, lens, self.scale, u_p)
        half = 2.0 ** -8 if self.dt == torch.bfloat16 else 2.0 ** -11
        off = (got.double() - want).abs()
        over = off - (want.abs() * half * (1 + 2 ** -7) + bound * (1 + half) + 2.0 ** -25)
        assert torch.isfinite(got).all() and (over <= 0).all(), f"largest error {off.max():.3g}, over its bound by {over.max():.3g}"


@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("fmt", ["plain", "int8", "int4"])
@pytest.mark.parametrize("B,nq,nkv,hd,P,lens", [
    (1, 1, 1, 64, 1, [0]),
    (1, 2, 2, 128, 0, [1]),
    (2, 6, 2, 128, 17, [0, 5]),
    (4, 24, 8, 128, 301, [9, 1, 0, 7]),
    (3, 32, 4, 64, 130, [64, 65, 63]),
    (5, 16, 1, 128, 64, [3, 0, 33, 16, 31]),
    (16, 12, 4, 128, 1000, [i * 5 % 23 for i in range(16)]),
    (33, 8, 2, 64, 515, [i * 7 % 40 for i in range(33)]),
    (64, 4, 1, 128, 700, [i % 3 for i in range(64)]),
    (2, 4, 4, 128, 4097, [129, 2]),
])
def test_against_64_bits(B, nq, nkv, hd, P, lens, fmt, dtype):
    s = Setup(B, nq, nkv, hd, P, lens, fmt, dtype, seed=B + P)
    s.attn()
    s.check()
    first = s.out.clone()
    s.attn()     # the workspace is as the call found it, and the order of additions does not depend on timing
    assert torch.equal(first, s.out)


@pytest.mark.parametrize("fmt", ["plain", "int8", "int4"])
def test_only_a_prefix_and_only_own_rows(fmt):
    s = Setup(7, 12, 4, 128, 333, None, fmt, "fp16", seed=5)
    s.attn()
    s.check()
    s = Setup(7, 12, 4, 128, None, [100, 0, 1, 64, 257, 31, 32], fmt, "bf16", seed=6)
    s.attn()
    s.check()
    assert not s.out[1].any()    # no slot at all: zeros


@pytest.mark.parametrize("fmt", ["plain", "int8", "int4"])
def test_no_slot_at_all(fmt):
    s = Setup(3, 4, 2, 64, 5, [2, 0, 1], fmt, "fp16", seed=7)
    s.prefix_len.zero_()
    s.attn()
    assert not s.out[1].any()
    s.check(P=0)


@pytest.mark.parametrize("fmt", ["plain", "int8", "int4"])
@pytest.mark.parametrize("dtype", sorted(DTYPES))
def test_peaked_and_flat_scores(fmt, dtype):
    """Scores spread over hundreds (one slot takes it all, most probabilities underflow), and scores that are all equal."""
    s = Setup(3, 6, 2, 128, 600, [40, 0, 77], fmt, dtype, seed=8, spread=6.0)
    s.attn()
    s.check()
    s = Setup(3, 6, 2, 128, 600, [40, 0, 77], fmt, dtype, seed=9)
    s.q.zero_()
    s.attn._keep[0].zero_()
    s.attn()
    s.check()


@pytest.mark.parametrize("fmt", ["int8", "int4"])
@pytest.mark.parametrize("size", [2.0 ** -14, 300.0])
def test_scales_of_any_size(fmt, size):
    """Values (and so their scales) far below and above one, and rows whose scales differ by orders of magnitude."""
    s = Setup(2, 4, 2, 128, 0, [70, 33], fmt, "bf16", seed=10)
    k, v = rows((2, 70, 2, 128), torch.bfloat16, 1), rows((2, 70, 2, 128), torch.bfloat16, 2)
    v = (v.float() * size * torch.logspace(-3, 0, 70)[None, :, None, None]).to(torch.bfloat16)
    s.own.write(k.to(DEV), v.to(DEV), torch.zeros(2, dtype=torch.int64, device=DEV))
    s.own_vals = tuple(ref.values(x, fmt).transpose(1, 2) for x in (k, v))
    s.attn()
    s.check()


@pytest.mark.parametrize("dtype", sorted(DTYPES))
def test_large_and_tiny_queries(dtype):
    """Queries near fp16's largest value and far below its smallest normal one, over quantised keys."""
    for size in (2.0 ** -20, 2000.0):
        s = Setup(2, 6, 2, 128, 90, [3, 9], "int8", dtype, seed=11)
        s.q = (s.q.float() * size).to(s.dt)
        s.attn._keep[0].copy_(s.q)
        s.scale = 0.05 / size
        kw = dict(prefix=s.pre, prefix_len=s.prefix_len, own=s.own, own_len=s.own_len)
        PrefixAttention(s.attn._keep[0], s.out, scale=s.scale, **kw)()
        s.check()


def test_rows_of_zeros_and_of_one_value():
    """Quantised rows with a zero scale among ordinary ones."""
    for fmt in ("int8", "int4"):
        s = Setup(1, 2, 1, 64, 0, [40], fmt, "fp16", seed=12)
        k, v = rows((1, 40, 1, 64), torch.float16, 1), rows((1, 40, 1, 64), torch.float16, 2)
        k[:, ::3], v[:, ::2], v[:, 5], k[:, 7] = 0, 0, 1.5, -2.0
        s.own.write(k.to(DEV), v.to(DEV), torch.zeros(1, dtype=torch.int64, device=DEV))
        s.own_vals = tuple(ref.values(x, fmt).transpose(1, 2) for x in (k, v))
        s.attn()
        s.check()
        v.zero_()     # nothing but zeros
        s.own.write(k.to(DEV), v.to(DEV), torch.zeros(1, dtype=torch.int64, device=DEV))
        s.attn()
        assert not s.out.any()


@pytest.mark.parametrize("fmt", ["plain", "int8", "int4"])
def test_a_nan_in_a_visible_row_shows(fmt):
    """A NaN in a value row reaches the sequences that see it and no other."""
    s = Setup(3, 4, 2, 64, 20, [9, 4, 0], fmt, "fp16", seed=13)
    x = rows((3, 1, 2, 64), torch.float16, 1)
    bad = x.clone()
    bad[0, 0, 1, 3] = float("nan")
    bad[1:] = float("nan")
    s.own.write(x.to(DEV), bad.to(DEV), torch.tensor([2, 5, 0], device=DEV))   # 1 and 2: beyond their lengths
    s.attn()
    assert torch.isnan(s.out[0, 2:]).any() and torch.isfinite(s.out[0, :2]).all() and torch.isfinite(s.out[1:]).all()


@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("fmt", ["plain", "int8", "int4"])
@pytest.mark.parametrize("B,nq,nkv,hd,P,lens", [
    (1, 1, 1, 64, 1, None),
    (1, 2, 2, 128, 127, [3]),
    (5, 16, 4, 128, 128, [0, 1, 2, 3, 4]),
    (11, 12, 4, 64, 129, None),
    (16, 48, 8, 128, 300, [i * 5 % 23 for i in range(16)]),
    (43, 6, 2, 128, 1000, None),
    (64, 16, 2, 64, 2500, [i % 3 for i in range(64)]),
    (150, 2, 1, 128, 6000, None),
    (100, 12, 4, 64, 12000, None),      # three row tiles of four heads: splits of many tiles
])
def test_tcgen05_kernel_against_64_bits(B, nq, nkv, hd, P, lens, fmt, dtype):
    """The tcgen05 kernel at sizes that the choice by rows would leave to the warp-level one as well: single rows and
    tiles, tiles that end inside, several row tiles, one and many splits."""
    s = Setup(B, nq, nkv, hd, P, lens, fmt, dtype, seed=B + P, kernel="tc")
    s.attn()
    assert rb.device_error() == 0
    s.check()
    first = s.out.clone()
    s.attn()
    assert torch.equal(first, s.out)


@pytest.mark.parametrize("fmt", ["plain", "int8", "int4"])
@pytest.mark.parametrize("dtype", sorted(DTYPES))
def test_tcgen05_kernel_peaked_flat_and_rising_scores(fmt, dtype):
    """Scores spread over hundreds, all equal, and rising along the prefix (the references are raised again and again)."""
    s = Setup(20, 6, 2, 128, 1500, [i % 5 for i in range(20)], fmt, dtype, seed=8, spread=6.0, kernel="tc")
    s.attn()
    s.check()
    s.q.zero_()
    s.attn._keep[0].zero_()
    s.attn()
    s.check()
    k = rows((1, 1500, 2, 128), s.dt, 1)
    k = (k.float() * torch.linspace(0, 12, 1500)[None, :, None, None]).to(s.dt)
    v = rows((1, 1500, 2, 128), s.dt, 2)
    s.pre.write(k.to(DEV), v.to(DEV), torch.zeros(1, dtype=torch.int64, device=DEV))
    s.pre_vals = tuple(ref.values(x[0], fmt).transpose(0, 1) for x in (k, v))
    s.q = rows((20, 6, 128), s.dt, 3)
    s.attn._keep[0].copy_(s.q)
    s.attn()
    s.check()


def test_tcgen05_kernel_lengths_and_nan():
    """Lengths that change under one object, none, out of range, and a NaN among the prefix's values."""
    for fmt in ("plain", "int8", "int4"):
        s = Setup(12, 8, 2, 128, 700, [i for i in range(12)], fmt, "fp16", seed=20, kernel="tc")
        for P in (700, 1, 300, 0):
            s.prefix_len.fill_(P)
            s.attn()
            s.check(P=P)
        s.out.fill_(7)
        s.prefix_len.fill_(704)
        s.attn()
        assert rb.device_error() == rb._lib.DEVERR_ARG and (s.out == 7).all()
        s.prefix_len.fill_(700)
        bad = torch.full((1, 1, 2, 128), float("nan"), dtype=torch.float16, device=DEV)
        s.pre.write(bad, bad, torch.tensor([650], device=DEV))
        s.attn()
        assert torch.isnan(s.out).all()
        s.prefix_len.fill_(650)
        s.attn()
        s.check(P=650)


def test_tcgen05_kernel_negative_and_zero_scale():
    for scale in (-0.1, 0.0):
        for fmt in ("plain", "int8", "int4"):
            for kernel in ("tc", "mma"):
                s = Setup(12, 8, 2, 64, 300, [i for i in range(12)], fmt, "bf16", seed=21)
                s.scale = scale
                PrefixAttention(s.attn._keep[0], s.out, prefix=s.pre, prefix_len=s.prefix_len, own=s.own, own_len=s.own_len,
                                scale=scale, kernel=kernel)()
                s.check()


def test_strided_queries_and_outputs():
    B, nq, nkv, hd = 5, 6, 2, 128
    s = Setup(B, nq, nkv, hd, 100, [3, 1, 0, 8, 2], "int8", "fp16", seed=14)
    fused = torch.zeros(B, (nq + 2 * nkv) * hd, dtype=torch.float16, device=DEV)
    fused[:, :nq * hd] = s.q.to(DEV).flatten(1)
    wide = torch.full((B, nq * hd + 64), 7.0, dtype=torch.float16, device=DEV)
    out = wide[:, :nq * hd].view(B, nq, hd)
    PrefixAttention(fused[:, :nq * hd].view(B, nq, hd), out, prefix=s.pre, prefix_len=s.prefix_len, own=s.own, own_len=s.own_len)()
    s.check(out)
    assert (wide[:, nq * hd:] == 7).all()


def test_lengths_outside_the_caches():
    s = Setup(4, 4, 2, 64, 30, [5, 2, 9, 1], "int8", "fp16", seed=15)
    s.own_len.copy_(torch.tensor([5, 13, -1, 1]))
    s.out.fill_(7)
    s.attn()
    assert rb.device_error() == rb._lib.DEVERR_ARG
    assert (s.out[1:3] == 7).all()          # nothing is stored for them
    got = s.out.clone()
    s.own_len.copy_(torch.tensor([5, 2, 9, 1]))
    s.attn()
    s.check()
    assert torch.equal(got[::3], s.out[::3])
    for bad in (-1, 34):
        s.prefix_len.fill_(bad)
        s.out.fill_(7)
        s.attn()
        assert rb.device_error() == rb._lib.DEVERR_ARG and (s.out == 7).all()
    s.prefix_len.fill_(30)
    s.attn()
    s.check()


@pytest.mark.parametrize("fmt", ["plain", "int4"])
def test_one_graph_for_every_length(fmt):
    s = Setup(6, 8, 2, 128, 900, [50, 3, 77, 0, 12, 31], fmt, "fp16", seed=16)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        s.attn()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            s.attn()
        for P, cut in ((900, 0), (1, 2), (513, 40), (0, 5)):
            lens = [max(0, n - cut) for n in s.lens]
            s.prefix_len.fill_(P)
            s.own_len.copy_(torch.tensor(lens))
            g.replay()
            side.synchronize()
            s.check(P=P, lens=lens)


def test_offsets_beyond_32_bits():
    """A 16-bit prefix of more than 2^32 bytes: its last slots decide (their keys are the queries)."""
    nkv, S, hd = 2, (1 << 23) + 77, 128          # 4.3 GB a side
    prefix = KVCache(1, nkv, S, hd, "plain")
    q = rows((2, nkv, hd), torch.float16, 17)
    k = torch.zeros(1, 2, nkv, hd, dtype=torch.float16)
    k[0] = q * 8
    v = rows((1, 2, nkv, hd), torch.float16, 18)
    prefix.write(k.to(DEV), v.to(DEV), torch.tensor([S - 2], device=DEV))
    out = torch.empty(2, nkv, hd, dtype=torch.float16, device=DEV)
    PrefixAttention(q.to(DEV), out, prefix=prefix, prefix_len=torch.tensor([S], device=DEV))()
    # the zero keys' S - 2 slots weigh exp(-score) each, and their values are zero
    score = torch.einsum("bhd,thd->bht", q.double(), k[0].double()) * hd ** -0.5
    p = torch.exp(score - score.amax(-1, keepdim=True))
    total = p.sum(-1, keepdim=True) + (S - 2) * torch.exp(-score.amax(-1, keepdim=True))
    want = torch.einsum("bht,thd->bhd", p / total, v[0].double())
    assert (out.cpu().double() - want).abs().max() <= 2.0 ** -9 * want.abs().max()


def test_refusals():
    q = torch.zeros(2, 4, 64, dtype=torch.float16, device=DEV)
    one = torch.ones(1, dtype=torch.int64, device=DEV)
    two = torch.ones(2, dtype=torch.int64, device=DEV)
    pre, own = KVCache(1, 2, 8, 64, "int8"), KVCache(2, 2, 8, 64, "int8")
    ok = dict(prefix=pre, prefix_len=one, own=own, own_len=two)
    PrefixAttention(q, torch.empty_like(q), **ok)
    for change in (dict(prefix=None, own=None), dict(prefix=own), dict(own=pre), dict(prefix_len=None), dict(own_len=one),
                   dict(own_len=two.int()), dict(prefix=KVCache(1, 2, 8, 64, "int4")), dict(prefix=KVCache(1, 4, 8, 64, "int8")),
                   dict(prefix=KVCache(1, 2, 8, 64, "int8", torch.bfloat16)), dict(prefix=None)):
        with pytest.raises(RuntimeError):
            PrefixAttention(q, torch.empty_like(q), **{**ok, **change})
    for bad in (q[:, :3], q[..., :32], q.bfloat16(), q.transpose(0, 1), q.cpu(), q.flatten(1)):
        with pytest.raises(RuntimeError):
            PrefixAttention(bad, torch.empty_like(q), **ok)
    wide = torch.zeros(2, 34, 64, dtype=torch.float16, device=DEV)
    with pytest.raises(RuntimeError):      # seventeen query heads a key-value head
        PrefixAttention(wide, torch.empty_like(wide), **ok)


@pytest.mark.parametrize("kernel", ["mma", "tc"])
@pytest.mark.parametrize("fmt", ["plain", "int8", "int4"])
@pytest.mark.parametrize("pre_slots,own_slots", [(0, None), (None, 0), (0, 0), (0, 40), (300, 0)])
def test_caches_without_a_slot(pre_slots, own_slots, fmt, kernel):
    """Caches of no slots alone, together and beside one with rows, over a workspace that holds anything: zeros where there
    is nothing to attend to, and a length above zero is one outside its cache."""
    B, nkv, hd = 3, 2, 64
    q = rows((B, 4, hd), torch.float16, 41)
    out = torch.full((B, 4, hd), 7.0, dtype=torch.float16, device=DEV)
    kw, vals = {}, {}
    for nm, n, slots in (("prefix", 1, pre_slots), ("own", B, own_slots)):
        if slots is None:
            continue
        full = KVCache(n, nkv, max(slots, 1), hd, fmt)
        if slots:
            k, v = rows((n, slots, nkv, hd), torch.float16, 42), rows((n, slots, nkv, hd), torch.float16, 43)
            full.write(k.to(DEV), v.to(DEV), torch.zeros(n, dtype=torch.int64, device=DEV))
            vals[nm] = tuple(ref.values(x, fmt).transpose(1, 2) for x in (k, v))
        else:
            full = KVCache.wrap(*(t if t is None else t[:, :, :0].contiguous() for t in (full.k, full.v, full.k_par, full.v_par)), dtype=full.dtype)
        kw[nm], kw[nm + "_len"] = full, torch.full((n,), slots, dtype=torch.int64, device=DEV)
    attn = PrefixAttention(q.to(DEV), out, kernel=kernel, **kw)
    attn.ws.fill_(1)
    attn()
    assert rb.device_error() == 0
    if vals:
        pre = tuple(x[0] for x in vals["prefix"]) if "prefix" in vals else None
        want, bound = ref.attention(q, pre, vals.get("own"), [own_slots] * B, hd ** -0.5, 2.0 ** -11)
        assert ((out.cpu().double() - want).abs() <= want.abs() * 2.0 ** -11 * (1 + 2 ** -7) + bound * (1 + 2.0 ** -11) + 2.0 ** -25).all()
    else:
        assert not out.any()
    if pre_slots == 0:
        kw["prefix_len"].fill_(1)
        out.fill_(7)
        attn()
        assert rb.device_error() == rb._lib.DEVERR_ARG and (out == 7).all()
        kw["prefix_len"].zero_()
    if own_slots == 0:
        kw["own_len"][1] = 1
        out.fill_(7)
        attn()
        assert rb.device_error() == rb._lib.DEVERR_ARG and (out[1] == 7).all() and not (out[0] == 7).any() and not (out[2] == 7).any()


@pytest.mark.parametrize("kernel", ["mma", "tc"])
@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("fmt", ["plain", "int8", "int4"])
@pytest.mark.parametrize("scale", [0.0, 1e-20, -1e-30])
def test_no_scale_and_no_query(fmt, dtype, kernel, scale):
    """A scale of zero, or next to it, over query rows of zeros: every visible slot weighs the same."""
    s = Setup(5, 8, 2, 64, 300, [3, 0, 1, 70, 2], fmt, dtype, seed=31)
    s.q[:, ::2] = 0
    s.attn._keep[0].copy_(s.q)
    s.scale = scale
    PrefixAttention(s.attn._keep[0], s.out, prefix=s.pre, prefix_len=s.prefix_len, own=s.own, own_len=s.own_len, scale=scale,
                    kernel=kernel)()
    s.check()


def slot_without_weight(B, nq, nkv, hd, S, fmt, dtype, spread, out_at, ratio, seed, size=1.0):
    """q, k, v whose slot out_at has values 2^ratio times the others' and a score a hundred below every other one."""
    dt = DTYPES[dtype]
    g = torch.Generator().manual_seed(seed)
    base = torch.randn(nkv, hd, generator=g)
    q = base.repeat_interleave(nq // nkv, 0) + 0.1 * torch.randn(B, nq, hd, generator=g)
    k = spread * torch.randn(1, S, nkv, hd, generator=g)
    v = torch.randn(1, S, nkv, hd, generator=g) * size
    k[0, out_at] = -100 * hd ** 0.5 * base / base.square().sum(-1, keepdim=True)
    v[0, out_at] *= 2.0 ** ratio
    return q.to(dt), k.to(dt), v.to(dt)


def check_by_weight(out, q, k, v, fmt, dtype):
    want, bound = ref.attention_by_weight(q, tuple(ref.values(x[0], fmt).transpose(0, 1) for x in (k, v)), q.shape[2] ** -0.5, 2.0 ** -11)
    half = 2.0 ** -8 if dtype == "bf16" else 2.0 ** -11
    got = out.cpu()
    off = (got.double() - want).abs()
    over = off - (want.abs() * half * (1 + 2 ** -7) + bound * (1 + half) + 2.0 ** -25 * (dtype == "fp16"))
    assert torch.isfinite(got).all() and (over <= 0).all(), f"largest error {off.max():.3g}, over its bound by {over.max():.3g}"


@pytest.mark.parametrize("kernel", ["mma", "tc"])
@pytest.mark.parametrize("fmt", ["int8", "int4"])
@pytest.mark.parametrize("dtype,ratio,size", [("fp16", 9, 1.0), ("fp16", 20, 2.0 ** -9), ("bf16", 16, 1.0), ("bf16", 24, 1.0), ("bf16", 100, 1.0)])
@pytest.mark.parametrize("S,out_at", [(200, 0), (200, 150), (4000, 37), (4000, 3900)])
def test_a_large_row_without_weight(S, out_at, dtype, ratio, size, fmt, kernel):
    """One visible slot whose values, and so whose scale, are far larger than the others' but whose probability is next to
    nothing: the others keep their accuracy, which is bounded by their own weights and values. (8 heads of 16 sequences:
    few splits, so that most slots share a partial with that one.)"""
    q, k, v = slot_without_weight(16, 64, 8, 64, S, fmt, dtype, 1.0, out_at, ratio, seed=S + out_at, size=size)
    cache = KVCache(1, 8, S, 64, fmt, DTYPES[dtype])
    cache.write(k.to(DEV), v.to(DEV), torch.zeros(1, dtype=torch.int64, device=DEV))
    out = torch.empty(q.shape, dtype=q.dtype, device=DEV)
    PrefixAttention(q.to(DEV), out, prefix=cache, prefix_len=torch.tensor([S], device=DEV), kernel=kernel)()
    check_by_weight(out, q, k, v, fmt, dtype)


@pytest.mark.parametrize("fmt", ["int8", "int4"])
@pytest.mark.parametrize("dtype", sorted(DTYPES))
def test_a_flat_tail_beside_a_large_row_without_weight(fmt, dtype):
    """Own rows, one split each: a slot without values holds most of the weight, thousands hold 2^-18 to 2^-20 of it each,
    and the values of one without weight are 2^9 times larger. The tail's sum is the output."""
    B, nkv, S, hd = 40, 8, 4000, 128
    q, k, v = slot_without_weight(B, nkv, nkv, hd, S, fmt, dtype, 0.05, 77, 9, seed=3, size=0.25)
    top = q.float().mean(0)
    k[0, 1234] = (13.2 * hd ** 0.5 * top / top.square().sum(-1, keepdim=True)).to(k.dtype)
    v[0, 1234] = 0
    own = KVCache(B, nkv, S, hd, fmt, DTYPES[dtype])
    own.write(k.to(DEV).expand(B, -1, -1, -1), v.to(DEV).expand(B, -1, -1, -1), torch.zeros(B, dtype=torch.int64, device=DEV))
    out = torch.empty(q.shape, dtype=q.dtype, device=DEV)
    PrefixAttention(q.to(DEV), out, own=own, own_len=torch.full((B,), S, device=DEV))()
    check_by_weight(out, q, k, v, fmt, dtype)


@pytest.mark.parametrize("kernel", ["mma", "tc"])
@pytest.mark.parametrize("fmt", ["int8", "int4"])
@pytest.mark.parametrize("lo,hi", [(0, 0), (-100, -60), (-100, 100), (40, 112), (112, 112)])
def test_values_over_the_whole_range_of_bf16(lo, hi, fmt, kernel):
    """Values from 2^lo to 2^hi, and rows of zeros among them, in ascending, descending and mixed order."""
    S = 700
    g = torch.Generator().manual_seed(5)
    q, k, v = torch.randn(3, 8, 128, generator=g), torch.randn(1, S, 2, 128, generator=g) * 0.3, torch.randn(1, S, 2, 128, generator=g)
    size = torch.linspace(lo, hi, S, dtype=torch.float64)
    for order in (torch.arange(S), torch.arange(S).flip(0), torch.randperm(S, generator=g)):
        w = (v.clamp(-3, 3).double() * 2.0 ** size[order][None, :, None, None])
        w[:, ::5] = 0
        qq, kk, vv = q.bfloat16(), k.bfloat16(), w.float().bfloat16()
        cache = KVCache(1, 2, S, 128, fmt, torch.bfloat16)
        cache.write(kk.to(DEV), vv.to(DEV), torch.zeros(1, dtype=torch.int64, device=DEV))
        out = torch.empty(3, 8, 128, dtype=torch.bfloat16, device=DEV)
        PrefixAttention(qq.to(DEV), out, prefix=cache, prefix_len=torch.tensor([S], device=DEV), kernel=kernel)()
        check_by_weight(out, qq, kk, vv, fmt, "bf16")


@pytest.mark.parametrize("fmt,hd,heads,rep,S,kernel", [
    ("int8", 64, 16, 1, 20000, "mma"), ("int4", 128, 16, 2, 20000, "mma"), ("plain", 64, 16, 1, 20000, "mma"),   # few rows, all SMs busy
    ("int8", 128, 2, 1, 3000, "mma"),
    ("int8", 64, 2, 1, 10000, "tc"), ("int4", 128, 2, 1, 20000, "tc"), ("plain", 128, 16, 1, 20000, "tc"), ("int8", 64, 16, 8, 20000, "tc"),
    ("plain", 128, 2, 1, 1500, "mma"), ("int8", 128, 2, 16, 1500, "tc"),
])
def test_choice_of_the_kernel(fmt, hd, heads, rep, S, kernel):
    """Without a word about the kernel the one that was measured faster runs: its bits, where the two kernels' differ."""
    B = 4
    g = torch.Generator(device=DEV).manual_seed(7)
    cache = KVCache(1, heads, S, hd, fmt)
    x = torch.randn(2, 1, S, heads, hd, generator=g, device=DEV).half()
    cache.write(x[0], x[1], torch.zeros(1, dtype=torch.int64, device=DEV))
    q = torch.randn(B, heads * rep, hd, generator=g, device=DEV).half()
    got = {}
    for k in (None, "mma", "tc"):
        got[k] = torch.empty_like(q)
        PrefixAttention(q, got[k], prefix=cache, prefix_len=torch.tensor([S], device=DEV), kernel=k)()
    assert not torch.equal(got["mma"], got["tc"]) and torch.equal(got[None], got[kernel])


@pytest.mark.parametrize("kernel", ["mma", "tc"])
@pytest.mark.parametrize("fmt", ["plain", "int8", "int4"])
@pytest.mark.parametrize("scale", [3.3e38, -3.3e38])
def test_largest_scale_and_no_query(fmt, kernel, scale):
    """Scales whose product with log2 e is no fp32 number any more, over queries of zeros: scores of zero."""
    for dtype in sorted(DTYPES):
        s = Setup(5, 8, 2, 64, 300, [3, 0, 1, 70, 2], fmt, dtype, seed=32)
        s.q.zero_()
        s.attn._keep[0].zero_()
        s.scale = scale
        PrefixAttention(s.attn._keep[0], s.out, prefix=s.pre, prefix_len=s.prefix_len, own=s.own, own_len=s.own_len, scale=scale,
                        kernel=kernel)()
        s.check()


@pytest.mark.parametrize("fmt", ["plain", "int8", "int4"])
def test_tcgen05_kernel_with_the_shortest_wait_limit(fmt):
    """With a limit of a microsecond, waits on products that are under way run out. The kernel ends them before it gives its
    memory back: it reports the wait or, where none ran out, the right output, and the next call is as ever."""
    s = Setup(40, 6, 2, 128, 9000, None, fmt, "fp16", seed=51, kernel="tc")
    for _ in range(3):
        rb._lib.set_wait_limit(1000)
        try:
            s.attn()
            torch.cuda.synchronize()
        finally:
            rb._lib.set_wait_limit(0)
        err = rb.device_error()
        assert err in (0, rb._lib.DEVERR_PFX_WAIT)
        if not err:
            s.check()
        s.attn()
        assert rb.device_error() == 0
        s.check()
