"""The quantised KV cache (rb_kv_write, rb_kv_read) against the formats' definition in 64 bits: codes, scales and the
values read back are equal, not close (the codes do not depend on the width of the arithmetic, the values are rounded
once)."""
import pytest
import torch

import rumik_fast_b200 as rb
from rumik_fast_b200.kv_cache import KVCache
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


def rows(shape, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g)
    x[..., ::16] *= 6
    return x.to(dtype)


def codes_of(cache):
    """(k, v) codes [..., hd] as int64, scales and minima in 64 bits, on the CPU."""
    got = []
    for c, p in ((cache.k, cache.k_par), (cache.v, cache.v_par)):
        c, p = c.cpu(), p.cpu()
        if cache.fmt == "int8":
            got.append((c.to(torch.int64) - 128, p.double(), torch.zeros_like(p, dtype=torch.float64)))
        else:
            codes = torch.stack([c & 15, c >> 4], -1).flatten(-2).to(torch.int64)
            halves = p.contiguous().view(torch.int16).view(p.shape + (2,))
            got.append((codes, halves[..., 0].contiguous().view(torch.bfloat16).double(),
                        halves[..., 1].contiguous().view(cache.dtype).double()))
    return got


def same(a, b):
    return a.shape == b.shape and torch.equal(torch.nan_to_num(a.double(), nan=-12345.0), torch.nan_to_num(b.double(), nan=-12345.0))


@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("fmt", ["int8", "int4", "plain"])
@pytest.mark.parametrize("n,T,nkv,hd,S", [(1, 1, 1, 64, 1), (3, 5, 2, 128, 17), (16, 1, 8, 128, 33), (1, 259, 3, 64, 300), (2, 33, 5, 128, 64)])
def test_write_and_read(n, T, nkv, hd, S, fmt, dtype):
    dt = DTYPES[dtype]
    k, v = rows((n, T, nkv, hd), dt, T), rows((n, T, nkv, hd), dt, T + 1)
    cache = KVCache(n, nkv, S, hd, fmt, dt)
    pos = torch.arange(n) % max(1, S - T + 1)      # a start of its own for each sequence
    cache.write(k.to(DEV), v.to(DEV), pos.to(DEV))
    got_k, got_v = cache.read(0, S)
    for x, got, side in ((k, got_k.cpu(), 0), (v, got_v.cpu(), 1)):
        want = torch.zeros(n, nkv, S, hd, dtype=dt)   # slots that were not written stand for zero
        for b in range(n):
            want[b, :, pos[b]:pos[b] + T] = ref.read_back(x[b], fmt).transpose(0, 1)
        assert same(got, want)
        if fmt != "plain":
            c, s, m = codes_of(cache)[side]
            for b in range(n):
                wc, ws, wm = (t.transpose(0, 1) for t in ref.quantise(x[b], fmt))
                at = slice(int(pos[b]), int(pos[b]) + T)
                assert torch.equal(c[b, :, at], wc) and same(s[b, :, at], ws)
                if fmt == "int4":
                    assert same(m[b, :, at], wm)
    part = cache.read(S // 2, S - S // 2)
    assert same(part[0], got_k[:, :, S // 2:]) and same(part[1], got_v[:, :, S // 2:])


@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("fmt", ["int8", "int4"])
def test_hard_rows(fmt, dtype):
    """Rows of zeros, of one value, of subnormals, at the type's largest value, of exact ties, and rows with a NaN or an
    infinity (all of which read back as NaN) beside ordinary ones."""
    dt = DTYPES[dtype]
    fi = torch.finfo(dt)
    hd = 64
    x = rows((1, 14, 1, hd), dt, 3)
    x[0, 0] = 0
    x[0, 1] = -0.0
    x[0, 2] = 1.7
    x[0, 3] = -2.5
    x[0, 4] = fi.max
    x[0, 5, 0, ::2], x[0, 5, 0, 1::2] = fi.max, -1.0
    x[0, 6] = 0
    x[0, 6, 0, 5] = fi.tiny / 8                      # a subnormal
    x[0, 7] = (torch.arange(hd) % 9).to(dt) * fi.tiny / 16
    x[0, 8] = ((torch.arange(hd) - 32).to(torch.float32) * 0.5).to(dt)
    x[0, 8, 0, 0] = 127.0                            # s = 1: halves are exact ties
    x[0, 9] = ((torch.arange(hd) % 31).to(torch.float32) * 0.5).to(dt)  # int4: range 15, s = 1, halves are ties
    x[0, 10, 0, 7] = float("nan")
    x[0, 11, 0, 63] = float("inf")
    x[0, 12, 0, 0] = -float("inf")
    x[0, 13, 0, :] = -3.0
    x[0, 13, 0, 9] = 100.0
    cache = KVCache(1, 1, 14, hd, fmt, dt)
    cache.write(x.to(DEV), x.flip(1).to(DEV), torch.zeros(1, dtype=torch.int64, device=DEV))
    k, v = cache.read(0, 14)
    want = ref.read_back(x[0], fmt).transpose(0, 1)[None]
    assert same(k.cpu(), want) and same(v.cpu(), want.flip(2))
    assert torch.isnan(k[0, 0, 10:13]).all() and torch.isfinite(k[0, 0, :10]).all() and torch.isfinite(k[0, 0, 13]).all()


def test_range_beyond_fp32():
    """bf16 rows whose range overflows fp32 have no int4 scale (NaN); int8 keeps them, clamped to finite values."""
    x = torch.zeros(1, 1, 1, 64, dtype=torch.bfloat16)
    x[..., 0], x[..., 1] = 3.3e38, -3.3e38
    pos = torch.zeros(1, dtype=torch.int64, device=DEV)
    for fmt in ("int4", "int8"):
        cache = KVCache(1, 1, 1, 64, fmt, torch.bfloat16)
        cache.write(x.to(DEV), x.to(DEV), pos)
        got = cache.read(0, 1)[0].cpu()
        assert same(got, ref.read_back(x[0], fmt).transpose(0, 1)[None])
        assert torch.isnan(got).all() if fmt == "int4" else torch.isfinite(got).all()


@pytest.mark.parametrize("fmt", ["int8", "int4", "plain"])
def test_views_of_a_fused_projection(fmt):
    """k and v as the views of one [B, q | k | v] projection output, one token without a token axis, and transposed rows."""
    B, nkv, hd = 3, 2, 128
    fused = rows((B, (4 + 2 * nkv) * hd), torch.float16, 9).to(DEV)
    k = fused[:, 4 * hd:(4 + nkv) * hd].view(B, nkv, hd)
    v = fused[:, (4 + nkv) * hd:].view(B, nkv, hd)
    pos = torch.tensor([0, 7, 3], device=DEV)
    cache = KVCache(B, nkv, 8, hd, fmt)
    cache.write(k, v, pos)
    got = cache.read(0, 8)
    for x, g in ((k, got[0]), (v, got[1])):
        for b in range(B):
            assert same(g[b, :, pos[b]].cpu(), ref.read_back(x[b].cpu(), fmt))
    head_major = rows((B, nkv, 5, hd), torch.float16, 10).to(DEV)   # [B, nkv, T, hd] seen as [B, T, nkv, hd]
    cache.write(head_major.transpose(1, 2), head_major.transpose(1, 2), torch.zeros(B, dtype=torch.int64, device=DEV))
    assert same(cache.read(0, 5)[1].cpu(), ref.read_back(head_major.cpu(), fmt))


def test_slots_outside_the_cache_are_not_written():
    x = rows((4, 3, 2, 64), torch.float16, 11).to(DEV)
    cache = KVCache(4, 2, 8, 64, "int8")
    before = [t.clone() for t in cache.tensors()]
    cache.write(x, x, torch.tensor([-1, 6, 2, 2 ** 62], device=DEV))
    assert rb.device_error() == rb._lib.DEVERR_ARG
    want = ref.read_back(x.cpu(), "int8").transpose(1, 2)
    got = cache.read(0, 8)[0].cpu()
    assert same(got[0, :, :2], want[0, :, 1:]) and same(got[1, :, 6:], want[1, :, :2]) and same(got[2, :, 2:5], want[2])
    for t, b in zip(cache.tensors(), before):   # sequence 3 is untouched, and so are the other slots
        assert torch.equal(t[3], b[3]) and torch.equal(t[0, :, 2:], b[0, :, 2:]) and torch.equal(t[1, :, :6], b[1, :, :6])


def test_offsets_beyond_32_bits():
    """A cache of more than 2^32 bytes: its last sequence's last slots."""
    n, nkv, S, hd = 5, 8, 1 << 20, 128
    cache = KVCache(n, nkv, S, hd, "int8")     # 5.4 GB of codes a side
    x = rows((n, 3, nkv, hd), torch.float16, 12).to(DEV)
    cache.write(x, x, torch.full((n,), S - 3, dtype=torch.int64, device=DEV))
    k, v = cache.read(S - 4, 4)
    want = ref.read_back(x.cpu(), "int8").transpose(1, 2)
    assert same(k[:, :, 1:].cpu(), want) and same(v[:, :, 1:].cpu(), want) and not k[:, :, 0].any()


def test_empty_calls_and_another_stream():
    cache = KVCache(2, 2, 4, 64, "int4")
    cache.write(torch.empty(2, 0, 2, 64, device=DEV, dtype=torch.float16), torch.empty(2, 0, 2, 64, device=DEV, dtype=torch.float16),
                torch.zeros(2, dtype=torch.int64, device=DEV))
    assert cache.read(4, 0)[0].shape == (2, 2, 0, 64)
    x = rows((2, 4, 2, 64), torch.float16, 13).to(DEV)
    pos = torch.zeros(2, dtype=torch.int64, device=DEV)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        cache.write(x, x, pos)
        k, _ = cache.read(0, 4)
    side.synchronize()
    assert same(k.cpu(), ref.read_back(x.cpu(), "int4").transpose(1, 2))


def test_refusals():
    cache = KVCache(2, 2, 4, 64, "int8")
    x = torch.zeros(2, 1, 2, 64, device=DEV, dtype=torch.float16)
    pos = torch.zeros(2, dtype=torch.int64, device=DEV)
    for bad in (x.bfloat16(), x[:1], x[..., :32], x.transpose(2, 3), x.cpu()):
        with pytest.raises(RuntimeError):
            cache.write(bad, x, pos)
    with pytest.raises(RuntimeError):
        cache.write(x, x, pos.int())
    with pytest.raises(RuntimeError):
        cache.write(x, x, pos[:1])
    with pytest.raises(rb.RumikKernelError):   # rows that are not 16-byte aligned
        cache.write(torch.zeros(2 * 2 * 64 + 1, device=DEV, dtype=torch.float16)[1:].view(2, 1, 2, 64), x, pos)
    for a, n in ((-1, 2), (0, 5), (3, 2), (0, -1)):
        with pytest.raises(RuntimeError):
            cache.read(a, n)
    with pytest.raises(RuntimeError):
        KVCache(1, 1, 1, 96, "int8")
    with pytest.raises(RuntimeError):
        KVCache(1, 1, 1, 64, "int2")
    with pytest.raises(RuntimeError):
        KVCache.wrap(cache.k, cache.v)
    with pytest.raises(RuntimeError):
        KVCache.wrap(cache.k, cache.v, cache.k_par, None, dtype=torch.float16)
