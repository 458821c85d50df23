"""The C ABI of the caches, the prefix attention and the beams without a GPU: bad arguments come back with their status
before any CUDA call, empty calls succeed."""
import ctypes
import os
import re

from rumik_fast_b200 import _lib

A = 0x1000  # a 16-byte-aligned dummy address; validation rejects the call before it is dereferenced


def cache(**kw):
    c = _lib.KvCache(A, A, A, A, _lib.KV_INT8, _lib.F16, 2, 4, 128, 64)
    for k, v in kw.items():
        setattr(c, k, v)
    return c


def strides(*s):
    return (ctypes.c_int64 * 3)(*s)


def test_kv_write_validation(native_lib):
    def write(k=A, v=A, ks=(1024, 512, 128), vs=(1024, 512, 128), T=1, pos=A, **kw):
        return native_lib.rb_kv_write(ctypes.byref(cache(**kw)), k, v, strides(*ks), strides(*vs), T, pos, 0, None)

    assert write(T=0) == _lib.OK
    assert write(n_seqs=0) == _lib.OK
    assert write(T=-1) == _lib.ERR_SHAPE
    assert write(fmt=3) == _lib.ERR_SHAPE
    assert write(dtype=_lib.F32) == _lib.ERR_DTYPE
    assert write(head_dim=96) == _lib.ERR_SHAPE
    assert write(n_kv_heads=0) == _lib.ERR_SHAPE
    assert write(cache_len=-1) == _lib.ERR_SHAPE
    assert write(cache_len=0) == _lib.ERR_SHAPE
    assert write(k=None) == _lib.ERR_NULL
    assert write(pos=None) == _lib.ERR_NULL
    assert write(k_par=None) == _lib.ERR_NULL
    assert write(k_par=A + 1) == _lib.ERR_ALIGN
    assert write(fmt=_lib.KV_INT4, v_par=A + 2) == _lib.ERR_ALIGN
    assert write(v=A + 8) == _lib.ERR_ALIGN
    assert write(ks=(1024, 516, 128)) == _lib.ERR_ALIGN
    assert native_lib.rb_kv_write(None, A, A, strides(8, 8, 8), strides(8, 8, 8), 1, A, 0, None) == _lib.ERR_NULL


def test_kv_read_validation(native_lib):
    def read(start=0, count=1, k=A, v=A, **kw):
        return native_lib.rb_kv_read(ctypes.byref(cache(**kw)), k, v, start, count, 0, None)

    assert read(count=0) == _lib.OK
    assert read(start=64, count=0) == _lib.OK
    assert read(start=64) == _lib.ERR_SHAPE
    assert read(count=65) == _lib.ERR_SHAPE
    assert read(start=-1) == _lib.ERR_SHAPE
    assert read(start=1, count=2 ** 63 - 1) == _lib.ERR_SHAPE
    assert read(k=None) == _lib.ERR_NULL
    assert read(v=A + 4) == _lib.ERR_ALIGN


def test_prefix_attn_validation(native_lib):
    def attn(prefix={}, own={}, **kw):
        p, o = cache(n_seqs=1, **prefix) if prefix is not None else None, cache(**own) if own is not None else None
        a = _lib.PrefixAttnArgs(A, 1024, A, 1024, 2, 8, ctypes.pointer(p) if p else None, A, ctypes.pointer(o) if o else None, A,
                                1.0, A, 1 << 40)
        for k, v in kw.items():
            setattr(a, k, v)
        return native_lib.rb_prefix_attn(ctypes.byref(a), 0, None)

    assert attn(n_seqs=0, own=dict(n_seqs=0)) == _lib.OK
    assert attn(prefix=None, own=None) == _lib.ERR_NULL
    assert attn(own=dict(n_seqs=3)) == _lib.ERR_SHAPE
    assert attn(own=dict(fmt=_lib.KV_INT4)) == _lib.ERR_SHAPE
    assert attn(own=dict(dtype=_lib.BF16)) == _lib.ERR_SHAPE
    assert attn(own=dict(n_kv_heads=2)) == _lib.ERR_SHAPE
    assert attn(own=dict(head_dim=64)) == _lib.ERR_SHAPE
    assert attn(prefix=dict(k=None)) == _lib.ERR_NULL
    assert attn(n_q_heads=6) == _lib.ERR_SHAPE
    assert attn(n_q_heads=68) == _lib.ERR_SHAPE          # seventeen query heads a key-value head
    assert attn(n_seqs=1025, own=dict(n_seqs=1025)) == _lib.ERR_SHAPE
    assert attn(q=None) == _lib.ERR_NULL
    assert attn(prefix_len=None) == _lib.ERR_NULL
    assert attn(own_len=None) == _lib.ERR_NULL
    assert attn(ws=None) == _lib.ERR_NULL
    assert attn(ldq=1020) == _lib.ERR_SHAPE
    assert attn(ldo=1028) == _lib.ERR_ALIGN
    assert attn(q=A + 8) == _lib.ERR_ALIGN
    assert attn(scale=float("nan")) == _lib.ERR_SHAPE
    assert attn(scale=float("inf")) == _lib.ERR_SHAPE
    assert native_lib.rb_prefix_attn(None, 0, None) == _lib.ERR_NULL
    assert native_lib.rb_prefix_attn_workspace(None) == -_lib.ERR_NULL


def test_beam_select_validation(native_lib):
    def select(**kw):
        a = _lib.BeamSelectArgs(A, _lib.F16, 100, 2, 4, 100, 99, A, A, None, None, 0, A, A, A, A, A, 1 << 40)
        for k, v in kw.items():
            setattr(a, k, v)
        return native_lib.rb_beam_select(ctypes.byref(a), 0, None)

    assert select(requests=0) == _lib.OK
    for kw in (dict(requests=-1), dict(n_beams=0), dict(n_beams=33), dict(n_vocab=0), dict(n_vocab=(1 << 20) + 1), dict(end_idx=100),
               dict(end_idx=-1), dict(ld=99), dict(requests=20000), dict(ws_bytes=16)):
        assert select(**kw) == _lib.ERR_SHAPE, kw
    assert select(logits_dtype=3) == _lib.ERR_DTYPE
    for nm in ("logits", "scores", "done", "out_scores", "out_parents", "out_tokens", "out_done", "ws"):
        assert select(**{nm: None}) == _lib.ERR_NULL, nm
    assert select(logits=A + 1) == _lib.ERR_ALIGN
    assert select(ws=A + 8) == _lib.ERR_ALIGN
    assert native_lib.rb_beam_select(None, 0, None) == _lib.ERR_NULL
    assert native_lib.rb_beam_select_workspace(1, 33, 10) == -_lib.ERR_SHAPE
    assert native_lib.rb_beam_select_workspace(1, 4, 16385) > 0


def test_beam_reorder_validation(native_lib):
    def reorder(p=A, heads=2, row=128, count=1, R=1, nb=4, S=16, parents=A, slots=A):
        return native_lib.rb_beam_reorder((_lib.BeamTensor * 1)(_lib.BeamTensor(p, heads, row)), count, R, nb, S, parents, slots, 0, None)

    assert reorder(count=0) == _lib.OK and reorder(R=0) == _lib.OK and reorder(S=0) == _lib.OK
    for kw in (dict(count=-1), dict(R=-1), dict(nb=0), dict(nb=33), dict(S=-1), dict(heads=0), dict(row=0), dict(row=3)):
        assert reorder(**kw) == _lib.ERR_SHAPE, kw
    assert reorder(p=None) == _lib.ERR_NULL and reorder(parents=None) == _lib.ERR_NULL and reorder(slots=None) == _lib.ERR_NULL
    assert reorder(p=A + 1) == _lib.ERR_ALIGN


def test_no_read_only_loads_of_what_the_launch_before_may_write():
    """Lengths, positions, parents and scores are written by launches that may still run when these kernels become resident
    (programmatic dependent launch). __ldg is a load of memory that is read-only for a kernel's whole life: it need not stay
    behind the kernel's wait, so none of these kernels uses it."""
    csrc = os.path.join(os.path.dirname(os.path.abspath(_lib.__file__)), "csrc")
    for name in ("kv_cache.cu", "prefix_attn.cu", "prefix_attn_tc.cu", "beams.cu"):
        with open(os.path.join(csrc, name)) as f:
            code = re.sub(r"//[^\n]*", "", f.read())
        assert "griddep_wait()" in code, name
        assert not re.search(r"__ldg\s*\(|ld\.global\.nc|__restrict__", code), name


def test_beam_select_workspace_follows_the_launch(native_lib):
    """A launch has at most some thousand CTAs, or one a row: the workspace is for that many lists, not for one every 4,096
    logits of every row; and it grows with the vocabulary and the rows as far as the launch does."""
    need = native_lib.rb_beam_select_workspace
    assert need(2047, 32, 1 << 20) < 1 << 26                     # 65,504 rows of one list each
    assert need(8, 16, 130001) >= 128 * 32 * 16 * 8              # 32 chunks a row fit the CTAs
    for requests, beams in ((1, 1), (1, 32), (3, 5), (100, 16), (2047, 32)):
        sizes = [need(requests, beams, v) for v in (1, 4096, 4097, 70001, 1 << 20)]
        rows = requests * beams
        assert all(s >= rows * (beams * 16 + 8) for s in sizes), "one list, one row of candidates and a sum for each row"
        assert max(sizes) <= max(rows, 4096) * (beams + 1) * 8 + rows * beams * 8 + (rows + requests) * 4 + 5 * 16
