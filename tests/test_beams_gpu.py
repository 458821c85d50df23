"""The beam selection and the reordering of the beams' rows (rb_beam_select, rb_beam_reorder). Selected beams, tokens and
moved rows are equal to the plain 64-bit form's; scores agree to fp32 rounding: |score| 2^-23 for each of the two
additions and 2^-20 for the logarithm of a sum of up to 2^20 exponentials."""
import pytest
import torch

import rumik_fast_b200 as rb
from rumik_fast_b200.beams import BeamReorder, BeamSelect
from rumik_fast_b200.kv_cache import KVCache
from tests import continuations_ref as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(scope="module", autouse=True)
def _gpu(native_lib):
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    rb.device_error()
    yield
    assert rb.device_error() == 0


def check(logits, scores, done, end, got, masked=False):
    s, parents, tokens, fin, margin = ref.select(logits, scores, done, end, masked)
    assert margin > 1e-4, "the inputs leave the order to rounding"
    assert torch.equal(got["parents"].cpu(), torch.from_numpy(parents)) and torch.equal(got["tokens"].cpu(), torch.from_numpy(tokens))
    assert torch.equal(got["done"].cpu(), torch.from_numpy(fin))
    g, w = got["scores"].cpu().double(), torch.from_numpy(s)
    fine = torch.isfinite(w)
    assert torch.equal(fine, torch.isfinite(g)) and torch.equal(g[~fine], w[~fine])
    assert ((g - w).abs()[fine] <= 2 * 2.0 ** -23 * w.abs()[fine].clamp(min=8) + 2.0 ** -20).all()


def inputs(R, nb, V, dtype, seed, spread=2.5):
    """Logits and scores whose order is not decided by rounding (the scores are drawn again until it is not)."""
    g = torch.Generator().manual_seed(seed)
    logits = (torch.randn(R, nb, V, generator=g) * spread).to(dtype)
    done = torch.zeros(R, nb, dtype=torch.bool)
    done[:, nb // 2::3] = nb > 3
    for _ in range(50):
        scores = -2 - 5 * torch.rand(R, nb, generator=g)
        if ref.select(logits, scores, done, V - 1)[4] > 2e-4:
            break
    return logits, scores, done


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("R,nb,V", [(1, 1, 1), (1, 1, 5), (2, 3, 2), (1, 4, 16385), (3, 5, 4096), (2, 16, 4097), (1, 32, 9000), (5, 8, 127), (1, 2, 70001)])
def test_select(R, nb, V, dtype):
    logits, scores, done = inputs(R, nb, V, dtype, R + nb + V)
    sel = BeamSelect(logits.to(DEV), scores.to(DEV), done.to(DEV), end_idx=V - 1)
    check(logits, scores, done, V - 1, sel())
    first = {k: v.clone() for k, v in sel().items()}
    assert all(torch.equal(v, first[k]) for k, v in sel().items())


def test_largest_vocabulary():
    logits, scores, done = inputs(1, 2, 1 << 20, torch.float16, 3)
    check(logits, scores, done, 5, BeamSelect(logits.to(DEV), scores.to(DEV), done.to(DEV), end_idx=5)())


@pytest.mark.parametrize("order", ["up", "down", "shuffled"])
@pytest.mark.parametrize("nb,V", [(16, 9000), (32, 16500)])
def test_rows_of_several_batches(nb, V, order):
    """More rows than CTAs at once: a CTA takes several batches of its row, whose logits rise, fall or do neither."""
    at = torch.arange(V)
    if order == "down":
        at = at.flip(0)
    elif order == "shuffled":
        at = at[torch.randperm(V, generator=torch.Generator().manual_seed(V))]
    logits = (at * 0.002).float().expand(40, nb, V).contiguous()
    scores = (-0.0103 * torch.arange(nb)).float().expand(40, nb).contiguous()
    done = torch.zeros(40, nb, dtype=torch.bool)
    check(logits, scores, done, 3, BeamSelect(logits.to(DEV), scores.to(DEV), done.to(DEV), end_idx=3)())


def test_ties_go_to_the_lowest_beam_and_row():
    """All logits and scores equal, and a few equal peaks: every order is decided by the index."""
    for V in (7, 4096, 10000):
        logits = torch.zeros(2, 4, V, dtype=torch.float16)
        scores = torch.full((2, 4), -1.0)
        done = torch.zeros(2, 4, dtype=torch.bool)
        got = BeamSelect(logits.to(DEV), scores.to(DEV), done.to(DEV), end_idx=0)()
        assert torch.equal(got["parents"].cpu(), torch.zeros(2, 4, dtype=torch.int64))
        assert torch.equal(got["tokens"].cpu(), torch.arange(4).expand(2, 4))
        assert got["done"].cpu().tolist() == [[True, False, False, False]] * 2
        logits[:, :, V - 3:] = 4.0
        got = BeamSelect(logits.to(DEV), scores.to(DEV), done.to(DEV), end_idx=0)()
        assert got["parents"].cpu().tolist() == [[0, 0, 0, 1]] * 2
        assert got["tokens"].cpu().tolist() == [[V - 3, V - 2, V - 1, V - 3]] * 2


def test_masked_rows_and_the_first_step():
    """Rows masked with -inf and with the type's lowest value, beams with a score of -inf (the first step of a search),
    more beams than live candidates, and the end masked while step < min_new."""
    V = 5000
    for dtype in (torch.float16, torch.float32):
        logits, scores, done = inputs(2, 6, V, dtype, 21)
        done[:] = False
        scores[:, 1:] = -float("inf")
        logits[:, :, 100:4900] = -float("inf")
        logits[:, :, 4900:] = torch.finfo(dtype).min
        check(logits, scores, done, 7, BeamSelect(logits.to(DEV), scores.to(DEV), done.to(DEV), end_idx=7)())
        logits[:, 0, 3:] = -float("inf")      # three candidates for six places: the rest by index, at -inf
        check(logits, scores, done, 2, BeamSelect(logits.to(DEV), scores.to(DEV), done.to(DEV), end_idx=2)())
        step = torch.tensor([4], device=DEV)
        sel = BeamSelect(logits.to(DEV), scores.to(DEV), done.to(DEV), end_idx=2, step=step, min_new=5)
        check(logits, scores, done, 2, sel(), masked=True)
        step += 1
        check(logits, scores, done, 2, sel())
        logits[:] = -float("inf")             # nothing at all
        check(logits, scores, done, 2, BeamSelect(logits.to(DEV), scores.to(DEV), done.to(DEV), end_idx=2)())


def test_finished_beams_only_and_token_ids():
    logits, scores, done = inputs(2, 4, 300, torch.bfloat16, 22)
    done[:] = True
    done[1, 2] = False
    ids = torch.randperm(100000, generator=torch.Generator().manual_seed(1))[:300]
    got = BeamSelect(logits.to(DEV), scores.to(DEV), done.to(DEV), end_idx=0, ids=ids.to(DEV))()
    _, _, rows, _, _ = ref.select(logits, scores, done, 0)
    assert torch.equal(got["tokens"].cpu(), ids[torch.from_numpy(rows)])
    got["tokens"].copy_(torch.from_numpy(rows))
    check(logits, scores, done, 0, got)


def test_rows_without_a_distribution():
    """A NaN or +inf in a live beam's row: the beam has no candidates, and the error word says so. A NaN score: no error,
    the beam does not count; a finished beam's logits are not looked at."""
    for bad in (float("nan"), float("inf")):
        logits, scores, done = inputs(1, 4, 4500, torch.float32, 23)
        done[0] = torch.tensor([False, False, True, False])
        logits[0, 1, 4400], logits[0, 2, 5] = bad, bad
        got = BeamSelect(logits.to(DEV), scores.to(DEV), done.to(DEV), end_idx=9)()
        torch.cuda.synchronize()
        assert rb.device_error() == rb._lib.DEVERR_ARG
        check(logits, scores, done, 9, got)
        logits[0, 1, 4400] = 0
        scores[0, 0] = bad
        check(logits, scores, done, 9, BeamSelect(logits.to(DEV), scores.to(DEV), done.to(DEV), end_idx=9)())


def test_strided_logits():
    """The rows of a padded head output."""
    logits, scores, done = inputs(3, 4, 1001, torch.float16, 24)
    wide = torch.full((3, 4, 1024), 60000.0, dtype=torch.float16, device=DEV)
    wide[..., :1001] = logits.to(DEV)
    check(logits, scores, done, 1000, BeamSelect(wide[..., :1001], scores.to(DEV), done.to(DEV), end_idx=1000)())


def test_extreme_logits():
    """Logits far apart and far from zero: the normaliser neither overflows nor loses the small scores."""
    logits, scores, done = inputs(1, 3, 6000, torch.float32, 25, spread=1.0)
    logits[0, 0] += 20000.0
    logits[0, 1] -= 20000.0
    logits[0, 2, 17] = 500.0
    # at 20000 a logit is known to 2^-9: scores of beams 0 and 1 carry that, so only the order within reach is checked
    got = BeamSelect(logits.to(DEV), scores.to(DEV), done.to(DEV), end_idx=0)()
    s, parents, tokens, _, _ = ref.select(logits, scores, done, 0)
    assert torch.isfinite(got["scores"]).all() and (got["scores"].cpu().double() - torch.from_numpy(s)).abs().max() <= 2.0 ** -8


@pytest.mark.parametrize("R,nb,heads,S,tail", [(1, 1, 1, 1, (64,)), (1, 2, 2, 9, (128,)), (2, 4, 3, 33, (8,)), (1, 8, 8, 300, (128,)),
                                               (3, 5, 2, 17, (1,)), (1, 16, 2, 50, (64,)), (1, 32, 1, 129, (4,))])
@pytest.mark.parametrize("dtype", [torch.float16, torch.int32])
def test_reorder(R, nb, heads, S, tail, dtype):
    g = torch.Generator().manual_seed(R * 100 + nb)
    t = [torch.randint(-9000, 9000, (R * nb, heads, S) + tail, generator=g).to(dtype) for _ in range(3)]
    t.append(torch.randint(0, 256, (R * nb, 2 * heads, S, 64), generator=g, dtype=torch.uint8))
    for trial in range(4):
        parents = torch.randint(0, nb, (R, nb), generator=g) if trial else torch.arange(nb).flip(0).expand(R, nb).contiguous()
        if trial == 3:
            parents = torch.arange(nb).expand(R, nb).contiguous()     # everybody stays
        slots = torch.randint(0, S + 1, (R * nb,), generator=g)
        slots[0] = S
        dev = [x.to(DEV) for x in t]
        BeamReorder(dev, parents.to(DEV), slots.to(DEV))()
        for x, d in zip(t, dev):
            assert torch.equal(d.cpu(), ref.reorder(x, parents, slots))


@pytest.mark.parametrize("fmt", ["plain", "int8", "int4"])
def test_reorder_caches_with_their_parameters(fmt):
    """A list of caches of odd lengths (rows and 2- and 4-byte parameters), more tensors than one launch takes."""
    nb, nkv, S, hd = 4, 2, 21, 64
    g = torch.Generator().manual_seed(5)
    caches = [KVCache(nb, nkv, S, hd, fmt) for _ in range(60)]
    pos = torch.zeros(nb, dtype=torch.int64, device=DEV)
    for c in caches:
        x = torch.randn(nb, S, nkv, hd, generator=g).half().to(DEV)
        c.write(x, x * 2, pos)
    parents, slots = torch.tensor([[2, 0, 0, 3]]), torch.tensor([13, 21, 8, 0])
    before = [[t.cpu() for t in c.tensors()] for c in caches]
    BeamReorder([t for c in caches for t in c.tensors()], parents.to(DEV), slots.to(DEV))()
    for c, old in zip(caches, before):
        for t, o in zip(c.tensors(), old):
            assert torch.equal(t.cpu(), ref.reorder(o, parents, slots))


def test_reorder_misaligned_tensors():
    """Tensors that start two bytes into an allocation: narrower accesses, the same result."""
    base = torch.arange(2 * 3 * 5 * 8 + 1, dtype=torch.int16)
    t = base.to(DEV)[1:].view(2, 3, 5, 8)
    parents, slots = torch.tensor([[1, 0]]), torch.tensor([5, 4])
    BeamReorder([t], parents.to(DEV), slots.to(DEV))()
    assert torch.equal(t.cpu(), ref.reorder(base[1:].view(2, 3, 5, 8), parents, slots))


def test_reorder_indices_outside():
    """A parent or a length that is none leaves its request as it is; the others are reordered."""
    t = torch.arange(6 * 2 * 4 * 8, dtype=torch.int32).view(6, 2, 4, 8)
    for parents, slots in (([[1, 3, 0], [1, 1, 1]], [4, 4, 4, 2, 3, 1]), ([[1, 0, 0], [1, 1, 1]], [4, 5, 4, 2, 3, 1]),
                           ([[-1, 0, 0], [1, 1, 1]], [4, 4, 4, 2, 3, 1])):
        d = t.to(DEV)
        BeamReorder([d], torch.tensor(parents, device=DEV), torch.tensor(slots, device=DEV))()
        assert rb.device_error() == rb._lib.DEVERR_ARG
        assert torch.equal(d[:3].cpu(), t[:3])
        assert torch.equal(d[3:].cpu(), ref.reorder(t[3:], torch.tensor(parents[1:]), torch.tensor(slots[3:])))


def test_refusals():
    f = lambda *s, dt=torch.float32: torch.zeros(*s, dtype=dt, device=DEV)  # noqa: E731
    logits, scores, done = f(1, 4, 10), f(1, 4), f(1, 4, dt=torch.bool)
    BeamSelect(logits, scores, done, end_idx=9)
    for bad in (dict(logits=logits.double()), dict(logits=logits[0]), dict(logits=f(1, 10, 4).transpose(1, 2)), dict(scores=scores.half()),
                dict(scores=f(2, 4)), dict(done=f(1, 4)), dict(end_idx=10), dict(end_idx=-1), dict(step=f(1)), dict(ids=f(9, dt=torch.int64)),
                dict(logits=f(1, 33, 10), scores=f(1, 33), done=f(1, 33, dt=torch.bool))):
        with pytest.raises(RuntimeError):
            BeamSelect(**{**dict(logits=logits, scores=scores, done=done, end_idx=9), **bad})
    t, parents, slots = f(4, 2, 8, 64), f(1, 4, dt=torch.int64), f(4, dt=torch.int64)
    BeamReorder([t], parents, slots)
    for bad in (([], parents, slots), ([t[:3]], parents, slots), ([t, f(4, 2, 9, 64)], parents, slots), ([t.transpose(1, 2)], parents, slots),
                ([f(4, 2, 8, 1, dt=torch.uint8)], parents, slots), ([t], parents.int(), slots), ([t], parents, slots[:3]), ([t], parents[0], slots)):
        with pytest.raises(RuntimeError):
            BeamReorder(*bad)


@pytest.mark.parametrize("nb,end", [(2, 1), (4, 5), (6, 3), (8, 0)])
def test_finished_beams_without_a_score(nb, end):
    """A finished beam whose score is not finite has no candidate: its rows fill up in their order like a live one's, its
    end row among them and not before them."""
    for seed, bad in enumerate((-float("inf"), float("nan"), float("inf"))):
        logits, scores, done = inputs(2, nb, 40, torch.float16, 60 + seed)
        done[:], scores[:] = True, bad                    # nobody has one
        check(logits, scores, done, end, BeamSelect(logits.to(DEV), scores.to(DEV), done.to(DEV), end_idx=end)())
        scores[1, nb - 1] = -1.5                          # the last one of a request is finished with a score
        check(logits, scores, done, end, BeamSelect(logits.to(DEV), scores.to(DEV), done.to(DEV), end_idx=end)())


@pytest.mark.parametrize("shift", [20000.0, -20000.0, 3.0e6])
def test_scores_of_logits_far_from_zero(shift):
    """Logits that lie around 20,000 or 3,000,000 are exact inputs: their differences, and so the scores, are as exact as
    those of logits around zero (the module's bound, which does not depend on the logits' size)."""
    g = torch.Generator().manual_seed(26)
    logits = torch.randn(2, 4, 6000, generator=g) * 4.0 + shift
    done = torch.zeros(2, 4, dtype=torch.bool)
    for _ in range(200):
        scores = -2 - 5 * torch.rand(2, 4, generator=g)
        if ref.select(logits, scores, done, 0)[4] > 2e-4:
            break
    check(logits, scores, done, 0, BeamSelect(logits.to(DEV), scores.to(DEV), done.to(DEV), end_idx=0)())
