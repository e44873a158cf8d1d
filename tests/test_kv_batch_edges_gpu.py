"""Operators over a caller's paged cache where numbers are hard: infinities, weights far below another, values near the end of the numbers, shares that are joined; the definition is
tests/kv_reference.py."""
import math

import pytest
import torch

from tests.kv_reference import DTYPES, attend, make_cache, stored_rows, tolerance, visible
from tests.test_kv_batch_gpu import fill, rows, sequences, stored_poison, tree

pytestmark = pytest.mark.gpu


def agrees(got, q, cache, fmt, states, counts, weight, scale=None, window=0, first=0, trees=None, few=None):
    """every row against the definition; a result that is not finite has to be that very one.  weight: by how much of itself a weight may be off; few: what f16 weights
    that are subnormal numbers may come to, where that is less than every key's.  Returns the definition's results."""
    heads, dim = q.shape[1], q.shape[2]
    scale = dim ** -0.5 if scale is None else scale
    r, outs = 0, []
    for i, (s, n) in enumerate(zip(states, counts)):
        k, v = stored_rows(cache, s, fmt)
        see = visible(s.seq_len - n, n, window, first, None if trees is None else trees[i])
        out, mean, size = attend(q[r:r + n].double(), k, v, see, scale)
        if not k.isfinite().all():                                  # how large scores are, of keys that are numbers
            size = attend(q[r:r + n].double(), k.nan_to_num(nan=0.0, posinf=0.0, neginf=0.0), v.nan_to_num(nan=0.0, posinf=0.0, neginf=0.0), see, scale)[2]
        tol = tolerance(out, mean, size, dim, s.seq_len, q.dtype, weight)
        # denominators may be sums of the rounded weights p (1 + d), |d| <= weight: sum p (1 + d) v / sum p (1 + d) is off by sum p d (v - out) / sum p (1 + d), at most weight (mean + |out|)
        tol = tol + weight * out.abs()
        # a weight under 2^-118 of the row's largest is 0 (kv_reference leaves 2^-8 of the range of 32 bits): off by less than that of its |v|, and a product under 2^-118 likewise
        tol = tol + s.seq_len * 2.0 ** -118 * (v[v.isfinite()].abs().max() + 1)
        if fmt == "f16":                                            # subnormal weights are off by 2^-25; the row's largest weighs 2^8 or more
            tol = tol + (s.seq_len * 2.0 ** -33 * v[v.isfinite()].abs().max() if few is None else few)
        x = got[r:r + n].double()
        whole = out.isfinite()
        assert torch.equal(x.isfinite(), whole), (i, n, s.seq_len, (x.isfinite() != whole).nonzero()[:4].tolist())
        assert torch.equal(x[~whole].nan_to_num(nan=7.0, posinf=1.0, neginf=-1.0), out[~whole].nan_to_num(nan=7.0, posinf=1.0, neginf=-1.0)), (i, n, s.seq_len)
        bad = (x - out).abs()[whole] > tol[whole]
        assert not bad.any(), (i, n, s.seq_len, int(bad.sum()), float(((x - out).abs()[whole] / tol[whole]).max()))
        outs.append(out); r += n
    assert r == got.shape[0]
    return torch.cat(outs)


def batch_of(cache, lens, counts, seed=0):
    from krasis_amd.kv_cache import KVBatch
    states = sequences(cache, [n - c for n, c in zip(lens, counts)], seed)
    batch = KVBatch(cache, states, counts)
    for s, c in zip(states, counts):
        s.advance(c)
    return batch, states


def pages_for(lens, page):
    return sum(-(-n // page) for n in lens) + 2


# ---------------------------------------------------------------------------------------------------------------- infinities
SPLIT = [6001, 9005]


@pytest.mark.parametrize("window,first", [(0, 0), (20, 0), (20, 4), (50, 70)])
@pytest.mark.parametrize("lens,counts", [([1, 5, 33, 97, 160], [1, 1, 1, 1, 1]), ([1, 5, 33, 97, 161], [1, 1, 1, 2, 1]), ([70, 130, 41], [40, 64, 41]), (SPLIT, [1, 1]), (SPLIT, [2, 1]), (SPLIT, [40, 33])])
@pytest.mark.parametrize("fmt", ["bf16", "f16"])
def test_infinite_values_reach_the_rows_that_see_them_as_they_are(fmt, lens, counts, window, first):
    """Channels apart for each: the last key's, the window's first key's and the first key's values are infinite, one before all windows, one a NaN, and one channel has both signs."""
    cache = make_cache(2, 64, fmt, pages_for(lens, 16))
    fill(cache, fmt, 1)
    batch, states = batch_of(cache, lens, counts)
    stored_poison(cache, fmt, states)
    for s, c in zip(states, counts):
        n = s.seq_len
        for pos, channel, bad in ((n - 1, 3, math.inf), (max(0, n - 20), 9, -math.inf), (max(0, n - c), 12, -math.inf), (0, 40, math.inf), (n // 2, 20, math.nan), (n // 3, 21, -math.inf),
                                  (n - 1, 50, -math.inf), (0, 50, math.inf), (min(n - 1, 31), 33, math.inf), (min(n - 1, 64), 34, -math.inf)):
            cache.v_cache[0, s.pages[pos // 16], pos % 16, 1, channel] = bad
    q = rows(sum(counts), 6, 64, DTYPES[fmt], 3)
    got = batch.attend(0, q, window=window, keep_first=first)
    if not window:
        assert (max(batch._need.values()) > 0) == (lens is SPLIT)
    out = agrees(got, q, cache, fmt, states, counts, 2.0 ** -8 if fmt == "bf16" else 2.0 ** -11, window=window, first=first)
    assert bool((out == math.inf).any()) and bool((out == -math.inf).any()) and bool(out.isfinite().any())


@pytest.mark.parametrize("fmt", ["bf16", "mx8"])
def test_infinite_keys_draw_everything_or_nothing(fmt):
    """A key whose products are all -infinity has no weight; one of +infinity leaves no number.  Over pages of eight bits a block that held one reads as NaN."""
    lens, counts = [33, 90, 200], [1, 2, 40]
    cache = make_cache(2, 64, fmt, pages_for(lens, 16))
    fill(cache, fmt, 2)
    batch, states = batch_of(cache, lens, counts)
    stored_poison(cache, fmt, states)
    q = rows(sum(counts), 4, 64, torch.bfloat16, 3).abs()
    for s in states:
        at = (0, s.pages[0], 7, 1)
        if fmt == "bf16":
            cache.k_cache[at][5] = -math.inf
        else:
            cache.k_scale[at][0] = 255
    got = batch.attend(0, q)
    out = agrees(got, q, cache, fmt, states, counts, 2.0 ** -8)
    assert bool(out[:, :2].isfinite().all()) and bool(out[:, 2:].isnan().all() if fmt == "mx8" else out[:, 2:].isfinite().all())


# ---------------------------------------------------------------------------------------------------------------- weights far apart
def scored(cache, fmt, states, counts, heads, dim, dtype, score, value, seed=5):
    """keys whose products with every query are score(positions) and a little, values value(positions) in all channels; the queries, for scale 1"""
    g = torch.Generator(device="cuda").manual_seed(seed)
    kvh = cache.num_kv_heads
    for s in states:
        n = s.seq_len
        pos = torch.arange(n, device="cuda")
        k = 0.05 * torch.randn((n, kvh, dim), generator=g, device="cuda")
        k[:, :, 2] = (score(pos, n) / 8)[:, None]
        v = value(pos, n)[:, None, None] * (1 + 0.25 * torch.rand((n, kvh, dim), generator=g, device="cuda"))
        page = torch.tensor(s.pages, device="cuda")[pos // cache.page_size]
        cache.k_cache[0, page, pos % cache.page_size] = k.to(DTYPES[fmt]); cache.v_cache[0, page, pos % cache.page_size] = v.to(DTYPES[fmt])
    q = torch.randn((sum(counts), heads, dim), generator=g, device="cuda")
    q[:, :, 2] = 8.0
    return q.to(dtype)


@pytest.mark.parametrize("gap", [12, 17, 20, 24])
@pytest.mark.parametrize("place", ["first", "middle", "three"])
@pytest.mark.parametrize("dim,lens,counts", [(64, [4096], [1]), (128, [300, 20000], [1, 1]), (256, [700, 5000], [4, 1]), (64, [4500, 77], [40, 33]), (128, [2049, 9000], [64, 20]), (256, [3000], [70])])
def test_keys_far_under_one_that_draws_nearly_all(dim, lens, counts, place, gap):
    """f16 pages, where keys weigh exp(-gap) of one whose value is next to nothing: together they are the result.  A weight is an f16 number next to a reference, 2^8 at the largest of its half
    tile or more: 32 keys beside the large one are off by 2^-25 of 2^8 of its weight, or all of their own; the others by half a step of 2^-11."""
    cache = make_cache(2, dim, "f16", pages_for(lens, 16))
    fill(cache, "f16", 1)
    batch, states = batch_of(cache, lens, counts)
    stored_poison(cache, "f16", states)
    at = {"first": lambda p, n: p == 0, "middle": lambda p, n: p == n // 2, "three": lambda p, n: (p == 5) | (p == n // 3) | (p == n // 2)}[place]
    q = scored(cache, "f16", states, counts, 4, dim, torch.float16, lambda p, n: torch.where(at(p, n), float(gap), 0.0), lambda p, n: torch.where(at(p, n), 0.0, 256.0))
    got = batch.attend(0, q, scale=1.0)
    beside = 32 * (3 if place == "three" else 1)
    out = agrees(got, q, cache, "f16", states, counts, 2.0 ** -11, scale=1.0, few=beside * min(2.0 ** -33, math.exp(4 - gap)) * 320.0)
    assert float(out.abs().min()) > 0


@pytest.mark.parametrize("dim,lens,counts", [(64, [3000], [1]), (128, [2000, 700], [2, 40])])
def test_scores_that_go_up_and_down(dim, lens, counts):
    """f16 pages: scores that fall and rise by 40 natural units over the sequence, small values where the weights are; what is far under the largest weight has no part"""
    cache = make_cache(2, dim, "f16", pages_for(lens, 16))
    fill(cache, "f16", 1)
    batch, states = batch_of(cache, lens, counts)
    q = scored(cache, "f16", states, counts, 4, dim, torch.float16, lambda p, n: 20.0 * torch.cos(p * (9.0 / n)), lambda p, n: 1.0 + 0.1 * (p % 7))
    agrees(batch.attend(0, q, scale=1.0), q, cache, "f16", states, counts, 2.0 ** -11, scale=1.0)


# ---------------------------------------------------------------------------------------------------------------- values near the end of the numbers
@pytest.mark.parametrize("rise", [6, 25, 29, 60])
@pytest.mark.parametrize("dim,lens,counts", [(64, [300], [1]), (128, [300, 900], [1, 3]), (64, [300], [40]), (128, [300, 900], [70, 64]), (256, [500], [33])])
def test_large_values_under_rising_scores(dim, lens, counts, rise):
    """bf16 pages: values of 2^117 under scores that rise by `rise` powers of two, far behind the first keys.  No sum of weights times values passes the plain form's, at most 900 times 2^117."""
    cache = make_cache(2, dim, "bf16", pages_for(lens, 16))
    fill(cache, "bf16", 1)
    batch, states = batch_of(cache, lens, counts)
    stored_poison(cache, "bf16", states)
    q = scored(cache, "bf16", states, counts, 4, dim, torch.bfloat16, lambda p, n: torch.where(p > n // 2, rise * math.log(2.0), 0.0), lambda p, n: torch.full(p.shape, 2.0 ** 117, device="cuda"))
    got = batch.attend(0, q, scale=1.0)
    out = agrees(got, q, cache, "bf16", states, counts, 2.0 ** -8, scale=1.0)
    assert bool(out.isfinite().all()) and float(out.abs().max()) > 2.0 ** 116


# ---------------------------------------------------------------------------------------------------------------- how near
@pytest.mark.parametrize("fmt,dim,lens,counts", [("bf16", 128, [97, 500], [1, 1]), ("mx8", 128, [97, 9000], [1, 1]), ("mx4", 64, [3000], [2]), ("e4m3", 256, [700, 90], [1, 2]), ("mx4", 128, [2000], [1])])
def test_single_tokens_weigh_in_sixteen_bits(fmt, dim, lens, counts):
    """sequences of at most 16 rows, bf16 queries: weights are two bf16 pieces, off by 2^-8 of 2^-8"""
    cache = make_cache(2, dim, fmt, pages_for(lens, 16))
    fill(cache, fmt, 3)
    batch, states = batch_of(cache, lens, counts)
    q = rows(sum(counts), 8, dim, torch.bfloat16, 4)
    agrees(batch.attend(0, q), q, cache, fmt, states, counts, 2.0 ** -16)


# ---------------------------------------------------------------------------------------------------------------- shares that are joined
@pytest.mark.parametrize("fmt,dtype,dim,lens,counts,window,first", [
    ("mx8", "bf16", 128, [4096, 4000, 3900, 4090, 4096, 3333, 4001, 4077], [12] * 8, 0, 0), ("mx8", "bf16", 128, [4096, 4000, 3900, 4090], [12, 3, 1, 12], 3000, 4), ("mx4", "f16", 64, [9001, 8000], [64, 60], 0, 0),
    ("mx8", "bf16", 128, [9001, 8000], [64, 33], 5, 7000), ("f16", "f16", 128, [9001, 8700], [64, 40], 4000, 8), ("bf16", "bf16", 64, [20000], [4], 0, 0), ("bf16", "bf16", 64, [20000], [4], 3, 18000)])
def test_trees_whose_sequences_are_shared_out(fmt, dtype, dim, lens, counts, window, first):
    cache = make_cache(2, dim, fmt, pages_for(lens, 64), page=64)
    fill(cache, fmt, 1, spread=1)
    batch, states = batch_of(cache, lens, counts)
    stored_poison(cache, fmt, states)
    trees = [tree(n, 3 + i) for i, n in enumerate(counts)]
    q = rows(sum(counts), 8, dim, DTYPES[dtype], 4)
    got = batch.attend_tree(0, q, trees, window=window, keep_first=first)
    assert min(batch._need.values()) > 0                            # partial results, joined
    weight = 2.0 ** -8 if dtype == "bf16" else 2.0 ** -11 if fmt == "f16" else 2.0 ** -16
    agrees(got, q, cache, fmt, states, counts, weight, window=window, first=first, trees=trees)


def test_two_streams_with_shares_each():
    """calls on two streams at once, both with partial results of their own"""
    lens, counts = [9000, 100, 400], [1, 1, 40]
    cache = make_cache(2, 128, "mx8", pages_for(lens, 16))
    fill(cache, "mx8", 1)
    batch, _ = batch_of(cache, lens, counts)
    q = rows(42, 16, 128, torch.bfloat16, 2)
    calls = lambda: batch.attend(0, q), lambda: batch.attend(0, q, window=4000, keep_first=4)
    want = [c() for c in calls]
    assert len(batch._need) == 2 and min(batch._need.values()) > 0
    torch.cuda.synchronize()
    streams, got = (torch.cuda.Stream(), torch.cuda.Stream()), ([], [])
    for _ in range(20):
        for s, c, g in zip(streams, calls, got):
            with torch.cuda.stream(s):
                g.append(c())
    torch.cuda.synchronize()
    assert all(torch.equal(x, w) for g, w in zip(got, want) for x in g)


def test_a_first_call_may_be_captured():
    """none of the kernels has run before in this form: what a first launch needs is no stream's work"""
    lens, counts = [5000, 70], [1, 33]
    for fmt, dtype, dim in (("mx4", torch.float16, 192), ("e4m3", torch.float16, 96)):
        cache = make_cache(1, dim, fmt, pages_for(lens, 128), page=128)
        fill(cache, fmt, 1)
        batch, states = batch_of(cache, lens, counts)
        q, k = rows(34, 5, dim, dtype, 2), rows(34, 1, dim, dtype, 3)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            batch.write(0, k, k)
            got = batch.attend(0, q)
        for _ in range(3):
            graph.replay()
            torch.cuda.synchronize()
            agrees(got, q, cache, fmt, states, counts, 2.0 ** -16)
            assert torch.equal(got, batch.attend(0, q))


# ---------------------------------------------------------------------------------------------------------------- scores
@pytest.mark.parametrize("power", [20, 27, 30, 34, 40, 60])
@pytest.mark.parametrize("fmt,dtype", [("bf16", "bf16"), ("f16", "f16"), ("mx8", "bf16"), ("mx8", "f16")])
@pytest.mark.parametrize("dim,lens,counts", [(64, [90], [1]), (128, [200, 9000], [2, 1]), (128, [200], [40]), (64, [9000, 100], [33, 70])])
def test_scores_of_any_size(fmt, dtype, dim, lens, counts, power):
    """Scores of up to 2^power: one key draws all, as every other is far under it.  32 bits hold scores to 2^-24 of their size, no more; weights are those of the scores that 32 bits hold."""
    cache = make_cache(2, dim, fmt, pages_for(lens, 16))
    fill(cache, fmt, 1)
    batch, states = batch_of(cache, lens, counts)
    stored_poison(cache, fmt, states)
    q = rows(sum(counts), 4, dim, DTYPES[dtype], 3)
    got = batch.attend(0, q, scale=2.0 ** (power - 3)).double()
    r = 0
    for s, n in zip(states, counts):
        k, v = stored_rows(cache, s, fmt)
        see = visible(s.seq_len - n, n).cuda()
        for h in range(4):
            score = torch.where(see, q[r:r + n, h].double() @ k[:, h // 2].t().contiguous(), -math.inf)
            top, at = score.topk(min(2, s.seq_len), -1)
            # two keys within what sums of 32 bits leave of the products are not told apart; the others have to be
            error = 2 * (dim + 16) * 2.0 ** -24 * (q[r:r + n, h].double().abs() @ k[:, h // 2].abs().t().contiguous()).amax(-1)
            alone = (top[:, 0] - top[:, -1] - error) * 2.0 ** (power - 3) > 40.0 if top.shape[1] > 1 else torch.ones(n, dtype=torch.bool, device="cuda")
            want = v[at[:, 0], h // 2]
            assert int(alone.sum()) * 2 > n or n < 3, int(alone.sum())
            assert bool(((got[r:r + n, h] - want).abs() <= torch.finfo(q.dtype).eps / 2 * want.abs() + 2.0 ** -24)[alone].all()), (s.seq_len, n, h, got[r:r + n, h][alone][:, :4], want[alone][:, :4])
            assert bool(got[r:r + n, h].isfinite().all())
        r += n


@pytest.mark.parametrize("scale", [0.0, 1e-30, 1e-41])
def test_scales_of_next_to_nothing(scale):
    lens, counts = [50, 300, 90], [1, 2, 40]
    cache = make_cache(2, 64, "mx8", pages_for(lens, 16))
    fill(cache, "mx8", 1)
    batch, states = batch_of(cache, lens, counts)
    q = rows(sum(counts), 4, 64, torch.bfloat16, 3)
    agrees(batch.attend(0, q, scale=scale), q, cache, "mx8", states, counts, 2.0 ** -8, scale=scale)
