"""Operators over a caller's paged cache (krasis_amd.kv_cache.KVBatch) against their definitions in 64 bits (tests/kv_reference.py)."""
import math
import random

import numpy as np
import pytest
import torch

from tests.kv_reference import DTYPES, attend, depths, make_cache, nearest, stored_rows, tolerance, values, visible

pytestmark = pytest.mark.gpu
FORMATS = ["bf16", "f16", "e4m3", "mx8", "mx4"]


def sequences(cache, lens, seed=0):
    """sequences of lens tokens over shuffled pages, none of them written"""
    from krasis_amd.kv_cache import SequenceKVState
    random.Random(seed).shuffle(cache._free_pages)
    out = []
    for i, n in enumerate(lens):
        s = SequenceKVState(cache, i); s.ensure_capacity(n); s.advance(n)
        out.append(s)
    return out


def rows(n, heads, dim, dtype, seed, key=True):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn((n, heads, dim), generator=g, device="cuda")
    if key and n:
        x *= torch.where(torch.rand((heads, dim), generator=g, device="cuda") < 0.05, 5.0, 1.0)
    return x.to(dtype)


def fill(cache, fmt, seed, spread=0):
    """pages of arbitrary numbers of the format; spread: scales over 2 spread + 1 powers of two"""
    g = torch.Generator(device="cuda").manual_seed(seed)
    for c, s in ((cache.k_cache, cache.k_scale), (cache.v_cache, cache.v_scale)):
        if fmt in ("bf16", "f16", "e4m3"):
            for l in range(c.shape[0]):
                c[l].copy_(torch.randn(c.shape[1:], generator=g, device="cuda").to(c.dtype))
        else:
            raw = torch.randint(0, 256, c.shape, generator=g, device="cuda", dtype=torch.uint8)
            if fmt == "mx8":
                raw = torch.where((raw & 127) == 127, raw ^ 64, raw)             # no NaN
                raw = torch.where((raw & 127) > 0x60, raw ^ 32, raw)             # at most 32 in magnitude
            c.view(torch.uint8).copy_(raw)
            s.copy_((torch.randint(-spread, spread + 1, s.shape, generator=g, device="cuda") + (127 - (4 if fmt == "mx8" else 1))).to(torch.uint8))


def stored_poison(cache, fmt, states):
    """everything that no sequence holds, the rest of last pages among it, becomes NaN"""
    page = cache.page_size
    used = torch.zeros((cache.max_pages, page), dtype=torch.bool)
    for s in states:
        for p in range(s.seq_len):
            used[s.pages[p // page], p % page] = True
    free = (~used).cuda()
    for c, s in ((cache.k_cache, cache.k_scale), (cache.v_cache, cache.v_scale)):
        for l in range(cache.num_layers):
            if s is not None:
                s[l][free] = 255
            if fmt in ("bf16", "f16"):
                c[l][free] = math.nan
            elif fmt != "mx4":
                c[l].view(torch.uint8)[free] = 127


def check(got, q, cache, fmt, states, counts, scale=None, window=0, first=0, trees=None, pieces=None):
    """every row of got against the definition over the pages as they are; states hold the new tokens already.  pieces: bits a weight is rounded to, None where it depends on the path"""
    heads, dim = q.shape[1], q.shape[2]
    scale = dim ** -0.5 if scale is None else scale
    native = fmt in ("bf16", "f16")
    r = 0
    assert got.shape == q.shape and got.dtype == q.dtype
    for i, (s, n) in enumerate(zip(states, counts)):
        if not n:
            continue
        k, v = stored_rows(cache, s, fmt)
        see = visible(s.seq_len - n, n, window, first, None if trees is None else trees[i])
        out, mean, size = attend(q[r:r + n].double(), k, v, see, scale)
        # weights are f16 over f16 pages, else bf16, one piece of it when q is bf16; half a step each.  Two pieces leave half a step of the second, 2^-8 of 2^-8.
        weight = 2.0 ** -8 if q.dtype == torch.bfloat16 else 2.0 ** -11 if native else 2.0 ** -16
        tol = tolerance(out, mean, size, dim, s.seq_len, q.dtype, weight)
        # 32 bits end at 2^-126: a weight under it is 0 (off by less than 2^-126 of its |v|), and so is a product of a weight and a value (off by less than 2^-126), for every key
        tol = tol + s.seq_len * 2.0 ** -126 * (v[v.isfinite()].abs().max() + 1)
        if fmt == "f16":                                              # weights below 2^-14 are subnormal numbers: half a step of those
            tol = tol + s.seq_len * 2.0 ** -25 * v[v.isfinite()].abs().max()
        x = got[r:r + n].double()
        bad = ~((x - out).abs() <= tol) & ~(x.isnan() & out.isnan()) & ~(x == out)
        assert not bad.any(), (i, n, s.seq_len, int(bad.sum()), bad.nonzero()[0].tolist(), float((x - out).abs().nan_to_num().max()), float(tol.max()))
        r += n
    assert r == got.shape[0]


# ---------------------------------------------------------------------------------------------------------------- rows in and out
def hard_rows(n, heads, dim, dtype, seed):
    """random rows over many magnitudes; blocks of ties, zeros of both signs, the largest and the smallest numbers, NaN and infinities"""
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn((n, heads, dim), generator=g, device="cuda") * torch.exp2(torch.randint(-12, 9, (n, heads, 1), generator=g, device="cuda").float())
    x = x.to(dtype)
    ties = torch.tensor([0.25, -0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -5.0, 6.0, 0.2490234375, 0.251953125, 4.984375, 5.03125, 0.0, -0.0, 1.0625, 1.1875, 17.0, 19.0, 0.0009765625, 0.0029296875,
                         448.0, -448.0, 432.0, 416.0, 464.0, 440.0, 0.001953125, -0.00390625, 3.0, 1.5], device="cuda").to(dtype)
    small = torch.finfo(dtype).smallest_normal
    x[0, 0, :32] = ties; x[0, -1, 32:64] = ties.flip(0) / 64
    x[1, 0, :32] = 0.0; x[1, 0, 5] = -0.0
    x[2, 0, :32] = small; x[2, 0, 3] = small / 4; x[2, -1, :32] = small / 8
    x[3, 0, :32] = torch.finfo(dtype).max / 4; x[3, 0, 7] = 1.0
    x[4, 0, :32] = torch.where(ties.abs() >= 448, torch.zeros_like(ties), ties)
    x[5, 0, 3] = math.nan; x[6, 0, 40] = math.inf; x[6, -1, 1] = -math.inf
    x[7, 0, :32] = 463.0; x[7, 0, 1] = 470.0; x[7, 0, 2] = -466.0; x[7, 0, 4] = 464.0
    return x


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("heads,dim,page", [(2, 64, 16), (3, 96, 5), (1, 256, 64)])
def test_rows_are_quantised_as_defined_and_read_back(fmt, dtype, heads, dim, page):
    from krasis_amd.kv_cache import KVBatch
    cache = make_cache(heads, dim, fmt, 400 // page, page, layers=2)
    states = sequences(cache, [3, 40, 0, 17])
    fill(cache, fmt, 1)
    counts = [9, 1, 30, 0]
    x, y = hard_rows(40, heads, dim, dtype, 2), hard_rows(40, heads, dim, dtype, 3).flip(0)
    was = [None if t is None else t.view(torch.uint8).clone() for t in (cache.k_cache, cache.v_cache, cache.k_scale, cache.v_scale)]
    batch = KVBatch(cache, states, counts)
    qkv = torch.cat([x, y, x], 1)                                   # rows as slices of one projection
    batch.write(1, qkv[:, :heads], qkv[:, heads:2 * heads])
    for out in (torch.bfloat16, torch.float16):
        k, v = batch.read(1, out)
        for got, given in ((k, x), (v, y)):
            want = nearest(given, fmt)
            want32 = want.float()                                   # every stored number is one of 32 bits
            assert torch.equal(want32.double().nan_to_num(), want.nan_to_num())
            assert torch.equal(got.nan_to_num(nan=7.0).double(), want32.to(out).nan_to_num(nan=7.0).double()), fmt
            assert torch.equal(got.isnan(), want.isnan())
    # the pages themselves stand for the same numbers, and nothing else in them has changed
    batch.commit()
    at = torch.cat([torch.arange(s.seq_len - n, s.seq_len) for s, n in zip(states, counts)])
    own = torch.zeros((cache.max_pages, page), dtype=torch.bool)
    r = 0
    for s, n in zip(states, counts):
        k, v = stored_rows(cache, s, fmt, layer=1)
        for got, given in ((k, x), (v, y)):
            assert torch.equal(got[s.seq_len - n:].nan_to_num(nan=7.0), nearest(given[r:r + n], fmt).nan_to_num(nan=7.0))
        for p in range(s.seq_len - n, s.seq_len):
            own[s.pages[p // page], p % page] = True
        r += n
    assert at.numel() == 40
    for t, old in zip((cache.k_cache, cache.v_cache, cache.k_scale, cache.v_scale), was):
        if t is not None:
            now = t.view(torch.uint8)
            assert torch.equal(now[0], old[0]) and torch.equal(now[1][~own.cuda()], old[1][~own.cuda()])


@pytest.mark.parametrize("fmt", ["e4m3", "mx8", "mx4"])
def test_every_code_and_scale_reads_as_its_number(fmt):
    from krasis_amd.kv_cache import KVBatch
    cache = make_cache(2, 64, fmt, 20)
    (s,) = sequences(cache, [256])
    codes = torch.arange(256, device="cuda", dtype=torch.uint8)
    width = cache.k_cache.shape[-1]
    for p in range(256):
        at = (0, s.pages[p // 16], p % 16)
        for t in (cache.k_cache, cache.v_cache):
            t.view(torch.uint8)[at] = codes.roll(-p)[:2 * width].view(2, width)
        if cache.k_scale is not None:
            cache.k_scale[at] = 27 + p % 220; cache.v_scale[at] = 255 if p == 9 else 127
    for out in (torch.bfloat16, torch.float16):
        got = KVBatch.stored(cache, [s]).read(0, out)
        for g, want in zip(got, stored_rows(cache, s, fmt)):
            assert torch.equal(g.isnan(), want.isnan())
            assert torch.equal(g.nan_to_num(nan=0.0, posinf=math.inf, neginf=-math.inf), want.float().to(out).nan_to_num(nan=0.0, posinf=math.inf, neginf=-math.inf))


# ---------------------------------------------------------------------------------------------------------------- attention
def run(fmt, dtype, heads, kv_heads, dim, lens, counts, page=16, window=0, first=0, trees=None, scale=None, seed=0, spread=0, alter=None, call=None):
    from krasis_amd.kv_cache import KVBatch
    cache = make_cache(kv_heads, dim, fmt, sum(-(-n // page) for n in lens) + 2, page)
    states = sequences(cache, [n - c for n, c in zip(lens, counts)], seed)
    fill(cache, fmt, seed + 1, spread)
    batch = KVBatch(cache, states, counts)
    q = rows(sum(counts), heads, dim, DTYPES[dtype], seed + 2)
    for s, c in zip(states, counts):
        s.advance(c)
    stored_poison(cache, fmt, states)
    if alter:
        alter(cache, states, q)
    if trees is None:
        got = batch.attend(0, q, scale=scale, window=window, keep_first=first)
    else:
        got = batch.attend_tree(0, q, trees, scale=scale, window=window, keep_first=first)
    check(got, q, cache, fmt, states, counts, scale, window, first, trees)
    if call:
        call(batch, q, got)


@pytest.mark.parametrize("fmt,dtype", [("bf16", "bf16"), ("f16", "f16"), ("e4m3", "bf16"), ("e4m3", "f16"), ("mx8", "bf16"), ("mx8", "f16"), ("mx4", "bf16"), ("mx4", "f16")])
@pytest.mark.parametrize("dim", [64, 96, 128, 192, 256])
def test_single_tokens_and_portions(fmt, dtype, dim):
    run(fmt, dtype, 8, 2, dim, [1, 33, 97, 300, 64, 5], [1, 1, 2, 1, 4, 0], spread=2)                     # at most 16 rows of a sequence
    run(fmt, dtype, 8, 2, dim, [70, 200, 129, 40], [70, 5, 64, 33], spread=2, seed=3)                     # more
    run(fmt, dtype, 3, 1, dim, [90, 31, 260, 1], [90, 1, 1, 1], page=5, spread=1, seed=5)                  # both, odd groups and pages


@pytest.mark.parametrize("window,first", [(1, 0), (1, 1), (7, 0), (64, 3), (65, 70), (100, 1), (1000, 4), (40, 100000), (2 ** 31 - 1, 2 ** 31 - 1)])
@pytest.mark.parametrize("fmt", ["mx8", "bf16"])
def test_windows_and_first_tokens(fmt, window, first):
    run(fmt, "bf16", 6, 2, 64, [1, 40, 300, 519, 260, 130], [1, 1, 1, 4, 200, 130], page=32, window=window, first=first)
    run(fmt, "bf16", 4, 4, 64, [700, 64], [130, 64], page=16, window=window, first=first, seed=4)


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (16, 1), (7, 1), (40, 2), (5, 5), (17, 1)])
def test_groups_of_heads(heads, kv_heads):
    run("mx4", "bf16", heads, kv_heads, 128, [50, 129, 1], [1, 40, 1], page=16)


def tree(n, seed):
    rng = random.Random(seed)
    return [-1 if i == 0 or rng.random() < 0.2 else rng.randint(max(0, i - 6), i - 1) for i in range(n)]


@pytest.mark.parametrize("window,first", [(0, 0), (1, 0), (5, 2), (40, 40), (300, 1)])
@pytest.mark.parametrize("fmt,dtype,dim", [("mx8", "bf16", 128), ("mx4", "f16", 64), ("f16", "f16", 256)])
def test_trees(fmt, dtype, dim, window, first):
    counts = [1, 12, 64, 33, 4, 0, 2]
    trees = [tree(n, 7 + n) for n in counts]
    trees[3] = list(range(-1, 32))                                  # a chain
    trees[4] = [-1, -1, -1, -1]
    run(fmt, dtype, 8, 2, dim, [1, 300, 64, 90, 130, 10, 66], counts, window=window, first=first, trees=trees)


def test_a_chain_of_drafts_is_a_portion():
    def both(batch, q, got):
        assert torch.equal(got, batch.attend(0, q))
        flat = torch.tensor([i - 1 for c in batch.counts for i in range(c)], dtype=torch.int32, device="cuda")
        assert torch.equal(got, batch.attend_tree(0, q, flat)) and torch.equal(got, batch.attend_tree(0, q, flat.cpu()))
        wrong = flat.clone(); wrong[0] = 5                          # no earlier draft: the token before them
        assert torch.equal(got, batch.attend_tree(0, q, wrong))
    run("mx8", "bf16", 8, 2, 128, [80, 30], [40, 30], trees=[list(range(-1, 39)), list(range(-1, 29))], call=both)


@pytest.mark.parametrize("fmt,dtype,dim,lens,counts,window", [
    ("mx4", "bf16", 128, [30011, 517, 9000], [1, 1, 1], 0), ("mx8", "f16", 256, [20003, 20], [1, 1], 0), ("e4m3", "bf16", 64, [33000], [17], 0), ("bf16", "bf16", 128, [8200, 3000], [30, 1], 0),
    ("mx8", "bf16", 96, [20001] * 3, [1, 2, 40], 9000)])
def test_long_sequences_are_shared_out_and_joined(fmt, dtype, dim, lens, counts, window):
    run(fmt, dtype, 8, 2, dim, lens, counts, page=64, window=window, first=3 if window else 0)


@pytest.mark.parametrize("counts", [[1, 2], [40, 64]])
@pytest.mark.parametrize("fmt,dtype", [("mx8", "bf16"), ("mx4", "f16"), ("f16", "f16"), ("bf16", "bf16"), ("e4m3", "f16")])
def test_values_that_are_not_finite_reach_the_rows_that_see_them_alone(fmt, dtype, counts):
    lens = [70, 90]

    def alter(cache, states, q):
        for s, n in zip(states, counts):
            for which, pos, bad in (("v", s.seq_len - 1, math.inf), ("v", s.seq_len - 2, math.nan), ("v", 11, -math.inf), ("k", s.seq_len - 1, math.nan), ("k", 3, math.inf), ("v", 12, math.nan)):
                at = (0, s.pages[pos // 16], pos % 16, 0)
                c, sc = (cache.k_cache, cache.k_scale) if which == "k" else (cache.v_cache, cache.v_scale)
                if sc is not None:
                    sc[at][-1] = 255
                elif fmt == "e4m3":
                    c.view(torch.uint8)[at][7] = 127
                else:
                    c[at][7] = bad
    run(fmt, dtype, 8, 2, 64, lens, counts, window=20, alter=alter)
    run(fmt, dtype, 8, 2, 64, lens, counts, window=20, first=4, alter=alter, seed=2)
    run(fmt, dtype, 8, 2, 64, lens, counts, trees=[tree(n, 5) for n in counts], alter=alter, seed=1)


def test_scores_far_apart_and_scales_far_from_one():
    def alter(cache, states, q):
        q.mul_(60.0)
        cache.v_scale.fill_(127 + 60); cache.v_scale[..., 1] = 127 - 60
    run("mx8", "bf16", 8, 2, 64, [200, 90], [1, 33], alter=alter)
    run("mx8", "f16", 8, 2, 128, [200, 90], [1, 33], scale=-0.25)


def test_slots_past_four_gigabytes():
    from krasis_amd.kv_cache import KVBatch
    page, pages = 64, 150000                                         # 9.6 million slots of 512 bytes
    cache = make_cache(4, 128, "e4m3", pages, page)
    cache._free_pages = list(range(pages))                           # the last ones first
    states = sequences_in_order(cache, [200, 70])
    x, y = rows(3 + 70, 4, 128, torch.bfloat16, 1), rows(3 + 70, 4, 128, torch.bfloat16, 2, key=False)
    for s in states:
        for p in s.pages:
            for c in (cache.k_cache, cache.v_cache):
                c[0, p].copy_(torch.randn((page, 4, 128), device="cuda"))
    states[1].seq_len = 0
    batch = KVBatch(cache, states, [3, 70])
    assert min(states[0].pages) * page * 512 > 2 ** 32
    batch.write(0, x, y)
    got = batch.read(0, torch.bfloat16)
    assert torch.equal(got[0].double(), nearest(x, "e4m3")) and torch.equal(got[1].double(), nearest(y, "e4m3"))
    q = rows(73, 8, 128, torch.bfloat16, 3)
    out = batch.attend(0, q)
    batch.commit()
    check(out, q, cache, "e4m3", states, [3, 70])


def sequences_in_order(cache, lens):
    from krasis_amd.kv_cache import SequenceKVState
    out = []
    for i, n in enumerate(lens):
        s = SequenceKVState(cache, i); s.ensure_capacity(n); s.advance(n)
        out.append(s)
    return out


# ---------------------------------------------------------------------------------------------------------------- as a program uses them
@pytest.mark.parametrize("fmt", ["mx8", "mx4", "e4m3"])
def test_prompts_portions_drafts_and_steps_together(fmt):
    """Three requests over two layers: a prompt in portions beside others' single tokens, drafts of which a path is kept, steps after it."""
    from krasis_amd.kv_cache import KVBatch, SequenceKVState
    layers, kvh, heads, dim = 2, 2, 8, 64
    cache = make_cache(kvh, dim, fmt, 200, 16, layers=layers)
    reqs = [SequenceKVState(cache, i) for i in range(3)]
    truth = [[([], []) for _ in reqs] for _ in range(layers)]         # rows given to write, by layer and request
    seed = 0

    def step(counts, trees=None, paths=None):
        nonlocal seed
        batch = KVBatch(cache, reqs, counts)
        for l in range(layers):
            seed += 3
            n = sum(counts)
            k, v, q = rows(n, kvh, dim, torch.bfloat16, seed), rows(n, kvh, dim, torch.bfloat16, seed + 1, key=False), rows(n, heads, dim, torch.bfloat16, seed + 2)
            batch.write(l, k, v)
            window, first = (0, 0) if l == 0 else (24, 2)
            got = batch.attend(l, q, window=window, keep_first=first) if trees is None else batch.attend_tree(l, q, trees, window=window, keep_first=first)
            r = 0
            for i, c in enumerate(counts):
                if c:
                    ks, vs = (torch.cat(x + [nearest(new[r:r + c], fmt)]) for x, new in zip(truth[l][i], (k, v)))
                    out, mean, size = attend(q[r:r + c].double(), ks, vs, visible(len(ks) - c, c, window, first, None if trees is None else trees[i]), dim ** -0.5)
                    tol = tolerance(out, mean, size, dim, len(ks), q.dtype, 2.0 ** -8)
                    assert bool(((got[r:r + c].double() - out).abs() <= tol).all()), (l, i, c)
                    path = range(c) if paths is None else paths[i]
                    for x, new in zip(truth[l][i], (k, v)):
                        x.append(nearest(new[r:r + c][list(path)], fmt))
                r += c
        batch.commit() if paths is None else batch.keep(paths)

    step([40, 1, 0]); step([33, 1, 20]); step([1, 1, 1])
    trees = [[-1, 0, 0, 2, -1, 3], [-1], [-1, -1, 1, 1, 3, 4, 2]]
    step([6, 1, 7], trees, [[0, 2, 3, 5], [], [1, 3, 4]])
    step([1, 1, 1]); step([1, 30, 1])
    assert [s.seq_len for s in reqs] == [80, 34, 26]
    for l in range(layers):
        for i, s in enumerate(reqs):
            k, v = stored_rows(cache, s, fmt, layer=l)
            assert torch.equal(k, torch.cat(truth[l][i][0])) and torch.equal(v, torch.cat(truth[l][i][1]))
    whole = KVBatch.stored(cache, reqs)
    k, v = whole.read(1, torch.bfloat16)
    assert torch.equal(k.double(), torch.cat([x for t in truth[1] for x in t[0]]).to(torch.bfloat16).double()) and v.shape == k.shape
    with pytest.raises(RuntimeError, match="already"):
        whole.commit()


def test_calls_into_a_graph_and_on_two_streams():
    from krasis_amd.kv_cache import KVBatch
    cache = make_cache(2, 128, "mx8", 1200, 16, layers=2)
    fill(cache, "mx8", 1)
    states = sequences(cache, [9000, 100, 400])
    counts = [1, 1, 40]
    batch = KVBatch(cache, states, counts)
    q, k, v = rows(42, 16, 128, torch.bfloat16, 2), rows(42, 2, 128, torch.bfloat16, 3), rows(42, 2, 128, torch.bfloat16, 4)

    def calls():
        batch.write(0, k, v)
        return batch.attend(0, q), batch.attend(0, q, window=50, keep_first=4), batch.read(0)[0]
    want = calls()
    assert all(torch.equal(a, b) for a, b in zip(want, calls()))       # equal bits every time
    graph, other = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        got = calls()
    with torch.cuda.graph(other):
        got2 = calls()
    for i in range(4):
        k.copy_(rows(42, 2, 128, torch.bfloat16, 10 + i)); q.copy_(rows(42, 16, 128, torch.bfloat16, 20 + i))
        graph.replay(); other.replay()
        torch.cuda.synchronize()
        want = calls()
        assert all(torch.equal(a, b) and torch.equal(a, c) for a, b, c in zip(want, got, got2)), i
    with pytest.raises(RuntimeError, match="before the capture"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            KVBatch(cache, states, counts)
    # two streams at once, each with shares to join
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    one, two = [], []
    for _ in range(5):
        with torch.cuda.stream(s1):
            one.append(batch.attend(0, q))
        with torch.cuda.stream(s2):
            two.append(batch.attend(0, q, window=50, keep_first=4))
    torch.cuda.synchronize()
    assert all(torch.equal(a, want[0]) for a in one) and all(torch.equal(a, want[1]) for a in two)


def test_a_microscaled_cache_is_handed_to_a_decoder():
    from krasis_amd.kv_cache import KVBatch, unpage_into_store
    cache = make_cache(2, 64, "mx8", 20, layers=3)
    fill(cache, "mx8", 1, spread=2)
    (s,) = sequences(cache, [37])

    class Store:
        def set_decode_state(self, *args): self.args = args
    store = Store()
    (k, v), = unpage_into_store(store, s, [None, 2], 64)
    assert store.args[0] == 37 and k.shape == (64, 128) and k.dtype == np.uint16
    want = stored_rows(cache, s, "mx8", layer=2)
    for got, w in zip((k, v), want):
        assert torch.equal(torch.from_numpy(got.view(np.float16)[:37]).double(), w.cpu().half().double().view(37, 128)) and not got[37:].any()


def test_refusals():
    from krasis_amd.kv_cache import KVBatch
    cache = make_cache(2, 64, "mx8", 20)
    (s,) = sequences(cache, [5])
    b = KVBatch(cache, [s], [3])
    ok = rows(3, 2, 64, torch.bfloat16, 1)
    for call, text in ((lambda: b.write(0, ok[:2], ok), "rows of 2 heads"), (lambda: b.write(0, ok, ok.half()), "k is"), (lambda: b.write(0, ok.float(), ok), "bfloat16 or float16"),
                       (lambda: b.write(0, ok.cpu(), ok), "cpu"), (lambda: b.write(1, ok, ok), "layer 1 of 1"), (lambda: b.read(0, torch.float32), "read as"),
                       (lambda: b.attend(0, rows(3, 3, 64, torch.bfloat16, 1)), "do not divide"), (lambda: b.attend(0, ok, window=-1), "window"),
                       (lambda: b.attend(0, ok, out=torch.empty_like(ok).half()), "out"), (lambda: b.attend_tree(0, ok, [-1, 1, 0]), "no earlier draft"),
                       (lambda: b.attend_tree(0, ok, [[-1, 0]]), "one number"), (lambda: b.attend_tree(0, ok, torch.zeros(3, device="cuda")), "int32"), (lambda: b.keep([[0, 3]]), "rising"),
                       (lambda: b.keep([[1, 1]]), "rising"), (lambda: b.attend(0, ok, scale=math.nan), "scale")):
        with pytest.raises(ValueError, match=text):
            call()
    assert s.seq_len == 5
    odd = torch.zeros(3 * 2 * 64 + 8, dtype=torch.bfloat16, device="cuda")[1:385].view(3, 2, 64)      # rows that begin anywhere, channels apart: copied
    odd.copy_(ok)
    b.write(0, odd, ok.transpose(1, 2).contiguous().transpose(1, 2))
    assert torch.equal(b.read(0, torch.bfloat16)[0].double(), nearest(ok, "mx8")) and torch.equal(b.read(0, torch.bfloat16)[1].double(), nearest(ok, "mx8"))
    assert torch.equal(b.attend(0, ok), b.attend(0, odd.view(3, 128)))
    b.commit()
    with pytest.raises(RuntimeError, match="already"):
        b.keep([[0]])
    empty = KVBatch(cache, [s], [0])
    assert empty.attend(0, ok[:0]).shape == (0, 2, 64) and empty.read(0)[0].shape == (0, 2, 64)
    empty.write(0, ok[:0], ok[:0]); KVBatch(cache, [], []).write(0, ok[:0], ok[:0])
    f = make_cache(2, 64, "f16", 20)
    (s,) = sequences(f, [5])
    with pytest.raises(ValueError, match="another 16-bit type"):
        KVBatch(f, [s], [3]).attend(0, ok)


def test_arguments_wider_than_the_librarys_are_refused():
    from krasis_amd.kv_cache import KVBatch
    cache = make_cache(2, 64, "mx8", 20)
    fill(cache, "mx8", 1)
    (s,) = sequences(cache, [5])
    b, q = KVBatch(cache, [s], [3]), rows(3, 2, 64, torch.bfloat16, 1)
    for window, first in ((2 ** 32 + 2, 0), (2, 2 ** 32), (2 ** 31, 0), (2, -1), (-2 ** 32 + 2, 0)):
        with pytest.raises(ValueError, match="window"):
            b.attend(0, q, window=window, keep_first=first)
        with pytest.raises(ValueError, match="window"):
            b.attend_tree(0, q, [-1, 0, 1], window=window, keep_first=first)
    assert torch.equal(b.attend(0, q), b.attend(0, q, window=2 ** 31 - 1, keep_first=2 ** 31 - 1))


@pytest.mark.parametrize("end", ["commit", "keep"])
def test_a_batch_ends_on_the_sequences_that_it_was_made_for(end):
    from krasis_amd.kv_cache import KVBatch
    cache = make_cache(2, 64, "mx8", 20)
    a, b = sequences(cache, [5, 7])
    one, two = KVBatch(cache, [a], [3]), KVBatch(cache, [a, b], [2, 1])      # both write a's places from 5 on
    one.commit()
    with pytest.raises(RuntimeError, match="has changed"):
        two.commit() if end == "commit" else two.keep([[0], [0]])
    assert (a.seq_len, b.seq_len) == (8, 7)
    late = KVBatch(cache, [b], [1])
    b.free()
    with pytest.raises(RuntimeError, match="has changed"):
        late.commit() if end == "commit" else late.keep([[0]])
    assert b.seq_len == 0


def test_paths_whose_move_was_refused_are_still_to_be_kept(monkeypatch):
    from krasis_amd.kv_cache import KVBatch
    cache = make_cache(2, 64, "mx8", 20)
    fill(cache, "mx8", 1)
    a, b = sequences(cache, [5, 7])
    batch, layer = KVBatch(cache, [a, b], [4, 2]), (cache.k_cache, cache.v_cache, cache.k_scale, cache.v_scale)
    slot = lambda s, p: (0, s.pages[p // 16], p % 16)
    want = [[t.view(torch.uint8)[slot(s, p)].clone() for s, p in ((a, 6), (a, 8), (b, 7))] for t in layer]

    def refuse(*args): raise ValueError("refused")
    with monkeypatch.context() as m:
        m.setattr(batch, "_call", refuse)
        with pytest.raises(ValueError, match="refused"):
            batch.keep([[1, 3], [0]])
    assert (a.seq_len, b.seq_len) == (5, 7)
    batch.keep([[1, 3], [0]])
    assert (a.seq_len, b.seq_len) == (7, 8)
    for t, rows_ in zip(layer, want):
        for got, w in zip((slot(a, 5), slot(a, 6), slot(b, 7)), rows_):
            assert torch.equal(t.view(torch.uint8)[got], w)
    for again in (batch.commit, lambda: batch.keep([[0], [0]])):
        with pytest.raises(RuntimeError, match="already"):
            again()
