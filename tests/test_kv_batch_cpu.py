"""Operators over a caller's paged cache without a GPU: the plan of a step, the geometry of the microscaled pages, and what is refused before anything is launched."""
import ctypes

import pytest
import torch

from tests.kv_reference import Heads, make_cache


def states(cache, lens):
    from krasis_amd.kv_cache import SequenceKVState
    out = []
    for i, n in enumerate(lens):
        s = SequenceKVState(cache, i); s.ensure_capacity(n); s.advance(n)
        out.append(s)
    return out


@pytest.mark.parametrize("page", [1, 5, 16, 64])
def test_a_plan_lists_every_new_row(page):
    from krasis_amd.kv_cache import plan_of
    cache = make_cache(2, 64, "e4m3", 400 // page + 8, page, device="cpu")
    a, b, c, e = states(cache, [37, 0, 16, 5])
    a.free(); a.ensure_capacity(21); a.advance(21)                 # pages out of order
    counts = [7, 1, 0, 33]
    for s, n in zip((a, b, c, e), counts):
        s.ensure_capacity(n)
    plan = plan_of(cache, [a, b, c, e], counts).tolist()
    assert plan[:6] == [4, 41, plan[2], page, cache.max_pages, 1]
    row0, rest = plan[8:13], plan[13:]
    assert row0 == [0, 7, 8, 8, 41]
    lens, page0, rest = rest[:4], rest[4:8], rest[8:]
    assert lens == [28, 1, 16, 38]
    pages, slots = rest[:plan[2]], rest[plan[2]:]
    want = []
    for s, n, at, new in zip((a, b, c, e), lens, page0, counts):
        held = -(-n // page)
        assert pages[at:at + held] == s.pages[:held]
        want += [s.pages[p // page] * page + p % page for p in range(n - new, n)]
    assert slots == want


def test_plans_that_share_a_page_to_be_written_say_so():
    from krasis_amd.kv_cache import plan_of
    cache = make_cache(2, 64, "mx8", 16, device="cpu")
    a, b = states(cache, [20, 20])
    b.pages[0] = a.pages[0]                                         # a shared prefix: not written
    assert plan_of(cache, [a, b], [4, 4])[5] == 1
    b.pages[1] = a.pages[1]
    assert plan_of(cache, [a, b], [4, 4])[5] == 0
    assert plan_of(cache, [], []).tolist()[:2] == [0, 0]


@pytest.mark.parametrize("change,text", [(lambda a: a.pages.__setitem__(0, 16), "lists page 16 of 16"), (lambda a: a.pages.__setitem__(1, -1), "lists page -1"),
                                         (lambda a: a.pages.pop(), "in 1 pages")])
def test_plans_refuse_bad_pages(change, text):
    from krasis_amd.kv_cache import plan_of
    cache = make_cache(2, 64, "mx8", 16, device="cpu")
    (a,) = states(cache, [20])
    change(a)
    with pytest.raises(ValueError, match=text):
        plan_of(cache, [a], [4])


def test_microscaled_caches():
    from krasis_amd.kv_cache import KVBatch, PagedKVCache, unpage_into_store
    m8, m4 = make_cache(2, 96, "mx8", 10, layers=3, device="cpu"), make_cache(2, 96, "mx4", 10, layers=3, device="cpu")
    assert m8.k_cache.shape == (3, 10, 16, 2, 96) and m8.k_cache.dtype == torch.float8_e4m3fn and m8.k_scale.shape == m4.v_scale.shape == (3, 10, 16, 2, 3)
    assert m4.v_cache.shape == (3, 10, 16, 2, 48) and m4.v_cache.dtype == torch.uint8 and m4.kv_dtype == torch.uint8
    assert m8._bytes_per_page() == 3 * 16 * 2 * 2 * (96 + 3) and m4._bytes_per_page() == 3 * 16 * 2 * 2 * (48 + 3)
    assert make_cache(2, 96, "e4m3", 10, device="cpu").k_scale is None
    for bad in (dict(kv_format="mx6"), dict(kv_format="mx8", dim=80)):
        with pytest.raises(ValueError, match="kv_format"):
            PagedKVCache(Heads(2, bad.pop("dim", 64)), 1, "cpu", max_pages=4, **bad)
    (s,) = states(m8, [5])
    with pytest.raises(ValueError, match="scales"):
        s.unpage(m8.k_cache[0])

    class Store:
        _kv_fp8 = True
    with pytest.raises(ValueError, match="FP16"):
        unpage_into_store(Store(), s, [0], 64)
    with pytest.raises(Exception, match="no CPU fallback"):
        KVBatch(m8, [s], [1])
    assert s.seq_len == 5 and len(s.pages) == 1


def test_batches_refuse_what_does_not_fit():
    from krasis_amd.kv_cache import KVBatch
    cache, other = make_cache(2, 64, "mx8", 8, device="cpu"), make_cache(2, 64, "mx8", 8, device="cpu")
    a, b = states(cache, [20, 3])
    (x,) = states(other, [3])
    for args, kind, text in ((([a], [1, 2]), ValueError, "1 sequences, 2 counts"), (([a], [-1]), ValueError, "negative"), (([a, x], [1, 1]), ValueError, "another cache"),
                             (([a, a], [1, 1]), ValueError, "twice"), (([a, b], [100, 100]), RuntimeError, r"KV cache exhausted: need \d+ pages, have \d+")):
        with pytest.raises(kind, match=text):
            KVBatch(cache, *args)
    assert cache.free_page_count == 5 and len(a.pages) == 2


def c_call(**over):
    """kr_kv_attend on pointers that are never followed"""
    from krasis_amd import _lib
    lib = _lib.load_library()
    cache = make_cache(2, over.pop("dim", 64), "mx8", 1024, device="cpu")
    a, b = states(cache, [20, 16000])
    from krasis_amd.kv_cache import plan_of
    new = over.pop("new", 1)
    b.ensure_capacity(new)
    plan = plan_of(cache, [a, b], [1, new])
    pages = _lib.KvPagesC(4096, 4096, 4096, 4096, 3, 16, 1024, 2, cache.gqa_head_dim)
    for k in ("format", "page_tokens", "n_pages", "kv_heads", "k", "k_scale"):
        if k in over:
            setattr(pages, k, over.pop(k))
    g = dict(q=4096, qt=256, qh=64, out=4096, dtype=0, heads=4, scale=0.1, window=0, first=0, parents=None, ws=4096, bytes=0)
    g.update(over)
    _lib.check(lib.kr_kv_attend(ctypes.byref(pages), plan.data_ptr(), 4096, g["q"], g["qt"], g["qh"], g["out"], g["dtype"], g["heads"], g["scale"], g["window"], g["first"], g["parents"],
                                g["ws"], g["bytes"], 1))


@pytest.mark.parametrize("over,text", [
    (dict(format=9), "unknown page format"), (dict(format=0), "scales belong"), (dict(k_scale=None), "scales belong"), (dict(k=4100), "aligned"), (dict(k=None), "aligned"),
    (dict(page_tokens=32), "the plan is for"), (dict(n_pages=17), "the plan is for"), (dict(kv_heads=0), "heads"), (dict(dim=32), "heads of 32 channels"), (dict(heads=3), "do not divide"),
    (dict(heads=0), "do not divide"), (dict(window=-1), "window"), (dict(first=-2), "keep_first"), (dict(dtype=2), "bf16 or f16"), (dict(scale=float("nan")), "scale"), (dict(q=4104), "aligned"),
    (dict(out=None), "aligned"), (dict(qt=100), "multiples of 8"), (dict(parents=4096, new=65), "65 drafts"),
    (dict(heads=32), "a workspace of 0 bytes")])
def test_attention_refuses(over, text):
    with pytest.raises(ValueError, match=text):
        c_call(**dict(over))


def test_pages_of_another_16_bit_type_are_refused():
    with pytest.raises(ValueError, match="another 16-bit type"):
        c_call16()


def c_call16():
    from krasis_amd import _lib
    from krasis_amd.kv_cache import plan_of
    cache = make_cache(2, 64, "f16", 16, device="cpu")
    plan = plan_of(cache, states(cache, [20]), [1])
    pages = _lib.KvPagesC(4096, 4096, None, None, 1, 16, 16, 2, 64)
    _lib.check(_lib.load_library().kr_kv_attend(ctypes.byref(pages), plan.data_ptr(), 4096, 4096, 256, 64, 4096, 0, 4, 0.1, 0, 0, None, None, 0, 1))


def test_rows_of_a_plan_that_shares_slots_are_not_written():
    from krasis_amd import _lib
    from krasis_amd.kv_cache import plan_of
    cache = make_cache(2, 64, "f16", 16, device="cpu")
    a, b = states(cache, [20, 20])
    b.pages[1] = a.pages[1]
    plan, strides = plan_of(cache, [a, b], [2, 2]), (ctypes.c_int64 * 4)(128, 64, 128, 64)
    pages = _lib.KvPagesC(4096, 4096, None, None, 1, 16, 16, 2, 64)
    with pytest.raises(ValueError, match="one slot"):
        _lib.check(_lib.load_library().kr_kv_write(ctypes.byref(pages), plan.data_ptr(), 4096, 4096, 4096, strides, 0, 1))
    plan = plan_of(cache, [a], [2])
    for args, text in (((4100, 4096, strides, 0), "aligned"), ((4096, 4096, (ctypes.c_int64 * 4)(100, 64, 128, 64), 0), "multiples of 8"), ((4096, 4096, strides, 3), "bf16 or f16")):
        with pytest.raises(ValueError, match=text):
            _lib.check(_lib.load_library().kr_kv_write(ctypes.byref(pages), plan.data_ptr(), 4096, *args, 1))


def test_workspaces_grow_with_the_shares():
    from krasis_amd import _lib
    from krasis_amd.kv_cache import plan_of
    cache = make_cache(2, 128, "mx4", 4096, device="cpu")
    pages, size = _lib.KvPagesC(4096, 4096, 4096, 4096, 4, 16, 4096, 2, 128), ctypes.c_size_t()
    short, long = states(cache, [90, 60000])
    long.ensure_capacity(40)

    def need(st, cnt, heads, window=0, tree=0):
        plan = plan_of(cache, st, cnt)
        _lib.check(_lib.load_library().kr_kv_attend_workspace(ctypes.byref(pages), plan.data_ptr(), heads, 0, window, 4, tree, ctypes.byref(size)))
        return size.value
    assert need([short], [1], 16) == 0 and need([long], [1], 16) > 0 and need([long], [40], 16, tree=1) > 0
    assert need([long], [1], 16, window=32) == 0


def test_sequences_may_write_to_different_slots_of_a_page():
    from krasis_amd.kv_cache import plan_of
    cache = make_cache(2, 64, "mx8", 16, device="cpu")
    a, b = states(cache, [20, 26])
    b.pages[1] = a.pages[1]                                         # a's rows at 4 and 5 of the page, b's at 10 and 11
    assert plan_of(cache, [a, b], [2, 2])[5] == 1
    assert plan_of(cache, [a, b], [7, 2])[5] == 0                   # a's at 4 to 10
    a.pages = tuple(a.pages)
    assert plan_of(cache, [a], [2])[5] == 1


def test_a_callers_own_cache_object_is_unpaged_as_before():
    from krasis_amd.kv_cache import SequenceKVState, unpage_into_store
    made = make_cache(2, 64, "f16", 8, device="cpu")

    class Own:                                                      # the surface that these two read, without what PagedKVCache has gained
        page_size, attention_type, kv_dtype, combined = made.page_size, "gqa", torch.float16, False
        k_cache, v_cache = made.k_cache, made.v_cache
        alloc_pages = made.alloc_pages

        def get_gqa_layer_caches(self, off): return self.k_cache[off], self.v_cache[off]
    made.k_cache.copy_(torch.arange(made.k_cache.numel()).view(made.k_cache.shape) % 1000)
    s = SequenceKVState(Own(), 0); s.ensure_capacity(20); s.advance(20)
    want = torch.stack([made.k_cache[0, s.pages[p // 16], p % 16].flatten() for p in range(20)])
    assert torch.equal(s.unpage(made.k_cache[0]), want)

    class Store:
        def set_decode_state(self, *args): self.args = args
    store = Store()
    (k, v), = unpage_into_store(store, s, [None, 0], 32)
    assert store.args[0] == 20 and torch.equal(torch.from_numpy(k.view("float16"))[:20], want) and not v.any()


def test_plans_are_made_on_the_host_whatever_the_default_device():
    from krasis_amd.kv_cache import plan_of
    cache = make_cache(2, 64, "mx8", 16, device="cpu")
    st = states(cache, [20, 5])
    want = plan_of(cache, st, [3, 2])
    with torch.device("meta"):                                      # a device whose addresses are 0: nothing is followed that is not there
        got = plan_of(cache, st, [3, 2])
    assert got.device.type == "cpu" and torch.equal(got, want)


@pytest.mark.parametrize("scale", [2.5e38, -3e38, float("inf")])
def test_scales_that_end_the_numbers_are_refused(scale):
    with pytest.raises(ValueError, match="scale"):
        c_call(scale=scale)
