"""The 4-bit cache's C interface and binding without a GPU: what they export, the sizes they report and the calls they refuse.

The addresses here are made up: a call that is not refused ends at the launch, which needs a GPU.  So none of this runs where there is one."""
import importlib
import os
import re

import pytest
import torch

import __graft_entry__ as entry

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
pytestmark = pytest.mark.skipif(torch.cuda.is_available(), reason="made-up addresses")



def code(name):
    text = open(os.path.join(ROOT, "include", "homcomp.h")).read()
    return int(re.search(rf"\b{name}\s*=?\s*\(?(-?\d+)", text).group(1))


OK, INVALID, ALIGNMENT, HIP = (code("HOMCOMP_" + n) for n in ("OK", "ERR_INVALID_ARG", "ERR_ALIGNMENT", "ERR_HIP"))


@pytest.fixture(scope="module")
def cache(pkg):
    return importlib.import_module(entry.PKG_NAME + ".cache")


def header():
    text = open(os.path.join(ROOT, "include", "homcomp_cache.h")).read()
    return re.sub(r"/\*.*?\*/", "", text, flags=re.S)


def test_header_binding_and_library_agree(cache):
    declared = sorted(set(re.findall(r"\b(homcomp_cache_[a-z0-9_]+)\s*\(", header())))
    assert declared == sorted(cache.EXPORTS)
    assert [s for s in declared if not hasattr(cache.lib(), s)] == []


@pytest.mark.parametrize("heads,d,page,want", [
    (1, 64, 32, 2560), (8, 128, 64, 8 * 2 * 5120), (3, 256, 65536, 3 * 2048 * 10240), (1024, 64, 32, 1024 * 2560),
    (0, 64, 32, 0), (1025, 64, 32, 0), (-1, 64, 32, 0), (1, 96, 32, 0), (1, 512, 32, 0), (1, 0, 32, 0),
    (1, 64, 16, 0), (1, 64, 48, 0), (1, 64, 131072, 0), (1, 64, 0, 0), (1, 64, -32, 0)])
def test_page_bytes(cache, heads, d, page, want):
    assert cache.lib().homcomp_cache_page_bytes(heads, d, page) == want
    if not want:
        with pytest.raises(ValueError):
            cache.page_bytes(heads, d, page)


AT = 1 << 20   # an address aligned to anything


def the_cache(cache, **kw):
    f = dict(pages=AT, n_pages=10, kv_heads=2, head_dim=64, page_tokens=32, n_seqs=3, table=AT, table_stride=4, lengths=AT)
    assert set(kw) <= set(f)
    return cache._CACHE.pack(*{**f, **kw}.values())


def attention(cache, **kw):
    f = dict(q=AT, q_row_stride=256, q_head_stride=64, out=2 * AT, out_row_stride=256, out_head_stride=64, type=0, q_heads=4, starts=AT, n_rows=5,
             max_rows=5, max_length=128, scale=0.125, causal=1, window=0, lse=0, prior=0, weights=0, weight_stride=0, scratch=0, scratch_bytes=0)
    assert set(kw) <= set(f)
    return cache._ATTENTION.pack(*{**f, **kw}.values())


def eviction(cache, **kw):
    f = dict(weights=AT, weight_stride=128, max_length=128, keep=64, first=2, recent=3, to_table=2 * AT, to_table_stride=2, to_lengths=3 * AT,
             to_weights=4 * AT, kept=5 * AT)
    assert set(kw) <= set(f)
    return cache._EVICTION.pack(*{**f, **kw}.values())


BAD_CACHES = [
    (dict(pages=0), INVALID), (dict(pages=AT + 8), ALIGNMENT), (dict(n_pages=1 << 31), INVALID), (dict(kv_heads=0), INVALID),
    (dict(head_dim=80), INVALID), (dict(page_tokens=40), INVALID), (dict(n_seqs=-1), INVALID), (dict(n_seqs=65536), INVALID),
    (dict(table=0), INVALID), (dict(table=AT + 2), ALIGNMENT), (dict(lengths=0), INVALID), (dict(lengths=AT + 1), ALIGNMENT),
    (dict(table_stride=1 << 27), INVALID), (dict(table_stride=(1 << 64) - 1), INVALID)]


def rows_call(cache, name, c, k=AT, v=2 * AT, type=0, row_stride=128, head_stride=64, starts=AT, n_rows=5):
    return getattr(cache.lib(), name)(c, k, v, type, row_stride, head_stride, starts, n_rows, 0)


@pytest.mark.parametrize("name", ["homcomp_cache_store", "homcomp_cache_load"])
@pytest.mark.parametrize("kw,want", [
    (dict(k=0), INVALID), (dict(v=0), INVALID), (dict(starts=0), INVALID), (dict(type=3), INVALID), (dict(type=-1), INVALID),
    (dict(k=AT + 1), ALIGNMENT), (dict(v=2 * AT + 2, type=2), ALIGNMENT), (dict(starts=AT + 2), ALIGNMENT),
    (dict(n_rows=1 << 31), INVALID), (dict(n_rows=(1 << 64) - 1), INVALID), (dict(n_rows=0), OK)])
def test_rows_refused(cache, name, kw, want):
    assert rows_call(cache, name, the_cache(cache), **kw) == want


def test_load_into_one_array_refused(cache):
    assert rows_call(cache, "homcomp_cache_load", the_cache(cache), v=AT) == INVALID


@pytest.mark.parametrize("kw,want", BAD_CACHES)
def test_bad_caches_refused(cache, kw, want):
    c, L = the_cache(cache, **kw), cache.lib()
    assert rows_call(cache, "homcomp_cache_store", c) == want
    assert rows_call(cache, "homcomp_cache_load", c) == want
    assert L.homcomp_cache_attend(c, attention(cache, scratch=AT, scratch_bytes=1 << 40), 0) == want
    assert L.homcomp_cache_evict(c, eviction(cache), 0) == want


def test_calls_beyond_a_launch_are_refused(cache):
    L, much = cache.lib(), dict(n_seqs=65535, kv_heads=1024)
    c, scratch = the_cache(cache, **much), dict(scratch=AT, scratch_bytes=1 << 60)
    assert L.homcomp_cache_attend(c, attention(cache, q_heads=1024, **scratch), 0) == INVALID
    assert L.homcomp_cache_evict(c, eviction(cache), 0) == INVALID
    assert rows_call(cache, "homcomp_cache_store", c) == INVALID
    few = the_cache(cache, n_seqs=1, kv_heads=64)
    assert rows_call(cache, "homcomp_cache_load", few, n_rows=(1 << 31) - 1) == INVALID
    assert L.homcomp_cache_attend(few, attention(cache, q_heads=64, n_rows=1 << 24, max_rows=1 << 24, **scratch), 0) == INVALID
    assert L.homcomp_cache_evict(the_cache(cache, n_seqs=16000, kv_heads=64),
                                 eviction(cache, keep=1 << 20, to_table_stride=1 << 15), 0) == INVALID


def test_null_structures_refused(cache):
    L = cache.lib()
    assert rows_call(cache, "homcomp_cache_store", None) == INVALID
    assert L.homcomp_cache_attend(None, attention(cache), 0) == L.homcomp_cache_attend(the_cache(cache), None, 0) == INVALID
    assert L.homcomp_cache_evict(None, eviction(cache), 0) == L.homcomp_cache_evict(the_cache(cache), None, 0) == INVALID
    assert L.homcomp_cache_attend_scratch(None, attention(cache)) == L.homcomp_cache_attend_scratch(the_cache(cache), None) == 0


@pytest.mark.parametrize("kw,want", [
    (dict(type=3), INVALID), (dict(q_heads=0), INVALID), (dict(q_heads=3), INVALID), (dict(q_heads=2 * 257), INVALID), (dict(q_heads=-2), INVALID),
    (dict(n_rows=1 << 30), INVALID), (dict(n_rows=4, max_rows=5), INVALID), (dict(scale=float("nan")), INVALID), (dict(scale=float("inf")), INVALID),
    (dict(q=0), INVALID), (dict(out=0), INVALID), (dict(out=AT), INVALID), (dict(starts=0), INVALID), (dict(starts=AT + 1), ALIGNMENT),
    (dict(q=AT + 1), ALIGNMENT), (dict(out=2 * AT + 2, type=2), ALIGNMENT), (dict(lse=AT + 2), ALIGNMENT), (dict(lse=2 * AT), INVALID),
    (dict(weights=3 * AT, weight_stride=127), INVALID), (dict(weights=3 * AT + 1, weight_stride=128), ALIGNMENT),
    (dict(weights=3 * AT, weight_stride=128, lse=3 * AT), INVALID),
    (dict(prior=3 * AT, weight_stride=128), INVALID), (dict(weights=3 * AT, prior=4 * AT + 2, weight_stride=128), ALIGNMENT)])
def test_attention_refused(cache, kw, want):
    kw = {"scratch": 7 * AT, "scratch_bytes": 1 << 40, **kw}
    assert cache.lib().homcomp_cache_attend(the_cache(cache), attention(cache, **kw), 0) == want


def test_attention_scratch(cache):
    L, c = cache.lib(), the_cache(cache, table_stride=64)
    kw = dict(max_length=2048, weights=3 * AT, weight_stride=2048)
    need = L.homcomp_cache_attend_scratch(c, attention(cache, **kw))
    assert need > 0
    for more in (dict(), dict(scratch=7 * AT), dict(scratch=7 * AT, scratch_bytes=need - 1)):
        assert L.homcomp_cache_attend(c, attention(cache, **kw, **more), 0) == INVALID
    assert L.homcomp_cache_attend(c, attention(cache, **kw, scratch=7 * AT + 8, scratch_bytes=need), 0) == ALIGNMENT
    # a short cache is one part, and with lse given nothing is needed
    assert L.homcomp_cache_attend_scratch(the_cache(cache, table_stride=1), attention(cache, max_length=32, max_rows=1, n_rows=3)) == 0
    assert L.homcomp_cache_attend_scratch(c, attention(cache, **kw, type=9)) == 0


@pytest.mark.parametrize("kw,want", [
    (dict(keep=0), INVALID), (dict(keep=65), INVALID), (dict(keep=1 << 40, to_table_stride=1 << 40), INVALID), (dict(first=60, recent=5), INVALID),
    (dict(first=(1 << 64) - 1, recent=2), INVALID), (dict(recent=(1 << 64) - 1), INVALID), (dict(weight_stride=127), INVALID),
    (dict(weights=0), INVALID), (dict(to_table=0), INVALID), (dict(to_lengths=0), INVALID), (dict(to_weights=0), INVALID), (dict(kept=0), INVALID),
    (dict(to_lengths=AT), INVALID), (dict(to_table=AT), INVALID), (dict(to_weights=AT), INVALID), (dict(kept=AT), INVALID), (dict(kept=4 * AT), INVALID),
    (dict(weights=AT + 4 + 2), ALIGNMENT), (dict(to_table=2 * AT + 1), ALIGNMENT), (dict(to_lengths=3 * AT + 2), ALIGNMENT),
    (dict(to_weights=4 * AT + 2), ALIGNMENT), (dict(kept=5 * AT + 3), ALIGNMENT)])
def test_eviction_refused(cache, kw, want):
    assert cache.lib().homcomp_cache_evict(the_cache(cache), eviction(cache, **kw), 0) == want


def test_no_sequences_do_nothing(cache):
    c, L = the_cache(cache, n_seqs=0, pages=0, table=0, lengths=0), cache.lib()
    assert rows_call(cache, "homcomp_cache_store", c) == rows_call(cache, "homcomp_cache_load", c) == OK
    assert L.homcomp_cache_attend(c, attention(cache), 0) == L.homcomp_cache_evict(c, eviction(cache), 0) == OK


def test_no_cpu_fallback(cache, pkg):
    assert rows_call(cache, "homcomp_cache_store", the_cache(cache)) == HIP
    assert cache.lib().homcomp_cache_attend(the_cache(cache), attention(cache, max_rows=1, scratch=7 * AT, scratch_bytes=1 << 40), 0) == HIP
    assert cache.lib().homcomp_cache_evict(the_cache(cache), eviction(cache), 0) == HIP


# ---------------------------------------------------------------- the binding
class Call:
    def __init__(self, cache):
        self.c = cache.Cache(torch.zeros(4, cache.page_bytes(2, 64, 32), dtype=torch.uint8), 2, 64, 32)
        self.args = dict(table=torch.zeros(2, 2, dtype=torch.int32), lengths=torch.zeros(2, dtype=torch.int32), starts=torch.zeros(3, dtype=torch.int32))
        self.k, self.v = torch.zeros(5, 2, 64), torch.zeros(5, 2, 64)
        self.q, self.out = torch.zeros(5, 4, 64), torch.zeros(5, 4, 64)

    def store(self, **kw):
        self.c.store(**{"k": self.k, "v": self.v, **self.args, **kw})

    def load(self, **kw):
        self.c.load(**{"k": self.k, "v": self.v, **self.args, **kw})

    def attend(self, **kw):
        self.c.attend(**{"q": self.q, "out": self.out, **self.args, **kw})

    def evict(self, **kw):
        a = dict(weights=torch.zeros(2, 2, 64), table=self.args["table"], lengths=self.args["lengths"], keep=32, to_table=torch.ones(2, 1, dtype=torch.int32),
                 to_lengths=torch.zeros(2, dtype=torch.int32))
        return self.c.evict(**{**a, **kw})


def I(*shape):
    return torch.zeros(*shape, dtype=torch.int32)


@pytest.mark.parametrize("pages", [torch.zeros(4, 5120), torch.zeros(5119, dtype=torch.uint8), torch.zeros(10240, dtype=torch.uint8)[::2]])
def test_pages_refused(cache, pages):
    with pytest.raises(ValueError):
        cache.Cache(pages, 2, 64, 32)


def test_a_cache_on_the_cpu_is_refused(cache):
    call = Call(cache)
    for f in (call.store, call.load, call.attend, call.evict):
        with pytest.raises(ValueError, match="GPU"):
            f()


COMMON = [dict(table=I(3, 2)), dict(table=I(2, 2).long()), dict(table=I(2, 4)[:, ::2]), dict(table=I(4)), dict(lengths=I(3)), dict(lengths=I(2).float()),
          dict(lengths=I(2, 1)), dict(lengths=I(2).to("meta"))]
STARTS = [dict(starts=I(2)), dict(starts=I(4)), dict(starts=I(3).long()), dict(starts=I(6)[::2])]


@pytest.mark.parametrize("kw", COMMON + STARTS + [
    dict(k=torch.zeros(5, 3, 64)), dict(k=torch.zeros(5, 2, 32)), dict(k=torch.zeros(5, 128)), dict(k=torch.zeros(5, 2, 64).bfloat16()),
    dict(k=torch.zeros(4, 2, 64)), dict(k=torch.zeros(5, 2, 128)[:, :, ::2]), dict(v=torch.zeros(5, 4, 64)[:, ::2]), dict(v=torch.zeros(5, 2, 64).to("meta"))])
def test_binding_refuses_rows(cache, kw):
    for f in (Call(cache).store, Call(cache).load):
        with pytest.raises(ValueError, match="^(?!.*GPU)"):
            f(**kw)


def test_binding_refuses_types_and_shared_memory(cache):
    call = Call(cache)
    with pytest.raises(TypeError):
        call.store(k=torch.zeros(5, 2, 64).double(), v=torch.zeros(5, 2, 64).double())
    one = torch.zeros(1, 2, 64).expand(5, 2, 64)
    with pytest.raises(ValueError, match="of its own"):
        call.load(k=one, v=one)
    with pytest.raises(ValueError, match="of its own"):
        call.attend(out=torch.zeros(5, 1, 64).expand(5, 4, 64))
    with pytest.raises(ValueError, match="GPU"):
        call.store(k=one, v=one)      # (reading one row several times is fine)


W = torch.zeros(2, 2, 64)


@pytest.mark.parametrize("kw", COMMON + STARTS + [
    dict(q=torch.zeros(5, 3, 64)), dict(q=torch.zeros(5, 256)), dict(q=torch.zeros(5, 4, 128)), dict(out=torch.zeros(5, 4, 64).half()),
    dict(out=torch.zeros(4, 4, 64)), dict(out=torch.zeros(5, 4, 64).to("meta")), dict(lse=torch.zeros(5, 2)), dict(lse=torch.zeros(4, 5).t()),
    dict(lse=torch.zeros(5, 4).double()), dict(prior=W), dict(weights=W[:, :, :63]), dict(weights=W[:1]), dict(weights=W.half()),
    dict(weights=torch.zeros(2, 2, 128)[:, :, ::2]), dict(weights=W, prior=torch.zeros(2, 2, 65)), dict(weights=torch.zeros(64)),
    dict(max_rows=-1), dict(max_length=-1), dict(window=-1), dict(weights=W, scratch=torch.zeros(5000).to("meta")),
    dict(weights=W, scratch=torch.zeros(5000)[::2])])
def test_binding_refuses_attention(cache, kw):
    with pytest.raises(ValueError, match="^(?!.*GPU)"):
        Call(cache).attend(**kw)


@pytest.mark.parametrize("kw", COMMON + [
    dict(keep=0), dict(keep=33), dict(first=-1), dict(recent=-1), dict(first=30, recent=3), dict(max_length=-1), dict(to_table=I(3, 1)),
    dict(to_table=I(2, 1).long()), dict(to_lengths=I(3)), dict(to_lengths=I(2).long()), dict(weights=W[:, :, :63]), dict(weights=W.double()),
    dict(weights=W[:, :1]), dict(to_weights=torch.zeros(2, 2, 31)), dict(to_weights=I(2, 2, 32)), dict(kept=torch.zeros(2, 2, 32)),
    dict(kept=I(2, 32, 2).transpose(1, 2))])
def test_binding_refuses_eviction(cache, kw):
    with pytest.raises(ValueError, match="^(?!.*GPU)"):
        Call(cache).evict(**kw)
