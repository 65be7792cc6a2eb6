"""GPU parity of the paged cache's append and attention through the C ABI
against a plain 64-bit reference: element types, page sizes, head counts, ragged
batches with sequences that bring nothing, absent pages, rows that are never
read (all NaN in these pools)."""
import ctypes as C

import numpy as np
import pytest

from helpers import bits, device_arrays, log, max_err
from paged_ref import NAMES, NP, Batch, to_bits, to_f64, tla

pytestmark = pytest.mark.gpu

F32, F16, BF16 = tla.KV_F32, tla.KV_F16, tla.KV_BF16
TYPES = [pytest.param(t, id=NAMES[t]) for t in (F32, F16, BF16)]


def cfg_of(eng):
    return eng.cfg


# ---- append ------------------------------------------------------------------------

@pytest.mark.parametrize("ty", TYPES)
@pytest.mark.parametrize("heads,page,pos,n_tok", [
    ((32, 4), 16, [0], [1]),
    ((32, 4), 16, [15, 16, 0, 250], [1, 1, 0, 3]),
    ((16, 1), 1, [3, 0], [5, 2]),
    ((8, 8), 8, [5, 100], [70, 1]),
    ((12, 4), 256, [0, 255, 511], [300, 2, 1]),
    ((32, 4), 64, list(range(0, 130)), [i % 3 for i in range(130)]),
])
def test_append(O, engines, ty, heads, page, pos, n_tok):
    eng = engines(2, 2048, *heads)
    b = Batch(1, eng.cfg, ty, page, pos, n_tok, layer=1, gap=24)
    with b.on(eng) as (cache, a):
        eng.paged_append(cache, b.pos, b.n_tok, 1, a["k"].ptr, a["v"].ptr)
        b.append(O)
        assert np.array_equal(a["kp"].download(), b.kp) and np.array_equal(a["vp"].download(), b.vp)


@pytest.mark.parametrize("ty", TYPES)
def test_append_rounds_to_nearest_and_keeps_what_is_not_finite(engines, ty):
    """Ties, values between the largest element and infinity, subnormals, NaN."""
    eng = engines(1, 2048, 16, 1)
    b = Batch(2, eng.cfg, ty, 16, [0], [1])
    edge = np.array([1 + 2 ** -9, 1 + 3 * 2 ** -9, 1 + 2 ** -12, 1 + 3 * 2 ** -12, 65519.9, 65520, 3.39e38, -3.4e38, 1e-8,
                     2 ** -25, 3 * 2 ** -26, 1e-40, -0.0, np.inf, -np.inf, np.nan], np.float32)
    b.k[0], b.v[0] = np.resize(edge, 64), np.resize(edge[::-1], 64)
    with b.on(eng) as (cache, a):
        eng.paged_append(cache, b.pos, b.n_tok, 0, a["k"].ptr, a["v"].ptr, rotate=False)
        page = b.table[0, 0]
        for name, x in (("kp", b.k), ("vp", b.v)):
            got = a[name].download()[0, page, :64]
            want = to_bits(x[0], ty)
            nan = np.isnan(x[0])
            assert np.array_equal(got[~nan], want[~nan])
            assert np.isnan(to_f64(got[nan], ty)).all()


def test_append_leaves_absent_pages(O, engines):
    eng = engines(1, 2048)
    b = Batch(3, eng.cfg, F16, 16, [20, 10], [40, 30])
    for bad, at in ((-1, 2), (b.n_pages, 3), (2 ** 31 - 1, 1)):
        b.table[0, at] = bad
    b.table[1, 0] = -2 ** 31
    b.run(eng, O)


# ---- attention ---------------------------------------------------------------------

@pytest.mark.parametrize("ty", TYPES)
@pytest.mark.parametrize("page", [1, 4, 8, 16, 32, 64, 256, 1024])
def test_attention_page_sizes(O, engines, ty, page):
    """Single tokens and chunks whose ends lie anywhere in pages and tiles."""
    eng = engines(1, 2048)
    Batch(page, eng.cfg, ty, page, [0, 1, 15, 31, 32, 63, 64, 100, 257, 0, 30, 129],
          [1, 1, 1, 1, 1, 1, 1, 1, 1, 1 + 32, 3, 70]).check(eng, O)


@pytest.mark.parametrize("ty", TYPES)
@pytest.mark.parametrize("heads", [(32, 8), (8, 8), (16, 1), (12, 4), (4, 2), (14, 2)])
def test_attention_head_counts(O, engines, ty, heads):
    eng = engines(1, 2048, *heads)
    Batch(7, eng.cfg, ty, 16, [0, 77, 300, 5, 0, 500], [1, 1, 1, 2, 45, 130]).check(eng, O)


@pytest.mark.parametrize("ty", TYPES)
@pytest.mark.parametrize("n_tok", [1, 2, 3, 4, 5, 7, 8, 9, 15, 16, 17, 31, 33, 64, 65, 130])
def test_attention_chunk_lengths(O, engines, ty, n_tok):
    eng = engines(1, 2048)
    Batch(n_tok, eng.cfg, ty, 16, [0, 333], [n_tok, n_tok]).check(eng, O)


@pytest.mark.parametrize("ty", TYPES)
@pytest.mark.parametrize("pos,n_tok", [([4095], [1]), ([16383], [1]), ([9000, 100, 3000, 12345], [1, 1, 1, 1]),
                                       ([4000], [40]), ([2000, 1500], [100, 1])])
def test_attention_long(O, engines, ty, pos, n_tok):
    eng = engines(1, 16384)
    Batch(11, eng.cfg, ty, 64, pos, n_tok).check(eng, O)


@pytest.mark.parametrize("ty", TYPES)
def test_attention_many_sequences(O, engines, ty):
    """As many as a call takes; some bring nothing."""
    eng = engines(1, 2048, 8, 8)
    g = np.random.default_rng(5)
    pos = g.integers(0, 200, 256)
    n_tok = g.choice([0, 1, 1, 1, 2, 9], 256)
    Batch(13, eng.cfg, ty, 16, pos, n_tok).check(eng, O)


def test_nothing_to_do(O, engines):
    eng = engines(1, 2048)
    b = Batch(17, eng.cfg, F16, 16, [5, 9], [0, 0])
    assert b.check(eng, O).size == 0


@pytest.mark.parametrize("ty", TYPES)
def test_attention_without_rotation_on_the_second_layer(O, engines, ty):
    eng = engines(2, 2048)
    Batch(19, eng.cfg, ty, 16, [40, 3], [1, 20], layer=1, gap=40).check(eng, O, rotate=False)


@pytest.mark.parametrize("ty", TYPES)
@pytest.mark.parametrize("std", [8.0, 0.01])
def test_attention_peaked_and_flat(O, engines, ty, std):
    """Scores of hundreds (one key takes all) and of nearly nothing."""
    eng = engines(1, 2048)
    Batch(23, eng.cfg, ty, 32, [700, 0], [1, 90], std=std).check(eng, O)


@pytest.mark.parametrize("ty", TYPES)
@pytest.mark.parametrize("page", [4, 16, 64])
def test_attention_absent_pages(O, engines, ty, page):
    """Absent at the front (given back), in the middle, everywhere: a row that
    sees nothing is zero."""
    eng = engines(1, 2048)
    b = Batch(29, eng.cfg, ty, page, [300, 500, 200, 0, 260, 130], [1, 40, 1, 70, 1, 1])
    b.table[0, :100 // page] = -1
    b.table[1, 64 // page:256 // page] = b.n_pages
    b.table[2] = -1
    b.table[3, 0] = -5  # the chunk's own first page
    b.table[4, ::2] = 2 ** 31 - 1
    b.table[5, 130 // page] = -1  # the page of the new token alone
    got = b.check(eng, O)
    assert not got[b.tok[2]].any()
    assert not got[b.tok[3]:b.tok[3] + min(page, 64)].any()


@pytest.mark.parametrize("ty", TYPES)
@pytest.mark.parametrize("n_tok", [2, 6, 40])
def test_what_is_not_finite_reaches_only_those_who_see_it(O, engines, ty, n_tok):
    """A chunk whose token has infinite or NaN keys or values: earlier tokens do
    not see it, later ones get what fp32 gives."""
    eng = engines(1, 2048)
    h, g = eng.cfg.n_head, eng.cfg.n_head // eng.cfg.n_head_kv
    for what, x in (("v", np.nan), ("v", np.inf), ("k", np.nan), ("k", np.inf)):
        b = Batch(31, eng.cfg, ty, 16, [50], [n_tok])
        at = n_tok // 2
        clean = Batch(31, eng.cfg, ty, 16, [50], [n_tok])
        clean.append(O, rotate=False)
        want, bound = clean.attend(O, rotate=False)
        getattr(b, what)[at, 64 + 5] = x  # kv head 1
        log(f"  {what} = {x} at token {at} of {n_tok}")
        got = b.run(eng, O, rotate=False).reshape(n_tok, h, 64)
        want, bound = want.reshape(got.shape), bound.reshape(got.shape)
        hit = np.zeros(got.shape, bool)
        if what == "v":  # one dimension of the heads that share it
            hit[at:, g:2 * g, 5] = True
        else:  # an infinite score is either everything (NaN) or nothing
            hit[at:, g:2 * g] = True
        assert np.all(np.abs(got - want)[~hit] <= bound[~hit])
        if np.isnan(x):
            assert np.isnan(got[hit]).all()
        elif what == "v":
            assert np.all(got[hit] == np.inf)
        else:
            q = b.q.reshape(n_tok, h, 64)[at:, g:2 * g, 5]
            rows = got[at:, g:2 * g]
            assert np.isnan(rows[q > 0]).all()
            assert np.isfinite(rows[q < 0]).all()  # weight 0


def test_output_in_place_of_the_queries(O, engines):
    eng = engines(1, 2048)
    for n_tok in ([1, 1], [3, 50]):
        b = Batch(37, eng.cfg, F16, 16, [700, 20], n_tok)
        b.append(O)
        want, bound = b.attend(O)
        with b.on(eng) as (cache, a):
            eng.paged_attention(cache, b.pos, b.n_tok, 0, a["q"].ptr, a["q"].ptr)
            assert np.all(np.abs(a["q"].download() - want) <= bound)


@pytest.mark.parametrize("n_tok", [1, 40])
def test_output_in_place_of_the_queries_with_infinite_values(O, engines, n_tok):
    """Rows that are computed once more read their queries once more."""
    eng = engines(1, 2048)
    b = Batch(38, eng.cfg, F16, 16, [60], [n_tok])
    b.append(O)
    want, bound = b.attend(O)
    page, at = b.table[0, 0], 3 * b.kv + 64 + 5
    b.vp[0, page, at] = to_bits(np.array([np.inf]), F16)[0]
    with b.on(eng) as (cache, a):
        eng.paged_attention(cache, b.pos, b.n_tok, 0, a["q"].ptr, a["q"].ptr)
        got = a["q"].download()
    hit = np.zeros((n_tok, 32, 64), bool)
    hit[:, 8:16, 5] = True
    hit = hit.reshape(n_tok, -1)
    assert np.all(got[hit] == np.inf)
    assert np.all(np.abs(got - want)[~hit] <= bound[~hit])


def test_sequences_that_share_pages(O, engines):
    """Two sequences with a prefix in common, each with tokens of its own."""
    eng = engines(1, 2048)
    b = Batch(41, eng.cfg, BF16, 16, [64, 64], [1, 9])
    b.table[1, :4] = b.table[0, :4]
    b.check(eng, O)


def test_keys_and_values_of_a_page_side_by_side(O, engines):
    """One pool [page][2][rows]: both pointers into it, strides of two pages."""
    eng = engines(1, 2048)
    b = Batch(43, eng.cfg, F16, 16, [100, 31], [1, 5])
    n = 16 * b.kv
    both = np.concatenate([b.kp[0, :, None], b.vp[0, :, None]], 1)  # [page][2][n]
    b.append(O)
    want, bound = b.attend(O)
    with device_arrays() as track, b.on(eng) as (cache, a):
        pool = track(eng.array(both))
        cache.key_pages, cache.value_pages = pool.ptr, pool.ptr + 2 * n
        cache.page_stride, cache.layer_stride = 2 * n, 0
        eng.paged_append(cache, b.pos, b.n_tok, 0, a["k"].ptr, a["v"].ptr)
        eng.paged_attention(cache, b.pos, b.n_tok, 0, a["out"].ptr, a["q"].ptr)
        got = pool.download()
        assert np.array_equal(got[:, 0], b.kp[0]) and np.array_equal(got[:, 1], b.vp[0])
        assert np.all(np.abs(a["out"].download()[:b.total] - want) <= bound)


@pytest.mark.parametrize("ty", TYPES)
def test_pages_past_four_gigabytes(O, engines, ty):
    """A pool whose pages lie 512 MiB apart: offsets of more than 32 bits."""
    eng = engines(1, 2048)
    b = Batch(47, eng.cfg, ty, 64, [100, 290], [1, 30])
    b.append(O)
    want, bound = b.attend(O)
    es = NP[ty]().itemsize
    stride = (1 << 29) // es
    row = b.stride * es
    with device_arrays() as track, b.on(eng) as (cache, a):
        assert b.n_pages * (1 << 29) >= 5 << 30
        pools = []
        for host in (b.kp, b.vp):
            pool = track(tla.DeviceArray(eng, ((b.n_pages - 1) << 29 | row,), np.uint8))
            for i in range(b.n_pages):
                page = np.ascontiguousarray(host[0, i])
                assert tla.lib().tla_memcpy_h2d(eng.h, pool.ptr + (i << 29), page.ctypes.data, row) == 0
            pools.append(pool)
        cache.key_pages, cache.value_pages = pools[0].ptr, pools[1].ptr
        cache.page_stride, cache.layer_stride = stride, 0
        eng.paged_append(cache, b.pos, b.n_tok, 0, a["k"].ptr, a["v"].ptr)
        eng.paged_attention(cache, b.pos, b.n_tok, 0, a["out"].ptr, a["q"].ptr)
        assert np.all(np.abs(a["out"].download()[:b.total] - want) <= bound)


def test_same_as_the_contiguous_cache(engines):
    """F32 pages against tla_prefill and tla_decode: the same cache rows bit for
    bit, outputs within the two kernels' bounds."""
    eng = engines(1, 2048)
    b = Batch(53, eng.cfg, F32, 32, [0], [90])
    one = b.g.standard_normal((3, 2048)).astype(np.float32)
    with device_arrays() as track, b.on(eng) as (cache, a):
        kc, vc = eng.kv_cache(1)
        track(kc), track(vc)
        out = track(eng.array((90, 2048)))
        eng.prefill(0, 90, 0, 1, out.ptr, a["q"].ptr, a["k"].ptr, a["v"].ptr, kc.ptr, vc.ptr)
        eng.paged_append(cache, [0], [90], 0, a["k"].ptr, a["v"].ptr)
        eng.paged_attention(cache, [0], [90], 0, a["out"].ptr, a["q"].ptr)
        assert max_err(out.download(), a["out"].download()[:90]) <= 1e-5
        q, k, v = (track(eng.array(np.ascontiguousarray(x))) for x in (one[:1], one[1:2, :256], one[2:, :256]))
        eng.decode([90], 0, 1, out.ptr, q.ptr, k.ptr, v.ptr, kc.ptr, vc.ptr)
        eng.paged_append(cache, [90], None, 0, k.ptr, v.ptr)
        eng.paged_attention(cache, [90], None, 0, a["out"].ptr, q.ptr)
        assert max_err(out.download()[:1], a["out"].download()[:1]) <= 1e-5
        for pool, flat in ((a["kp"].download(), kc.download()), (a["vp"].download(), vc.download())):
            rows = pool[0, b.table[0, :3], :32 * 256].reshape(96, 256)[:91]
            assert np.array_equal(rows, bits(flat[0, 0, :91]))


def test_engines_side_by_side(O, engines):
    """Calls of two engines in flight together, each with its own workspaces."""
    first, second = engines(1, 16384), tla.Engine(tla.Config(1, 2048, 32, 4, 16384, 10000.0))
    try:
        b = [Batch(59 + i, first.cfg, F16, 64, [9000 - 1000 * i, 40], [1, 20]) for i in range(2)]
        for x in b:
            x.append(O)
        want = [x.attend(O) for x in b]
        with b[0].on(first) as (c0, a0), b[1].on(second) as (c1, a1):
            for _ in range(5):
                first.paged_attention(c0, b[0].pos, b[0].n_tok, 0, a0["out"].ptr, a0["q"].ptr)
                second.paged_attention(c1, b[1].pos, b[1].n_tok, 0, a1["out"].ptr, a1["q"].ptr)
            for a, x, (w, bound) in ((a0, b[0], want[0]), (a1, b[1], want[1])):
                assert np.all(np.abs(a["out"].download()[:x.total] - w) <= bound)
    finally:
        second.close()


def test_repeated_calls_give_the_same_bits(O, engines):
    """Whoever merges the parts of a long sequence, they are added in one order."""
    eng = engines(1, 16384)
    b = Batch(61, eng.cfg, F16, 16, [16000, 5000, 100], [1, 30, 1])
    b.append(O)
    with b.on(eng) as (cache, a):
        outs = []
        for _ in range(6):
            eng.paged_attention(cache, b.pos, b.n_tok, 0, a["out"].ptr, a["q"].ptr)
            outs.append(bits(a["out"].download()))
        assert all(np.array_equal(o, outs[0]) for o in outs)


# ---- what is refused ---------------------------------------------------------------

def test_cache_alloc(engines):
    eng = engines(2, 2048)
    c = eng.paged_cache(10, 32, tla.KV_BF16)
    assert (c.type, c.page_size, c.n_pages, c.page_stride, c.layer_stride) == (BF16, 32, 10, 32 * 256, 320 * 256)
    assert not c.table and c.table_stride == 0
    host = np.ones(2 * 320 * 256, np.uint16)
    for p in (c.key_pages, c.value_pages):
        assert tla.lib().tla_memcpy_d2h(eng.h, host.ctypes.data, p, host.nbytes) == 0
        assert not host.any()
    eng.free_paged_cache(c)
    for bad, code in (((0, 16, F16), tla.TLA_ERR_INVALID_ARGUMENT), ((4, 24, F16), tla.TLA_ERR_UNSUPPORTED),
                      ((4, 2048, F16), tla.TLA_ERR_UNSUPPORTED), ((4, 0, F16), tla.TLA_ERR_UNSUPPORTED),
                      ((4, 16, 2), tla.TLA_ERR_INVALID_ARGUMENT)):
        with pytest.raises(tla.TlaError) as err:
            eng.paged_cache(*bad)
        assert err.value.code == code


def test_refusals_launch_nothing(engines):
    eng = engines(1, 2048)
    b = Batch(67, eng.cfg, F16, 16, [20, 40], [1, 3])
    with b.on(eng) as (cache, a):
        def both(code, change=None, pos=None, n_tok=None, layer=0, off=0, flags=0, n_seq=2, null=()):
            c = tla.PagedCache.from_buffer_copy(cache)
            for k, v in (change or {}).items():
                setattr(c, k, v)
            p = np.asarray(b.pos if pos is None else pos, np.int32)
            n = np.asarray(b.n_tok if n_tok is None else n_tok, np.int32)
            args = (eng.h, None if "cache" in null else C.byref(c), n_seq, None if "pos" in null else p.ctypes.data,
                    n.ctypes.data, layer, flags)
            x = None if "x" in null else a["k"].ptr + off
            y = None if "y" in null else a["v"].ptr
            assert tla.lib().tla_paged_append(*args, x, y) == code, tla.last_error()
            x = None if "x" in null else a["out"].ptr + off
            y = None if "y" in null else a["q"].ptr
            assert tla.lib().tla_paged_attention(*args, x, y) == code, tla.last_error()

        inv, rng, uns = tla.TLA_ERR_INVALID_ARGUMENT, tla.TLA_ERR_OUT_OF_RANGE, tla.TLA_ERR_UNSUPPORTED
        for null in ("cache", "pos", "x", "y"):
            both(inv, null=(null,))
        for field in ("key_pages", "value_pages", "table"):
            both(inv, {field: None})
        both(inv, {"key_pages": cache.key_pages + 8})
        both(inv, {"value_pages": cache.value_pages + 2})
        both(inv, {"type": 2})
        both(uns, {"page_size": 24})
        both(uns, {"page_size": 2048})
        both(uns, {"page_size": 0})
        both(inv, {"n_pages": 0})
        both(inv, {"table_stride": 0})
        both(inv, {"page_stride": 16 * 256 - 8})
        both(inv, {"page_stride": 16 * 256 + 4})
        both(inv, {"layer_stride": 12})
        both(inv, {"page_stride": 1 << 60})
        both(inv, n_seq=0)
        both(inv, n_seq=257)
        both(inv, flags=2)
        both(inv, n_tok=[1, -1])
        both(rng, layer=1)
        both(rng, layer=-1)
        both(rng, pos=[-1, 4])
        both(rng, pos=[2048, 4])
        both(rng, {"table_stride": 2}, pos=[20, 32])
        both(rng, pos=[2 ** 31 - 1, 4])
        both(inv, off=4)
        assert np.array_equal(a["kp"].download(), b.kp) and np.array_equal(a["vp"].download(), b.vp)
        assert np.all(a["out"].download() == 7.0)
        with pytest.raises(ValueError):
            eng.paged_append(cache, [1, 2], [1], 0, a["k"].ptr, a["v"].ptr)
