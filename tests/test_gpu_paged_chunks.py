"""GPU parity of paged attention's long chunks (more query rows than are
streamed past the keys: 4096 for a kv head) and of long sequences in small pages,
against the plain 64-bit reference."""
import numpy as np
import pytest

from paged_ref import NAMES, Batch, to_bits, tla

pytestmark = pytest.mark.gpu

F32, F16, BF16 = tla.KV_F32, tla.KV_F16, tla.KV_BF16
TYPES = [pytest.param(t, id=NAMES[t]) for t in (F32, F16, BF16)]
N = 260  # tokens of 16 heads on one kv head: 4160 rows


@pytest.mark.parametrize("ty", TYPES)
@pytest.mark.parametrize("page", [1, 2, 4, 8, 16, 64, 512])
def test_chunk_page_sizes(O, engines, ty, page):
    """A prompt from its beginning, and a chunk that begins inside a page."""
    eng = engines(1, 4096, 16, 1)
    Batch(101, eng.cfg, ty, page, [0, 37], [N, N + 9]).check(eng, O)


@pytest.mark.parametrize("ty,heads,n_tok", [(F32, (14, 2), 600), (F16, (14, 2), 600), (BF16, (14, 2), 600),
                                            (F32, (12, 4), 1367), (F16, (12, 4), 1367), (BF16, (12, 4), 1367),
                                            (F16, (8, 8), 4097)])
def test_chunk_head_counts(O, engines, ty, heads, n_tok):
    """Rows of 7, 3 and 1 heads to a token: tiles of 128 that end inside one."""
    eng = engines(1, 8192, *heads)
    Batch(103, eng.cfg, ty, 32, [21], [n_tok]).check(eng, O)


@pytest.mark.parametrize("ty", TYPES)
@pytest.mark.parametrize("page", [4, 16])
def test_chunks_whose_keys_are_shared_out(O, engines, ty, page):
    """Long contexts, in parts whose states are added, beside short ones."""
    eng = engines(1, 4096, 16, 1)
    Batch(107, eng.cfg, ty, page, [3500, 1000, 0], [N, 0, N]).check(eng, O)


@pytest.mark.parametrize("ty", TYPES)
@pytest.mark.parametrize("page", [8, 16, 64])
@pytest.mark.parametrize("singles", [3, 70])
def test_chunks_beside_single_tokens(O, engines, ty, page, singles):
    """In one launch (pages of 16 and more, up to 64 sequences) and in two."""
    eng = engines(1, 4096, 16, 1)
    pos = np.random.default_rng(109).integers(0, 900, singles)
    Batch(109, eng.cfg, ty, page, [*pos, 700], [*([1] * singles), N]).check(eng, O)


@pytest.mark.parametrize("ty", TYPES)
@pytest.mark.parametrize("page", [4, 16, 64])
def test_chunk_absent_pages(O, engines, ty, page):
    eng = engines(1, 4096, 16, 1)
    b = Batch(113, eng.cfg, ty, page, [500, 0, 300, 2000], [N, N, N, N])
    b.table[0, :192 // page] = -1
    b.table[1, 0] = -5  # the chunk's own first page
    b.table[2, 64 // page:384 // page] = b.n_pages
    b.table[3] = -1
    got = b.check(eng, O)
    assert not got[b.tok[1]:b.tok[1] + page].any()
    assert not got[b.tok[3]:].any()


@pytest.mark.parametrize("ty", TYPES)
@pytest.mark.parametrize("page", [4, 16])
@pytest.mark.parametrize("what,x", [("v", np.nan), ("v", np.inf), ("k", np.nan), ("k", np.inf)])
def test_chunk_with_what_is_not_finite(O, engines, ty, page, what, x):
    """A token in the chunk's middle with an infinite or NaN element: earlier
    tokens do not see it, later ones get what fp32 gives."""
    eng = engines(1, 4096, 16, 1)
    clean = Batch(127, eng.cfg, ty, page, [50], [N])
    clean.append(O, rotate=False)
    want, bound = clean.attend(O, rotate=False)
    b = Batch(127, eng.cfg, ty, page, [50], [N])
    at = 133
    getattr(b, what)[at, 5] = x
    got = b.run(eng, O, rotate=False).reshape(N, 16, 64)
    want, bound = want.reshape(got.shape), bound.reshape(got.shape)
    hit = np.zeros(got.shape, bool)
    hit[at:, :, 5 if what == "v" else slice(None)] = True
    assert np.all(np.abs(got - want)[~hit] <= bound[~hit])
    if np.isnan(x):
        assert np.isnan(got[hit]).all()
    elif what == "v":
        assert np.all(got[hit] == np.inf)
    else:
        q = b.q.reshape(N, 16, 64)[at:, :, 5]
        assert np.isnan(got[at:][q > 0]).all()
        assert np.isfinite(got[at:][q < 0]).all()


@pytest.mark.parametrize("ty", TYPES)
@pytest.mark.parametrize("infinite", [False, True])
def test_chunk_output_in_place_of_the_queries(O, engines, ty, infinite):
    eng = engines(1, 4096, 16, 1)
    b = Batch(131, eng.cfg, ty, 16, [1500, 30], [N, 1])
    b.append(O)
    want, bound = b.attend(O)
    hit = np.zeros((b.total, 16, 64), bool)
    if infinite:
        b.vp[0, b.table[0, 0], 3 * b.kv + 5] = to_bits(np.array([np.inf]), ty)[0]
        hit[:N, :, 5] = True
    hit = hit.reshape(b.total, -1)
    with b.on(eng) as (cache, a):
        eng.paged_attention(cache, b.pos, b.n_tok, 0, a["q"].ptr, a["q"].ptr)
        got = a["q"].download()
    assert np.all(got[hit] == np.inf)
    assert np.all(np.abs(got - want)[~hit] <= bound[~hit])


@pytest.mark.parametrize("ty", TYPES)
@pytest.mark.parametrize("std", [8.0, 0.01])
def test_chunk_peaked_and_flat(O, engines, ty, std):
    """Running maxima that move by hundreds, and that hardly move."""
    eng = engines(1, 4096, 16, 1)
    Batch(137, eng.cfg, ty, 32, [700], [N], std=std).check(eng, O)


@pytest.mark.parametrize("ty", TYPES)
def test_chunk_scores_that_grow(O, engines, ty):
    """Each tile's largest score far above the one before."""
    eng = engines(1, 4096, 16, 1)
    b = Batch(139, eng.cfg, ty, 16, [0], [N])
    b.q[:] = np.abs(b.q)
    b.k[:] = np.abs(b.k) * np.linspace(0.01, 12.0, N, dtype=np.float32)[:, None]
    b.check(eng, O, rotate=False)


@pytest.mark.parametrize("ty", TYPES)
@pytest.mark.parametrize("page", [1, 2, 4, 8])
def test_long_sequences_in_small_pages(O, engines, ty, page):
    """Keys in parts, every row of a tile looked up by itself; some are absent."""
    eng = engines(1, 8192)
    b = Batch(149, eng.cfg, ty, page, [7000, 33, 4095, 2500], [1, 1, 2, 9])
    b.table[0, 100:300] = -1
    b.table[2, ::3] = b.n_pages
    b.check(eng, O)


@pytest.mark.parametrize("ty", TYPES)
@pytest.mark.parametrize("n_tok", [1, 5, N])
@pytest.mark.parametrize("q,k,v", [(1, 1, 1e-6), (1, 1, 5e4), (1e-3, 1e-5, 1), (3e3, 1e-3, 1), (1e-20, 5e3, 1), (1e20, 1e-4, 1)])
def test_sizes_at_the_ends_of_the_types(O, engines, ty, n_tok, q, k, v):
    """F16's subnormal and largest values, and queries far outside F16's range."""
    eng = engines(1, 4096, 16, 1)
    b = Batch(151, eng.cfg, ty, 16, [200], [n_tok])
    for s, p in enumerate(b.pos):
        b.put(s, 0, b.g.standard_normal((p, b.kv)) * k, np.clip(b.g.standard_normal((p, b.kv)), -1.3, 1.3) * v)
    b.q *= np.float32(q)
    b.k *= np.float32(k)
    b.v = np.clip(b.v, -1.3, 1.3) * np.float32(v)
    b.check(eng, O)


@pytest.mark.parametrize("ty", TYPES)
@pytest.mark.parametrize("n_tok", [1, 5, N])
@pytest.mark.parametrize("x", [np.nan, np.inf])
def test_a_query_that_is_not_finite_stays_alone(O, engines, ty, n_tok, x):
    """Its row is NaN (an infinite one meets keys of both signs), its tile's others are
    as they were."""
    eng = engines(1, 4096, 16, 1)
    b = Batch(157, eng.cfg, ty, 16, [90], [n_tok])
    b.append(O, rotate=False)
    want, bound = b.attend(O, rotate=False)
    b.q[n_tok // 2, 3 * 64 + 7] = x
    got = b.run(eng, O, append=False, rotate=False).reshape(n_tok, 16, 64)
    hit = np.zeros(got.shape, bool)
    hit[n_tok // 2, 3] = True
    assert np.isnan(got[hit]).all()
    assert np.all(np.abs(got - want.reshape(got.shape))[~hit] <= bound.reshape(got.shape)[~hit])
