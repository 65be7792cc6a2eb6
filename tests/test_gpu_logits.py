"""GPU parity of the rules on logits: bit for bit against the same operations in
numpy, each rounded to fp32 on its own, and the token that is left on top."""
import ctypes as C

import numpy as np
import pytest

from helpers import bits, device_arrays, tla

pytestmark = pytest.mark.gpu


def reference(x, hist=None, n_hist=None, pen=None, bt=None, bv=None, nb=None, mask=None):
    x = x.astype(np.float32).copy()
    n, nv = x.shape
    with np.errstate(all="ignore"):
        for s in range(n):
            if hist is not None:
                h = hist[s, :min(max(n_hist[s], 0), hist.shape[1])].astype(np.int64)
                count = np.bincount(h[(h >= 0) & (h < nv)], minlength=nv).astype(np.float32)
                r, a, f = pen[s]
                y = np.where(x[s] > 0, x[s] / r, x[s] * r)
                y = y - (count * f + a)
                x[s] = np.where(count > 0, y, x[s])
            if bt is not None:
                last = {int(t): v for t, v in zip(bt[s, :min(max(nb[s], 0), bt.shape[1])], bv[s])}
                for t, v in last.items():
                    if 0 <= t < nv:
                        x[s, t] = x[s, t] + v
            if mask is not None:
                j = np.arange(nv)
                x[s, (mask[s, j // 32] >> (j % 32).astype(np.uint32)) & 1 == 0] = -np.inf
    tokens = np.full(n, -1, np.int32)
    for s in range(n):
        live = np.nonzero(x[s] > -np.inf)[0]  # neither -inf nor NaN
        if live.size:
            tokens[s] = live[np.argmax(x[s, live])]
    return x, tokens


def run(eng, x, hist=None, n_hist=None, pen=None, bt=None, bv=None, nb=None, mask=None, in_place=False):
    n, nv = x.shape
    with device_arrays() as track:
        d = lambda a, t: track(eng.array(np.ascontiguousarray(a, t))).ptr  # noqa: E731
        rules = tla.LogitRules()
        if hist is not None:
            rules.history, rules.history_len, rules.history_stride = d(hist, np.int32), d(n_hist, np.int32), hist.shape[1]
            rules.penalties = d(pen, np.float32)
        if bt is not None:
            rules.bias_token, rules.bias_value, rules.bias_len = d(bt, np.int32), d(bv, np.float32), d(nb, np.int32)
            rules.bias_stride = bt.shape[1]
        if mask is not None:
            rules.mask, rules.mask_stride = d(mask, np.uint32), mask.shape[1]
        src = track(eng.array(x))
        out = src if in_place else track(eng.array(np.full((n + 1, nv), 7.0, np.float32)))
        tok = track(eng.array(np.full(n + 1, -7, np.int32)))
        print(f"  logits {n} x {nv} history={hist is not None} biases={bt is not None} mask={mask is not None}", flush=True)
        eng.logits_process(n, nv, rules, out.ptr, src.ptr, tok.ptr)
        got, t = out.download(), tok.download()
        if not in_place:
            assert np.all(got[n:] == 7.0)
            assert np.array_equal(bits(src.download()), bits(x))
        assert t[n] == -7
        return got[:n], t[:n]


def same(got, want):
    """Equal bits, any NaN for a NaN."""
    nan = np.isnan(want)
    assert np.array_equal(np.isnan(got), nan)
    assert np.array_equal(bits(got)[~nan], bits(want)[~nan])


def inputs(seed, n, nv, nh=0, nb=0, mask=False):
    g = np.random.default_rng(seed)
    a = {"x": (g.standard_normal((n, nv)) * 3).astype(np.float32)}
    if nh:
        # few words, often; some numbers that are none
        a["hist"] = g.integers(-2, max(2, min(nv, nh // 3) + 2), (n, nh)).astype(np.int32)
        a["hist"][g.random((n, nh)) < 0.05] = 2 ** 31 - 1
        a["n_hist"] = g.integers(-1, nh + 2, n).astype(np.int32)
        a["pen"] = (g.random((n, 3)) * [0.5, 1, 0.5] + [1, 0, 0]).astype(np.float32)
    if nb:
        a["bt"] = g.integers(-1, nv + 1, (n, nb)).astype(np.int32)
        a["bt"][:, nb // 2:] = a["bt"][:, :nb - nb // 2]  # every token twice
        a["bv"] = (g.standard_normal((n, nb)) * 5).astype(np.float32)
        a["nb"] = g.integers(-1, nb + 2, n).astype(np.int32)
    if mask:
        words = (nv + 31) // 32 + 1
        a["mask"] = g.integers(0, 2 ** 32, (n, words), dtype=np.uint64).astype(np.uint32)
        a["mask"][::3] &= a["mask"][::3] >> 1 & 0x11111111
        a["mask"][n // 2] = 0
    return a


@pytest.mark.parametrize("nv", [1, 5, 31, 33, 1000, 4095, 4096, 4097, 32000, 32003, 100003])
@pytest.mark.parametrize("nh,nb,mask", [(0, 0, False), (700, 0, False), (0, 50, False), (0, 0, True), (300, 40, True)])
def test_rules(engines, nv, nh, nb, mask):
    eng = engines(1, 2048)
    for n in (1, 5):
        a = inputs(nv + nh, n, nv, nh, nb, mask)
        got, tok = run(eng, **a)
        want, best = reference(**a)
        same(got, want)
        assert np.array_equal(tok, best)


def test_long_histories_and_many_rows(engines):
    eng = engines(1, 2048)
    for n, nv, nh in ((3, 32000, 40000), (300, 999, 64), (64, 32000, 2048)):
        a = inputs(n, n, nv, nh, 20, True)
        got, tok = run(eng, **a)
        want, best = reference(**a)
        same(got, want)
        assert np.array_equal(tok, best)


def test_in_place(engines):
    eng = engines(1, 2048)
    a = inputs(3, 4, 5001, 100, 10, True)
    got, tok = run(eng, in_place=True, **a)
    want, best = reference(**a)
    same(got, want)
    assert np.array_equal(tok, best)


def test_ties_nans_and_infinities(engines):
    """The first of equal ones; a NaN never wins; -0 ties with +0; -inf is nothing."""
    eng = engines(1, 2048)
    nv = 9000
    x = np.full((8, nv), -1.0, np.float32)
    x[0, [4000, 8000, 77]] = 5.0
    x[1, 0] = np.nan
    x[1, 8999] = 3.0
    x[2] = np.nan
    x[3] = -np.inf
    x[4, 3] = -0.0
    x[4, 9] = 0.0
    x[5, 100] = np.inf
    x[5, 4100] = np.inf
    x[6] = -np.inf
    x[6, 8000] = -3.4e38
    x[7, :] = -0.0
    x[7, 5000] = 0.0
    got, tok = run(eng, x)
    same(got, x)
    assert tok.tolist() == [77, 8999, -1, -1, 3, 100, 8000, 0]


def test_penalties_at_their_ends(engines):
    """A repetition penalty of 0 or infinity, infinite logits and biases, as the formula gives."""
    eng = engines(1, 2048)
    nv = 64
    x = np.tile(np.array([2.0, -2.0, 0.0, np.inf, -np.inf, np.nan, -0.0, 1e-40], np.float32), (4, 8))
    hist = np.tile(np.arange(32, dtype=np.int32), (4, 2))
    pen = np.array([[0, 0, 0], [np.inf, 0, 1], [1.5, -np.inf, 0], [1, 0.1, 0.2]], np.float32)
    bt = np.tile(np.arange(3, 64, 7, dtype=np.int32), (4, 1))
    bv = np.tile(np.array([np.inf, -np.inf, 1], np.float32), (4, 3))
    a = dict(x=x, hist=hist, n_hist=np.full(4, 64, np.int32), pen=pen, bt=bt, bv=bv, nb=np.full(4, 9, np.int32))
    got, tok = run(eng, **a)
    want, best = reference(**a)
    same(got, want)
    assert np.array_equal(tok, best)
    assert nv == 64


def test_without_rules_or_tokens(engines):
    eng = engines(1, 2048)
    x = np.random.default_rng(1).standard_normal((3, 5000)).astype(np.float32)
    with device_arrays() as track:
        src, out, tok = track(eng.array(x)), track(eng.array(x.shape)), track(eng.array(np.zeros(3, np.int32)))
        eng.logits_process(3, 5000, None, out.ptr, src.ptr)
        assert np.array_equal(bits(out.download()), bits(x))
        eng.logits_process(3, 5000, None, out.ptr, src.ptr, tok.ptr)
        assert np.array_equal(tok.download(), x.argmax(-1))
        for s in range(3):
            assert eng.argmax(src.at(4 * 5000 * s), 5000) == int(tok.download()[s])


def test_repeated_calls(engines):
    """Arrival counters return to zero: calls of other shapes in between."""
    eng = engines(1, 2048)
    a, b = inputs(5, 6, 32000, 100, 10, True), inputs(6, 40, 5000, 50, 0, False)
    for _ in range(4):
        for c in (a, b):
            got, tok = run(eng, **c)
            want, best = reference(**c)
            same(got, want)
            assert np.array_equal(tok, best)


def test_refusals(engines):
    eng = engines(1, 2048)
    inv, uns = tla.TLA_ERR_INVALID_ARGUMENT, tla.TLA_ERR_UNSUPPORTED
    with device_arrays() as track:
        x = track(eng.array(np.full((2, 100), 7.0, np.float32)))
        p = x.ptr

        def call(code, n=2, nv=100, out=p, logits=p, **rules):
            r = tla.LogitRules(**rules)
            assert tla.lib().tla_logits_process(eng.h, n, nv, C.byref(r), out, logits, None) == code, tla.last_error()

        call(inv, n=0)
        call(inv, nv=0)
        call(uns, n=65537)
        call(uns, nv=2 ** 28 + 1)
        call(uns, n=65536, nv=2 ** 28)
        call(inv, out=None)
        call(inv, logits=None)
        call(inv, history=p, history_stride=4, penalties=p)
        call(inv, history=p, history_stride=4, history_len=p)
        call(inv, history=p, history_len=p, penalties=p)
        call(inv, bias_token=p, bias_value=p, bias_stride=3)
        call(inv, bias_token=p, bias_len=p, bias_stride=3)
        call(inv, bias_token=p, bias_value=p, bias_len=p)
        call(inv, mask=p, mask_stride=3)
        assert np.all(x.download() == 7.0)
        assert tla.lib().tla_logits_process(None, 1, 1, None, p, p, None) == inv
