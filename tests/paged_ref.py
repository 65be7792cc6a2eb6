"""Plain 64-bit reference of the paged operators, and the pools and page
tables that their tests run on."""
import contextlib
import importlib

import numpy as np
import torch

tla = importlib.import_module("tinyllama-engine_amd")

U = 2.0 ** -24  # half a step of fp32, relative
NP = {tla.KV_F32: np.uint32, tla.KV_F16: np.uint16, tla.KV_BF16: np.uint16}  # elements as bits
NAN = {tla.KV_F32: 0x7fc00000, tla.KV_F16: 0x7e00, tla.KV_BF16: 0x7fc0}
NAMES = {tla.KV_F32: "f32", tla.KV_F16: "f16", tla.KV_BF16: "bf16"}
TORCH = {tla.KV_F32: torch.float32, tla.KV_F16: torch.float16, tla.KV_BF16: torch.bfloat16}


def to_bits(x, ty):
    """fp32 values as element bits, rounded to nearest even."""
    t = torch.from_numpy(np.ascontiguousarray(x, np.float32)).to(TORCH[ty])
    if ty == tla.KV_F32:
        return t.numpy().view(np.uint32)
    return t.view(torch.int16).numpy().view(np.uint16)


def to_f64(bits, ty):
    if ty == tla.KV_F32:
        return bits.view(np.float32).astype(np.float64)
    if ty == tla.KV_F16:
        return bits.view(np.float16).astype(np.float64)
    return (bits.astype(np.uint32) << 16).view(np.float32).astype(np.float64)


def same_bits(a, b, ty):
    """Equal bits, any NaN for a NaN."""
    off = a != b
    return np.isnan(to_f64(a[off], ty)).all() and np.isnan(to_f64(b[off], ty)).all()


class Batch:
    """Sequences over pages: tables of distinct pages in random order, pools
    [n_layers][n_pages][page_stride] of element bits in host memory, every row
    NaN but those of positions below pos (values of numpy's generator)."""

    def __init__(self, seed, cfg, ty, page, pos, n_tok, layer=0, gap=0, spare=3, extra_cols=1, std=1.0):
        g = self.g = np.random.default_rng(seed)
        self.cfg, self.ty, self.page, self.layer = cfg, ty, page, layer
        self.pos = np.asarray(pos, np.int32)
        self.n_tok = np.asarray(n_tok, np.int32)
        self.tok = np.concatenate([[0], np.cumsum(self.n_tok)])
        self.total = int(self.tok[-1])
        ends = self.pos + self.n_tok
        held = -(-ends // page)
        width = int(held.max()) + extra_cols
        self.n_pages = int(held.sum()) + spare
        order = g.permutation(self.n_pages)
        # entries past a sequence's last page are numbers like any other's
        self.table = g.integers(0, self.n_pages, (len(self.pos), width)).astype(np.int32)
        at = 0
        for s, n in enumerate(held):
            self.table[s, :n] = order[at:at + n]
            at += n
        self.kv = cfg.n_head_kv * 64
        self.stride = page * self.kv + gap
        shape = (cfg.n_layers, self.n_pages, self.stride)
        self.kp, self.vp = (np.full(shape, NAN[ty], NP[ty]) for _ in range(2))
        for s, p in enumerate(self.pos):
            self.put(s, 0, g.standard_normal((p, self.kv)) * std, g.standard_normal((p, self.kv)))
        self.q = (g.standard_normal((self.total, cfg.n_head * 64)) * std).astype(np.float32)
        self.k = (g.standard_normal((self.total, self.kv)) * std).astype(np.float32)
        self.v = g.standard_normal((self.total, self.kv)).astype(np.float32)

    def rows(self, s, p0, n):
        """(page, element offset) of positions p0 .. p0 + n - 1 of sequence s; page -1: absent."""
        p = np.arange(p0, p0 + n)
        pages = self.table[s, p // self.page].astype(np.int64)
        pages[(pages < 0) | (pages >= self.n_pages)] = -1
        return pages, (p % self.page) * self.kv

    def put(self, s, p0, k, v):
        pages, off = self.rows(s, p0, len(k))
        for pool, x in ((self.kp, k), (self.vp, v)):
            b = to_bits(np.asarray(x, np.float32), self.ty) if len(x) else x
            for i, (g, o) in enumerate(zip(pages, off)):
                if g >= 0:
                    pool[self.layer, g, o:o + self.kv] = b[i]

    def rotated(self, O, x, heads):
        """x [total][heads * 64] rotated at its tokens' positions with the bits of rope()."""
        y = x.copy()
        for s in range(len(self.pos)):
            for t in range(self.n_tok[s]):
                r = self.tok[s] + t
                s_ = O.Shape(n_head=heads, n_head_kv=1)
                y[r], _ = O.rope(x[r], np.zeros(64, np.float32), int(self.pos[s] + t), s_)
        return y

    def append(self, O, rotate=True):
        k = self.rotated(O, self.k, self.cfg.n_head_kv) if rotate else self.k
        for s in range(len(self.pos)):
            a, b = self.tok[s], self.tok[s + 1]
            self.put(s, int(self.pos[s]), k[a:b], self.v[a:b])

    def attend(self, O, rotate=True):
        """(out, bound) [total][n_head * 64] in 64 bits.

        The bound on fp32's error: a score is a sum of 64 products of values each
        within 4 U (rotation and scaling, two or three pieces of 8 or 11 bits), off
        by at most 80 U sum|q k| / 8, like the largest one it is compared with, and
        their difference is rounded once more: a weight is off by a factor of
        exp(2 * 82 U A) for A the largest sum|q k| / 8, its own exp and pieces within
        16 U.  Weights are summed, with and without values, in runs of at least 8:
        n / 8 + 32 roundings each, and one division."""
        q = self.rotated(O, self.q, self.cfg.n_head) if rotate else self.q
        h, hkv = self.cfg.n_head, self.cfg.n_head_kv
        g = h // hkv
        out = np.zeros((self.total, h, 64))
        bound = np.zeros((self.total, h, 64))
        for s in range(len(self.pos)):
            n = int(self.pos[s] + self.n_tok[s])
            pages, off = self.rows(s, 0, n)
            there = np.nonzero(pages >= 0)[0]
            idx = off[there][:, None] + np.arange(self.kv)[None, :]
            k, v = (to_f64(pool[self.layer, pages[there][:, None], idx], self.ty).reshape(-1, hkv, 64)
                    for pool in (self.kp, self.vp))
            for t in range(self.n_tok[s]):
                m = int(np.searchsorted(there, self.pos[s] + t, side="right"))
                if m == 0:
                    continue
                r = self.tok[s] + t
                qr = q[r].astype(np.float64).reshape(hkv, g, 64)
                for j in range(hkv):
                    x = qr[j] @ k[:m, j].T / 8
                    a = (np.abs(qr[j]) @ np.abs(k[:m, j]).T / 8).max(-1)
                    w = np.exp(x - x.max(-1, keepdims=True))
                    w /= w.sum(-1, keepdims=True)
                    out[r, j * g:(j + 1) * g] = w @ v[:m, j]
                    bound[r, j * g:(j + 1) * g] = (U * (164 * a + 96 + m / 4))[:, None] * (w @ np.abs(v[:m, j]))
        return out.reshape(self.total, h * 64), bound.reshape(self.total, h * 64)

    @contextlib.contextmanager
    def on(self, eng):
        """The batch on the device: (cache, arrays q, k, v, out)."""
        made = {n: eng.array(a) for n, a in (("kp", self.kp), ("vp", self.vp), ("table", self.table),
                                             ("q", self.q), ("k", self.k), ("v", self.v)) if a.size}
        made["out"] = eng.array(np.full((max(self.total, 1) + 1, self.cfg.n_head * 64), 7.0, np.float32))
        for n in "qkv":
            made.setdefault(n, made["out"])
        try:
            yield tla.PagedCache(key_pages=made["kp"].ptr, value_pages=made["vp"].ptr, type=self.ty,
                                 page_size=self.page, n_pages=self.n_pages, page_stride=self.stride,
                                 layer_stride=self.n_pages * self.stride, table=made["table"].ptr,
                                 table_stride=self.table.shape[1]), made
        finally:
            for a in {id(a): a for a in made.values()}.values():
                a.free()

    def run(self, eng, O, append=True, rotate=True, layer=None):
        """Append and attend on the device: the output rows; checks that the pools
        then hold what they should, bit for bit, and that the row behind the last
        is left as it was."""
        layer = self.layer if layer is None else layer
        print(f"  paged {NAMES[self.ty]} page={self.page} heads={self.cfg.n_head}/{self.cfg.n_head_kv} "
              f"pos={self.pos.tolist()[:6]} n_tok={self.n_tok.tolist()[:6]} rotate={rotate}", flush=True)
        with self.on(eng) as (cache, a):
            if append:
                eng.paged_append(cache, self.pos, self.n_tok, layer, a["k"].ptr, a["v"].ptr, rotate)
                self.append(O, rotate)
            eng.paged_attention(cache, self.pos, self.n_tok, layer, a["out"].ptr, a["q"].ptr, rotate)
            out = a["out"].download()
            assert same_bits(a["kp"].download(), self.kp, self.ty), "key pages differ"
            assert same_bits(a["vp"].download(), self.vp, self.ty), "value pages differ"
        assert np.all(out[self.total:] == 7.0), "rows behind the last were written"
        return out[:self.total]

    def check(self, eng, O, **kw):
        got = self.run(eng, O, **kw)
        want, bound = self.attend(O, kw.get("rotate", True))
        err = np.abs(got - want)
        worst = float((err / np.maximum(bound, 1e-300)).max()) if err.size else 0.0
        print(f"    max-abs {err.max() if err.size else 0:.2e}, {worst:.2f} of the bound", flush=True)
        assert not np.isnan(got).any()
        assert np.all(err <= bound), f"{worst:.2f} of the bound"
        return got
