"""The operators of a serving step together, as a server calls them: prompts of
three lengths through the layers in one batch, then steps of one token each, over
one paged cache, with penalties on the logits, against tla_forward running every
sequence for itself over a contiguous cache."""
import numpy as np
import pytest

import quant_ref as Q
from helpers import device_arrays, log, tla
from test_gpu_logits import reference

pytestmark = pytest.mark.gpu

# of the largest logit: the bound of the forward pass for F32 pages; a key or value
# of F16 / BF16 pages is off by 2^-11 / 2^-8 of itself, in each of two layers
# whose attention is one of the two terms that a residual adds, and a score by
# 2^-11 / 2^-8 of sum|q k| / 8, some units here
TOL = {tla.KV_F32: 1e-4, tla.KV_F16: 1e-2, tla.KV_BF16: 8e-2}


class Server:
    """Pages, tables and the layers' calls of a small model."""

    def __init__(self, eng, model, spec, tensors, kv_type, page, track):
        self.e, self.m, self.s, self.track = eng, model, spec, track
        self.ty = {n: t[1] for n, t in tensors.items()}
        self.cache = eng.paged_cache(64, page, kv_type)
        self.page, self.free = page, list(np.random.default_rng(1).permutation(64))
        self.tables, self.pos, self.said = {}, {}, {}

    def close(self):
        self.e.free_paged_cache(self.cache)

    def buf(self, *shape):
        return self.track(self.e.array(shape))

    def w(self, name):
        return self.m.arrays[name].ptr

    def step(self, batch):
        """batch: {sequence: new tokens}; the logits of each one's last token."""
        e, s = self.e, self.s
        ids = list(batch)
        n_tok = np.array([len(batch[i]) for i in ids], np.int32)
        pos = np.array([self.pos.get(i, 0) for i in ids], np.int32)
        for i, p, n in zip(ids, pos, n_tok):
            t = self.tables.setdefault(i, [])
            while len(t) * self.page < p + n:
                t.append(self.free.pop())
            self.pos[i] = int(p + n)
            self.said.setdefault(i, []).extend(batch[i])
        table = np.full((len(ids), max(len(self.tables[i]) for i in ids)), -1, np.int32)
        for r, i in enumerate(ids):
            table[r, :len(self.tables[i])] = self.tables[i]
        tab = self.track(e.array(table))
        self.cache.table, self.cache.table_stride = tab.ptr, table.shape[1]
        total, embd, kv, ff = int(n_tok.sum()), s.n_embd, s.kv_dim, s.n_ff
        x, q, att = (self.buf(total, embd) for _ in range(3))
        k, v, hb = self.buf(total, kv), self.buf(total, kv), self.buf(total, 2, ff)
        for r, tok in enumerate(t for i in ids for t in batch[i]):
            e.embed(x.at(4 * embd * r), self.w("token_embd.weight"), tok, embd, s.n_vocab, self.ty["token_embd.weight"])
        for l in range(s.n_layers):
            b = f"blk.{l}."
            e.attn_qkv(total, q.ptr, k.ptr, v.ptr, x.ptr, self.w(b + "attn_norm.weight"), s.rms_norm_eps,
                       self.w(b + "attn_q.weight"), self.w(b + "attn_k.weight"), self.w(b + "attn_v.weight"),
                       self.ty[b + "attn_q.weight"])
            e.paged_append(self.cache, pos, n_tok, l, k.ptr, v.ptr)
            e.paged_attention(self.cache, pos, n_tok, l, att.ptr, q.ptr)
            e.attn_out(total, x.ptr, self.w(b + "attn_output.weight"), att.ptr, self.ty[b + "attn_output.weight"])
            e.ffn_block(total, x.ptr, self.w(b + "ffn_norm.weight"), s.rms_norm_eps, self.w(b + "ffn_gate.weight"),
                        self.w(b + "ffn_up.weight"), self.w(b + "ffn_down.weight"), ff, self.ty[b + "ffn_gate.weight"],
                        hb.ptr)
        logits, xb = self.buf(len(ids), s.n_vocab), self.buf(embd)
        out = "output.weight" if "output.weight" in self.ty else "token_embd.weight"
        for r, last in enumerate(np.cumsum(n_tok) - 1):
            e.rmsnorm(xb.ptr, x.at(4 * embd * int(last)), self.w("output_norm.weight"), embd, s.rms_norm_eps)
            e.matmul(logits.at(4 * s.n_vocab * r), self.w(out), xb.ptr, s.n_vocab, embd, self.ty[out])
        return logits

    def choose(self, ids, logits):
        """Each sequence's next token under its rules, and the rules."""
        e, n, nv = self.e, len(ids), self.s.n_vocab
        long = max(len(self.said[i]) for i in ids)
        hist = np.full((n, long), -1, np.int32)
        for r, i in enumerate(ids):
            hist[r, :len(self.said[i])] = self.said[i]
        rules = {"hist": hist, "n_hist": np.array([len(self.said[i]) for i in ids], np.int32),
                 "pen": np.tile(np.array([1.3, 0.2, 0.1], np.float32), (n, 1)),
                 "mask": np.random.default_rng(long).integers(0, 2 ** 32, (n, (nv + 31) // 32), dtype=np.uint64).astype(np.uint32)}
        d = {k: self.track(e.array(a)) for k, a in rules.items()}
        r = tla.LogitRules(history=d["hist"].ptr, history_len=d["n_hist"].ptr, history_stride=long, penalties=d["pen"].ptr,
                           mask=d["mask"].ptr, mask_stride=rules["mask"].shape[1])
        tok = self.track(e.array(np.zeros(n, np.int32)))
        e.logits_process(n, nv, r, logits.ptr, logits.ptr, tok.ptr)
        return tok.download(), rules


@pytest.mark.parametrize("kv_type", [tla.KV_F32, tla.KV_F16, tla.KV_BF16])
@pytest.mark.parametrize("wtype,page", [(Q.F32, 16), (Q.Q8_0, 32)])
def test_serving_steps(W, engines, kv_type, wtype, page):
    spec = W.ModelSpec(2, 512, 8, 2, 1024, 128, 999)
    tensors = W.make_model(spec, wtype, salt=5)
    eng = engines(2, 128, 8, 2)
    g = np.random.default_rng(3)
    batch = {i: [int(t) for t in g.integers(0, spec.n_vocab, n)] for i, n in ((7, 17), (3, 1), (5, 40))}
    dm = tla.DeviceModel(eng, tensors, spec.n_ff, spec.n_vocab, spec.rms_norm_eps)
    with device_arrays() as track:
        srv = Server(eng, dm, spec, tensors, kv_type, page, track)
        alone = {i: eng.kv_cache(1) for i in batch}
        for kv in alone.values():
            track(kv[0]), track(kv[1])
        one = track(eng.array((spec.n_vocab,)))
        try:
            for step in range(6):
                ids = list(batch)
                start = {i: srv.pos.get(i, 0) for i in ids}
                logits = srv.step(batch)
                got = logits.download()
                for r, i in enumerate(ids):
                    for j, t in enumerate(batch[i]):
                        eng.forward(dm, alone[i][0].ptr, alone[i][1].ptr, t, start[i] + j, one.ptr)
                    want = one.download()
                    err = float(np.abs(got[r] - want).max() / np.abs(want).max())
                    log(f"  step {step} sequence {i} at {srv.pos[i]}: {err:.2e} of the largest logit")
                    assert err <= TOL[kv_type]
                tokens, rules = srv.choose(ids, logits)
                ruled, best = reference(got, **rules)
                assert np.array_equal(logits.download().view(np.uint32), ruled.view(np.uint32))
                assert np.array_equal(tokens, best)
                batch = {i: [int(t)] for i, t in zip(ids, tokens)}
                if step == 2:  # a new conversation joins, another is done
                    srv.free += srv.tables.pop(7)
                    del batch[7]
                    batch[9] = [int(t) for t in g.integers(0, spec.n_vocab, 25)]
                    alone[9] = eng.kv_cache(1)
                    track(alone[9][0]), track(alone[9][1])
        finally:
            srv.close()
            dm.free()
