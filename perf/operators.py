"""Operators of a serving step over a paged cache, and what each costs.

A server keeps the keys and values of its sequences in pages of `page`
positions: sequence s's position p is row p % page of page table[s][p / page].
Each step then runs

    append   Engine.paged_append: the new tokens' k (rotated) and v into their rows
    attend   Engine.paged_attention: the new tokens' queries over their sequences,
             one token or a chunk of a prompt each, in one call
    logits   Engine.logits_process: penalties for tokens already said, biases and a
             grammar's mask on the logits, and the token that is left on top

A case is a dict of plain values whose "op" names the operator.  "cache" is the
type of the pages' elements; n_seq sequences hold up to ctx positions before the
call (uniform in [ctx / 8, ctx] when ragged) and bring n_tok tokens each, or one
token each but the first's n_tok when mixed.  With evicted, half the sequences
have given back their oldest pages, whose table entries are -1.

Heads of 64; TinyLlama's 32 / 4 heads and vocabulary of 32000, and other counts
the engine takes.
"""
from __future__ import annotations

import importlib
import math

import numpy as np
import torch

own = False

DEV = "cuda"
HEAD_DIM = 64
FREQ_BASE = 10000.0
F64 = torch.float64
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}


def listed():
    a = {"op": "append", "n_head": 32, "n_head_kv": 4, "ragged": False, "mixed": False, "evicted": False}
    t = dict(a, op="attend")
    return [
        # the rows of one decode step of a full server: latency
        dict(a, name="append_step", cache="f16", page=16, n_seq=64, ctx=2000, n_tok=1, ragged=True),
        # a chunk of a prompt into a cache that keeps every bit
        dict(a, name="append_chunk_f32", cache="f32", page=64, n_seq=1, ctx=1000, n_tok=555),
        # prompts of a whole batch at once
        dict(a, name="append_prompts", cache="bf16", page=32, n_seq=16, ctx=0, n_tok=2048),
        # one conversation's token: latency
        dict(t, name="attend_single", cache="f16", page=16, n_seq=1, ctx=127, n_tok=1),
        # one decode step of a full server, conversations of all lengths
        dict(t, name="attend_step", cache="f16", page=16, n_seq=64, ctx=2047, n_tok=1, ragged=True),
        # long documents, a small batch, exact keys and values
        dict(t, name="attend_long_f32", cache="f32", page=128, n_seq=8, ctx=16383, n_tok=1),
        # a prompt from its beginning
        dict(t, name="attend_prompt_f32", cache="f32", page=64, n_seq=1, ctx=0, n_tok=2048),
        # the next chunk of a long prompt
        dict(t, name="attend_chunk", cache="f16", page=64, n_seq=1, ctx=8000, n_tok=512),
        # a step with a chunk of one prompt and single tokens of the others, some
        # of which keep the newest part of their context only
        dict(t, name="attend_mixed", cache="bf16", page=16, n_seq=32, ctx=2047, n_tok=333, ragged=True, mixed=True,
             evicted=True),
        # one conversation's next token: latency
        {"name": "logits_single", "op": "logits", "n_seq": 1, "n_vocab": 32000, "history": 500, "biases": 0,
         "mask": False},
        # one step of a full server, some of it under a grammar
        {"name": "logits_step", "op": "logits", "n_seq": 64, "n_vocab": 32000, "history": 2048, "biases": 100,
         "mask": True},
        # a larger vocabulary of an odd size, and a larger batch
        {"name": "logits_wide", "op": "logits", "n_seq": 200, "n_vocab": 100003, "history": 1000, "biases": 300,
         "mask": True},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "attend", "logits"])
    if op == "logits":
        n_vocab = rng.choice([32000, _log(rng, 500, 100000)])
        return {"op": op, "n_seq": _log(rng, 1, max(1, min(200, 15000000 // n_vocab))), "n_vocab": n_vocab,
                "history": rng.choice([0, _log(rng, 1, 8192)]), "biases": rng.choice([0, _log(rng, 1, 300)]),
                "mask": rng.random() < 0.6}
    n_head, n_head_kv = rng.choice([(32, 4), (32, 4), (32, 8), (16, 2), (8, 8), (12, 4), (16, 1)])
    case = {"op": op, "n_head": n_head, "n_head_kv": n_head_kv, "cache": rng.choice(["f16", "bf16", "f32"]),
            "page": rng.choice([16, 16, 32, 64, 128, 256, 8, 1]), "n_seq": 1, "ctx": 0, "n_tok": 1,
            "ragged": rng.random() < 0.5, "mixed": False, "evicted": rng.random() < 0.25}
    if op == "append":
        case["n_seq"] = _log(rng, 1, 128)
        case["n_tok"] = rng.choice([1, _log(rng, 2, max(2, min(2048, 30000 // case["n_seq"])))])
        case["ctx"] = rng.choice([0, _log(rng, 16, 4000)])
    elif rng.random() < 0.5:  # single tokens
        case["ctx"] = _log(rng, 1, 16383)
        case["n_seq"] = _log(rng, 1, max(1, min(96, 130000 // (case["ctx"] + 1))))
    else:  # chunks; query and key pairs as in the listed ones
        case["n_tok"] = _log(rng, 2, 1500)
        case["ctx"] = rng.choice([0, _log(rng, 16, max(17, min(8000, 4000000 // case["n_tok"])))])
        pairs = case["n_tok"] * (case["ctx"] + case["n_tok"])
        case["n_seq"] = _log(rng, 1, max(1, min(32, 4000000 // pairs)))
        case["mixed"] = case["n_seq"] > 1 and rng.random() < 0.5
    return case


# ---- inputs ---------------------------------------------------------------------

_engines: dict = {}


def _engine(n_head, n_head_kv, n_ctx):
    """The process's engine for one configuration (a server keeps one)."""
    tla = importlib.import_module("tinyllama-engine_amd")
    n_ctx = max(128, 1 << (n_ctx - 1).bit_length())
    key = (n_head, n_head_kv, n_ctx)
    if key not in _engines:
        _engines[key] = tla.Engine(tla.Config(1, n_head * HEAD_DIM, n_head, n_head_kv, n_ctx, FREQ_BASE))
    return _engines[key]


def _angles(n_pos):
    """RoPE's angles [n_pos][32]: the 32-bit product of the position and the
    32-bit frequency, which is what the model was trained with."""
    expo = np.arange(0, HEAD_DIM, 2).astype(np.float32) / np.float32(HEAD_DIM)
    freq = np.float32(1) / np.power(np.float64(np.float32(FREQ_BASE)), expo.astype(np.float64)).astype(np.float32)
    return np.arange(n_pos).astype(np.float32)[:, None] * freq[None, :]


def _batch(case, rng):
    """(pos0, n_tok) of every sequence."""
    n, ctx = case["n_seq"], case["ctx"]
    pos0 = rng.integers(ctx // 8, ctx + 1, n) if case["ragged"] else np.full(n, ctx)
    n_tok = np.full(n, case["n_tok"])
    if case["mixed"]:
        n_tok[1:] = 1
    return pos0.astype(np.int32), n_tok.astype(np.int32)


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed))
    rng = np.random.default_rng(int(seed))
    s = {"case": dict(case), "op": case["op"]}
    if case["op"] == "logits":
        n, nv, nh, nb = case["n_seq"], case["n_vocab"], case["history"], case["biases"]
        s["logits"] = torch.randn(n, nv, generator=g, device=DEV) * 3
        # words repeat as in text: a token's rank goes as a power of a uniform number
        u = torch.rand(n, max(nh, 1), generator=g, device=DEV)
        s["history"] = (nv * u ** 4).long().clamp_(0, nv - 1).int()
        s["n_history"] = torch.randint(nh // 2, nh + 1, (n,), generator=g, device=DEV, dtype=torch.int32)
        r = torch.rand(n, 3, generator=g, device=DEV)
        s["penalties"] = r * torch.tensor([0.3, 1.0, 0.5], device=DEV) + torch.tensor([1.0, 0.0, 0.0], device=DEV)
        s["bias_tokens"] = torch.randint(0, nv, (n, max(nb, 1)), generator=g, device=DEV, dtype=torch.int32)
        s["biases"] = torch.randn(n, max(nb, 1), generator=g, device=DEV) * 4
        s["n_biases"] = torch.randint(nb // 2, nb + 1, (n,), generator=g, device=DEV, dtype=torch.int32)
        # a grammar lets a few words or most of them through; one row has no way on
        words = (nv + 31) // 32
        few = torch.ones(n, words, device=DEV, dtype=torch.int32)
        for _ in range(4):
            few &= torch.randint(-2 ** 31, 2 ** 31, (n, words), generator=g, device=DEV, dtype=torch.int64).int()
        most = torch.randint(-2 ** 31, 2 ** 31, (n, words), generator=g, device=DEV, dtype=torch.int64).int()
        s["mask"] = torch.where(torch.arange(n, device=DEV)[:, None] % 2 == 0, most, few)
        if n > 2:
            s["mask"][n // 2] = 0
        s["out"] = torch.zeros_like(s["logits"])
        s["tokens"] = torch.zeros(n, dtype=torch.int32, device=DEV)
        if own:
            tla = importlib.import_module("tinyllama-engine_amd")
            s["e"] = _engine(32, 4, 128)
            p = lambda k: s[k].data_ptr()  # noqa: E731
            s["rules"] = tla.LogitRules(
                **({"history": p("history"), "history_len": p("n_history"), "history_stride": nh,
                    "penalties": p("penalties")} if nh else {}),
                **({"bias_token": p("bias_tokens"), "bias_value": p("biases"), "bias_len": p("n_biases"),
                    "bias_stride": nb} if nb else {}),
                **({"mask": p("mask"), "mask_stride": words} if case["mask"] else {}))
        torch.cuda.synchronize()  # the engine has a stream of its own
        return s
    h, hkv, page, dt = case["n_head"], case["n_head_kv"], case["page"], DTYPES[case["cache"]]
    kv = hkv * HEAD_DIM
    pos0, n_tok = _batch(case, rng)
    s["pos0"], s["n_tok"] = pos0, n_tok
    total, longest = int(n_tok.sum()), int((pos0 + n_tok).max())
    # the pool's pages are handed out in the order in which sequences grew; some
    # are another's or free, their rows an earlier request's
    held = -(-(pos0 + n_tok) // page)
    width = int(held.max())
    n_pages = case["n_seq"] * -(-(case["ctx"] + case["n_tok"]) // page) + 3
    order = rng.permutation(n_pages)[:int(held.sum())]
    table = np.full((case["n_seq"], width), -1, np.int32)
    table[np.arange(width)[None, :] < held[:, None]] = order
    if case["evicted"]:
        gone = np.where(np.arange(case["n_seq"]) % 2 == 1, pos0 // page // 2, 0)
        table[np.arange(width)[None, :] < gone[:, None]] = -1
    s["table"] = torch.from_numpy(table).to(DEV)
    s["kp"] = torch.randn(n_pages, page, kv, generator=g, device=DEV).to(dt)
    s["vp"] = torch.randn(n_pages, page, kv, generator=g, device=DEV).to(dt)
    if case["op"] == "append":
        s["k"] = torch.randn(total, kv, generator=g, device=DEV)
        s["v"] = torch.randn(total, kv, generator=g, device=DEV)
    else:
        s["q"] = torch.randn(total, h * HEAD_DIM, generator=g, device=DEV) * 1.5
        s["out"] = torch.zeros_like(s["q"])
    # what a program that goes through the batch on the device keeps beside it
    s["seq"] = torch.from_numpy(np.repeat(np.arange(case["n_seq"]), n_tok)).to(DEV)
    s["nth"] = torch.from_numpy(np.concatenate([np.arange(t) for t in n_tok])).to(DEV)
    s["pos0_dev"] = torch.from_numpy(pos0.astype(np.int64)).to(DEV)
    s["len_dev"] = torch.from_numpy((pos0 + n_tok).astype(np.int64)).to(DEV)
    a = torch.from_numpy(_angles(longest)).to(DEV).to(F64)
    s["cos"], s["sin"] = a.cos().float(), a.sin().float()
    if own:
        tla = importlib.import_module("tinyllama-engine_amd")
        s["e"] = _engine(h, hkv, longest)
        s["cache"] = tla.PagedCache(key_pages=s["kp"].data_ptr(), value_pages=s["vp"].data_ptr(),
                                    type={"f32": tla.KV_F32, "f16": tla.KV_F16, "bf16": tla.KV_BF16}[case["cache"]],
                                    page_size=page, n_pages=n_pages, table=s["table"].data_ptr(), table_stride=width)
    torch.cuda.synchronize()  # the engine has a stream of its own
    return s


# ---- one pass -------------------------------------------------------------------

def run(s):
    if s["op"] == "append":
        if own:
            s["e"].paged_append(s["cache"], s["pos0"], s["n_tok"], 0, s["k"].data_ptr(), s["v"].data_ptr())
            return s["kp"], s["vp"]
        return _append(s)
    if s["op"] == "attend":
        if own:
            s["e"].paged_attention(s["cache"], s["pos0"], s["n_tok"], 0, s["out"].data_ptr(), s["q"].data_ptr())
            return s["out"]
        return _attend(s)
    if own:
        n, nv = s["logits"].shape
        s["e"].logits_process(n, nv, s["rules"], s["out"].data_ptr(), s["logits"].data_ptr(), s["tokens"].data_ptr())
        return s["out"], s["tokens"]
    return _logits(s)


def _rotate(x, cos, sin):
    """RoPE of x [n][heads][64]: consecutive pairs, cos and sin [n][32]."""
    a, b = x[..., 0::2], x[..., 1::2]
    c, d = cos[:, None, :], sin[:, None, :]
    return torch.stack([a * c - b * d, a * d + b * c], -1).flatten(-2)


def _append(s):
    case, kp, vp = s["case"], s["kp"], s["vp"]
    page, hkv = case["page"], case["n_head_kv"]
    pos = s["pos0_dev"][s["seq"]] + s["nth"]
    ids = s["table"][s["seq"], pos // page].long()
    there = (ids >= 0) & (ids < kp.shape[0])
    row = (ids * page + pos % page)[there]
    k = _rotate(s["k"].view(-1, hkv, HEAD_DIM), s["cos"][pos], s["sin"][pos]).flatten(1)
    kp.view(-1, hkv * HEAD_DIM)[row] = k[there].to(kp.dtype)
    vp.view(-1, hkv * HEAD_DIM)[row] = s["v"][there].to(vp.dtype)
    return kp, vp


def _attend(s):
    case, kp, vp, table = s["case"], s["kp"], s["vp"], s["table"]
    n, page, h, hkv = case["n_seq"], case["page"], case["n_head"], case["n_head_kv"]
    g, n_tok, n_key = h // hkv, int(s["n_tok"].max()), int((s["pos0"] + s["n_tok"]).max())
    # every sequence's rows, as one padded batch
    at = torch.arange(n_key, device=DEV)
    ids = table[:, at // page].long()
    seen = (ids >= 0) & (ids < kp.shape[0]) & (at[None, :] < s["len_dev"][:, None])
    row = torch.where(seen, ids * page + at % page, 0)
    gone = ~seen[:, :, None, None]
    k = kp.view(-1, hkv, HEAD_DIM)[row].float().masked_fill_(gone, 0).permute(0, 2, 3, 1).contiguous()
    v = vp.view(-1, hkv, HEAD_DIM)[row].float().masked_fill_(gone, 0).transpose(1, 2).contiguous()
    # and its queries [n][hkv][tokens x g][64]
    pos = s["pos0_dev"][s["seq"]] + s["nth"]
    q = torch.zeros(n, n_tok, h, HEAD_DIM, device=DEV)
    q[s["seq"], s["nth"]] = _rotate(s["q"].view(-1, h, HEAD_DIM), s["cos"][pos], s["sin"][pos])
    q = q.view(n, n_tok, hkv, g, HEAD_DIM).permute(0, 2, 1, 3, 4).reshape(n, hkv, n_tok * g, HEAD_DIM)
    p = torch.matmul(q, k).mul_(1 / math.sqrt(HEAD_DIM))
    qpos = s["pos0_dev"][:, None] + torch.arange(n_tok, device=DEV)[None, :]
    hidden = ~seen[:, None, :] | (at[None, None, :] > qpos[:, :, None])  # [n][tokens][keys]
    p.view(n, hkv, n_tok, g, n_key).masked_fill_(hidden[:, None, :, None, :], -math.inf)
    top = p.amax(-1, keepdim=True)
    p.sub_(torch.where(top == -math.inf, 0, top)).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p, v) / torch.where(total == 0, 1, total)
    o = o.view(n, hkv, n_tok, g, HEAD_DIM).permute(0, 2, 1, 3, 4).reshape(n, n_tok, h * HEAD_DIM)
    return o[s["seq"], s["nth"]]


def _allowed(mask, n_vocab):
    """The mask's bits [n][n_vocab], token j at bit j % 32 of word j / 32."""
    j = torch.arange(n_vocab, device=DEV)
    return (mask[:, j // 32] >> (j % 32).int()) & 1 == 1


def _logits(s):
    case, x = s["case"], s["logits"].clone()
    n, nv = x.shape
    if case["history"]:
        said = torch.arange(case["history"], device=DEV)[None, :] < s["n_history"][:, None]
        count = torch.zeros(n, nv, device=DEV).scatter_add_(1, s["history"].long(), said.float())
        rep, pres, freq = (s["penalties"][:, i:i + 1] for i in range(3))
        y = torch.where(x > 0, x / rep, x * rep) - (count * freq + pres)
        x = torch.where(count > 0, y, x)
    if case["biases"]:  # the last of a token's biases counts
        nth = torch.arange(1, case["biases"] + 1, device=DEV)[None, :].expand(n, -1)
        nth = torch.where(nth <= s["n_biases"][:, None], nth, 0)
        last = torch.zeros(n, nv, dtype=torch.int64, device=DEV)
        last.scatter_reduce_(1, s["bias_tokens"].long(), nth, "amax")
        x = torch.where(last > 0, x + s["biases"].gather(1, (last - 1).clamp_min(0)), x)
    if case["mask"]:
        x = torch.where(_allowed(s["mask"], nv), x, -math.inf)
    top = x.amax(-1, keepdim=True)
    first = torch.where(x == top, torch.arange(nv, device=DEV), nv).amin(-1)
    return x, torch.where(top[:, 0] == -math.inf, -1, first).int()


# ---- what a pass cannot do without -----------------------------------------------

def work(case):
    if case["op"] == "logits":
        n, nv = case["n_seq"], case["n_vocab"]
        return {"bytes": n * (8 * nv + (nv / 8 if case["mask"] else 0) + 4 * case["history"] * 0.75
                              + 8 * case["biases"] * 0.75 + 4), "flops": n * nv}
    kv, q, es = case["n_head_kv"] * HEAD_DIM, case["n_head"] * HEAD_DIM, BYTES[case["cache"]]
    n, t, ctx = case["n_seq"], case["n_tok"], case["ctx"]
    mean = (ctx // 8 + ctx) / 2 if case["ragged"] else ctx  # a ragged batch's mean length
    toks = [t] + [1 if case["mixed"] else t] * (n - 1)
    total = sum(toks)
    if case["op"] == "append":
        return {"bytes": total * kv * 2 * (4 + es), "flops": total * kv * 3}
    # evicted: every second sequence has lost half of its context
    kept = mean * (1 - 0.5 * (n // 2) / n) if case["evicted"] else mean
    keys = n * kept + total
    pairs = sum(u * kept + u * (u + 1) / 2 for u in toks)
    return {"bytes": 2 * keys * kv * es + total * q * 8, "flops": 4 * q * pairs}


# ---- the same in 64 bits ----------------------------------------------------------

def _turned(x, pos):
    """x [t][heads][64] in 64 bits, each pair taken as a complex number and
    turned by its position's angle."""
    a = torch.from_numpy(_angles(int(pos.max()) + 1)[pos]).to(DEV).to(F64)
    z = torch.view_as_complex(x.to(F64).reshape(*x.shape[:-1], HEAD_DIM // 2, 2).contiguous())
    return torch.view_as_real(z * torch.polar(torch.ones_like(a), a)[:, None, :]).flatten(-2)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "logits":
        return _exact_logits(case, s)
    page, h, hkv = case["page"], case["n_head"], case["n_head_kv"]
    table = s["table"].cpu().numpy()
    ends = np.cumsum(s["n_tok"])
    kp, vp = (s[k].to(F64).view(-1, hkv, HEAD_DIM) for k in ("kp", "vp"))
    n_pages = s["kp"].shape[0]
    if case["op"] == "append":
        for i, (p0, t, e) in enumerate(zip(s["pos0"].tolist(), s["n_tok"].tolist(), ends.tolist())):
            pos = np.arange(p0, p0 + t)
            ids = table[i, pos // page].astype(np.int64)
            ok = (ids >= 0) & (ids < n_pages)
            row = torch.from_numpy((ids * page + pos % page)[ok]).to(DEV)
            pick = torch.from_numpy(np.arange(e - t, e)[ok]).to(DEV)
            kp[row] = _turned(s["k"][pick].view(-1, hkv, HEAD_DIM), pos[ok]) if len(pick) else kp[row]
            vp[row] = s["v"][pick].to(F64).view(-1, hkv, HEAD_DIM)
        return kp.view(s["kp"].shape), vp.view(s["vp"].shape)
    out = torch.zeros(s["q"].shape[0], h, HEAD_DIM, dtype=F64, device=DEV)
    r = h // hkv
    for i, (p0, t, e) in enumerate(zip(s["pos0"].tolist(), s["n_tok"].tolist(), ends.tolist())):
        pos = np.arange(p0 + t)
        ids = table[i, pos // page].astype(np.int64)
        pos = pos[(ids >= 0) & (ids < n_pages)]
        if not len(pos):
            continue
        row = torch.from_numpy(table[i, pos // page].astype(np.int64) * page + pos % page).to(DEV)
        later = torch.from_numpy(pos[None, :] > np.arange(p0, p0 + t)[:, None]).to(DEV)
        q = _turned(s["q"][e - t:e].view(t, h, HEAD_DIM), np.arange(p0, p0 + t))
        for j in range(h):
            x = (q[:, j] @ kp[row, j // r].t().contiguous() / math.sqrt(HEAD_DIM)).masked_fill_(later, -math.inf)
            some = ~later.all(-1)
            out[e - t:e, j][some] = torch.softmax(x[some], -1) @ vp[row, j // r]
    return out.view(-1, h * HEAD_DIM)


def _exact_logits(case, s):
    x = s["logits"].to(F64)
    n, nv = x.shape
    rows = torch.arange(n, device=DEV)[:, None]
    if case["history"]:
        h = torch.where(torch.arange(case["history"], device=DEV) < s["n_history"][:, None], s["history"], nv).long()
        count = torch.bincount((h + rows * (nv + 1)).flatten(), minlength=n * (nv + 1)).view(n, nv + 1)[:, :nv]
        rep, pres, freq = s["penalties"].to(F64).unbind(1)
        hit = count > 0
        x = torch.where(hit & (x > 0), x / rep[:, None], torch.where(hit, x * rep[:, None], x))
        x = x - count * freq[:, None] - hit * pres[:, None]
    for k in range(case["biases"]):  # in order: what the next bias of a token replaces
        if k == 0:
            add = torch.zeros_like(x)
        live = (s["n_biases"] > k).nonzero()[:, 0]
        add[live, s["bias_tokens"][live, k].long()] = s["biases"][live, k].to(F64)
    if case["biases"]:
        x = x + add
    if case["mask"]:
        bits = torch.stack([s["mask"] >> b & 1 for b in range(32)], -1).flatten(1)[:, :nv]
        x = x.masked_fill(bits == 0, -math.inf)
    return x, None
