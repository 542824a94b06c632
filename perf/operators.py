"""Cases of the operators that score and continue sequences over an 8-bit paged key/value cache.

A sequence's keys and values lie in pages of `page` tokens, as int8 codes with one f32 scale for each (page, keys or
values, head): value = code * scale.  `codes` is [pages, 2, n_kv, page, hd] (with a leading layer axis where whole
pages move), keys row by row; the value plane of a head holds groups of four tokens, [page / 4, hd, 4].

Five kinds of case, each one operator or one step that a program makes of it:
  attend  attention of new tokens over the cache (single tokens, or short ragged chunks, causal at the end)
  append  new keys and values quantised into the cache, and the touched pages read back
  pages   fork (copy, share, drop) with the pages of the next token reserved, or compaction of the pool
  logits  log-probability, entropy, rank and best alternatives of given tokens from rows of logits
  score   log-probability and entropy of given tokens from hidden rows, through the lm_head

`own` false computes the plain form with elementary torch operations in 32 bits; `own` true calls the library.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PKG = os.path.join(ROOT, "minicpm5-vllm-tpu_b200")


_library = None


def _ops():
    """The library's module of operators, imported by the first pass that calls it."""
    global _library
    if _library is None:
        if PKG not in sys.path:
            sys.path.insert(0, PKG)
        from minicpm5_mk import ops
        _library = ops
    return _library


# ------------------------------------------------------------------------------------------------ cases
def _attend(name, S, n_q, n_kv, hd, page, max_len, max_q):
    return {"name": name, "kind": "attend", "S": S, "n_q": n_q, "n_kv": n_kv, "hd": hd, "page": page,
            "max_len": max_len, "max_q": max_q}


def _append(name, S, n_q, n_kv, hd, page, max_past, max_new):
    return {"name": name, "kind": "append", "S": S, "n_q": n_q, "n_kv": n_kv, "hd": hd, "page": page,
            "max_past": max_past, "max_new": max_new}


def _pages(name, action, rows, layers, n_kv, hd, page, max_len, pages):
    return {"name": name, "kind": "pages", "action": action, "rows": rows, "layers": layers, "n_kv": n_kv, "hd": hd,
            "page": page, "max_len": max_len, "pages": pages}


def _logits(name, T, V, k, bf16):
    return {"name": name, "kind": "logits", "T": T, "V": V, "k": k, "bf16": bf16}


def _score(name, T, V, H):
    return {"name": name, "kind": "score", "T": T, "V": V, "H": H}


def listed():
    return [
        # one user, the next token of a short answer (1B heads): latency alone
        _attend("attend_one", 1, 16, 2, 96, 64, 999, 1),
        # a serving batch in the middle of its answers (2B heads), every length different, one row idle
        _attend("attend_batch", 64, 16, 2, 128, 64, 8192, 1),
        # four long documents being continued, 128-token pages
        _attend("attend_long", 4, 16, 2, 128, 128, 131001, 1),
        # the tokens of several candidate answers scored at once after their prompts (1B heads, small pages)
        _attend("attend_chunk", 16, 16, 2, 96, 32, 8192, 64),
        # a decoding step's keys and values of one layer
        _append("append_step", 256, 16, 2, 96, 64, 4001, 1),
        # the prompts of a batch, ragged, one layer of the 2B
        _append("append_prompts", 8, 16, 2, 128, 64, 777, 8192),
        # a beam step of 256 rows over the 1B's 24 layers: half the rows are dropped, the others fork
        _pages("beam_step", "fork", 256, 24, 2, 96, 64, 393, 1500),
        # a pool half of whose pages were freed at random, closed up
        _pages("compact_pool", "compact", 64, 24, 2, 96, 64, 1024, 1200),
        # a decoding step's rows with vLLM's usual 20 alternatives, the checkpoint's vocabulary
        _logits("logits_step", 3, 130560, 20, False),
        # prompt log-probabilities from bf16 logits, five alternatives: ties abound
        _logits("logits_prompt", 2047, 73448, 5, True),
        # the answer tokens of a few candidates
        _score("score_answers", 37, 130560, 1536),
        # every token of an 8192-token prompt
        _score("score_prompt", 8192, 73448, 1536),
    ]


def _logint(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["attend", "attend", "append", "pages", "logits", "score"])
    n_q, n_kv = rng.choice([(16, 2), (16, 2), (4, 2), (4, 1), (8, 8), (12, 4)])
    hd, page = rng.choice([96, 128]), rng.choice([16, 32, 64, 128])
    if kind == "attend":
        S = _logint(rng, 1, 96)
        max_q = 1 if rng.random() < 0.6 else _logint(rng, 2, 64)
        top = min(131001, 1000000 // (S * n_kv), 67000000 // (S * max_q * n_q))
        c = _attend("", S, n_q, n_kv, hd, page, _logint(rng, min(17, top), top), max_q)
    elif kind == "append":
        S = _logint(rng, 1, 256)
        max_new = 1 if rng.random() < 0.5 else _logint(rng, 2, max(2, 120000 // (S * n_kv)))
        c = _append("", S, n_q, n_kv, hd, page, _logint(rng, 1, max(2, min(4096, 400000 // (S * n_kv)))), max_new)
    elif kind == "pages":
        rows, layers, max_len = _logint(rng, 2, 256), rng.choice([2, 3, 24, 42]), _logint(rng, 5, 1024)
        top = max(12, 900000000 // (layers * 2 * n_kv * page * hd))
        rows = max(2, min(rows, top // (2 * (-(-max_len // page) + 1))))
        max_len = min(max_len, page * max(1, top // (2 * rows) - 2))
        need = rows * (-(-max_len // page) + 2)
        c = _pages("", rng.choice(["fork", "compact"]), rows, layers, n_kv, hd, page, max_len, need + rng.randrange(need))
    elif kind == "logits":
        V = rng.choice([1000, 2048, 32001, 73448, 130560])
        c = _logits("", _logint(rng, 1, min(2047, 150000000 // V)), V, rng.choice([0, 1, 5, 20, 64]), rng.random() < 0.5)
    else:
        H, V = rng.choice([(384, 1000), (512, 2048), (1536, 73448), (2048, 73448), (1536, 130560)])
        c = _score("", _logint(rng, 1, int(8192 * 73448 * 1536 / (V * H)) if V > 10000 else 8192), V, H)
    del c["name"]
    return c


# ------------------------------------------------------------------------------------------------ inputs
def _host_rng(seed):
    return np.random.RandomState((seed * 1000003 + 17) % (2 ** 31))


def _sizes(c):
    """The ragged sizes of a case, the same for every seed: (lengths before, new tokens) per row."""
    r, k = np.random.RandomState(11), c["kind"]
    if k == "attend":
        lens = _lengths(r, c["S"], c["max_len"])
        if c["max_q"] == 1:
            return lens, np.ones(c["S"], np.int64)
        new = np.minimum(lens, 1 + r.randint(c["max_q"], size=c["S"]))
        new[int(np.argmax(lens))] = min(c["max_q"], c["max_len"])
        return lens, new
    if k == "append":
        past = r.randint(0, c["max_past"] + 1, size=c["S"]).astype(np.int64)
        new = np.maximum(1, (c["max_new"] * (0.15 + 0.85 * r.rand(c["S"]))).astype(np.int64))
        new[r.randint(c["S"])] = c["max_new"]
        if c["S"] >= 3:
            new[(int(np.argmax(new)) + 1) % c["S"]] = 0
        return past, new
    lens = np.maximum(1, (c["max_len"] * (0.5 + 0.5 * r.rand(c["rows"]))).astype(np.int64))
    lens[r.randint(c["rows"])] = c["max_len"]
    lens[0] = 0 if c["rows"] >= 3 else lens[0]
    return lens, np.ones(c["rows"], np.int64)


def _pool(g, pages, n_kv, page, hd, layers=None):
    """Codes of roughly normal keys and values: the largest of a page's head sits near 127."""
    lead = (pages,) if layers is None else (layers, pages)
    shape = (*lead, 2, n_kv, page, hd)
    codes = torch.empty(shape, dtype=torch.int8, device="cuda")
    flat = codes.view(-1)
    for part in flat.split(1 << 26):
        part.copy_(torch.randn(part.shape, device="cuda", generator=g).mul_(33).round_().clamp_(-127, 127))
    scales = 0.03 * (0.5 + torch.rand((*lead, 2, n_kv), device="cuda", generator=g))
    return codes, scales


def _dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).to("cuda")


def _lengths(r, n, top):
    """Lengths up to `top`, the largest among them; from three on one is 0 (an idle row of the batch)."""
    a = np.maximum(1, (top * (0.15 + 0.85 * r.rand(n))).astype(np.int64))
    a[r.randint(n)] = top
    if n >= 3:
        a[(int(np.argmax(a)) + 1 + r.randint(n - 1)) % n] = 0
    return a


def _tables(r, lens, page, pages=None):
    """Block tables of private pages in random order; -1 past each row's end."""
    need = -(-lens // page)
    total = int(need.sum())
    pages = max(1, total) if pages is None else pages
    ids, table, at = r.permutation(pages), np.full((len(lens), max(1, int(need.max()))), -1, np.int32), 0
    for i, n in enumerate(need):
        table[i, :n] = ids[at:at + n]
        at += n
    return table, pages


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = _host_rng(seed)
    c, k = case, case["kind"]
    if k == "attend":
        lens, n_new = _sizes(c)
        table, pages = _tables(r, lens, c["page"])
        codes, scales = _pool(g, pages, c["n_kv"], c["page"], c["hd"])
        T = int(n_new.sum())
        # the queries are a slice of the projection's rows, as in the model
        width = (c["n_q"] + 2 * c["n_kv"]) * c["hd"]
        qkv = (1.5 * torch.randn((T, width), device="cuda", generator=g)).to(torch.bfloat16)
        q = qkv[:, :c["n_q"] * c["hd"]].unflatten(1, (c["n_q"], c["hd"]))
        cu = np.zeros(c["S"] + 1, np.int32)
        np.cumsum(n_new, out=cu[1:])
        return {"case": c, "q": q, "codes": codes, "scales": scales, "table": _dev(table),
                "lens": _dev(lens.astype(np.int32)), "cu": _dev(cu) if c["max_q"] > 1 else None,
                "max_q": int(n_new.max()), "max_len": int(lens.max()), "softmax_scale": 1.0 / math.sqrt(c["hd"])}
    if k == "append":
        past, n_new = _sizes(c)
        table, pages = _tables(r, past + n_new, c["page"])
        codes, scales = _pool(g, pages, c["n_kv"], c["page"], c["hd"])
        cu = np.zeros(c["S"] + 1, np.int32)
        np.cumsum(n_new, out=cu[1:])
        width, at = (c["n_q"] + 2 * c["n_kv"]) * c["hd"], c["n_q"] * c["hd"]
        qkv = torch.randn((int(cu[-1]), width), device="cuda", generator=g).to(torch.bfloat16)
        kv = qkv[:, at:].unflatten(1, (2, c["n_kv"], c["hd"]))
        first = past // c["page"]
        row = np.concatenate([np.full(-(-(p + n) // c["page"]) - f if n else 0, i)
                              for i, (p, n, f) in enumerate(zip(past, n_new, first))]).astype(np.int64)
        slot = np.concatenate([np.arange(f, -(-(p + n) // c["page"])) if n else np.arange(0)
                               for p, n, f in zip(past, n_new, first)]).astype(np.int64)
        start = first * c["page"]
        return {"case": c, "k": kv[:, 0], "v": kv[:, 1], "codes": codes, "scales": scales, "table": _dev(table),
                "past": _dev(past.astype(np.int32)), "cu": _dev(cu), "max_new": int(n_new.max()),
                # the pages that the call touches, and the ranges read back from them
                "row": _dev(row), "slot": _dev(slot), "start": _dev(start.astype(np.int32)),
                "count": _dev((past + n_new - start).astype(np.int32)),
                "max_count": max(1, int((past + n_new - start).max()))}
    if k == "pages":
        R, P = c["rows"], c["page"]
        lens, n_new = _sizes(c)
        table, _ = _tables(r, lens, P, c["pages"])
        table = np.concatenate([table, np.full((R, 2), -1, np.int32)], 1)
        if c["action"] == "fork":  # rows in fours share the whole pages of a common beginning
            for i in range(R):
                lead = i - i % 4
                n = min(lens[lead] // P, lens[i] // P) // 2
                table[i, :n] = table[lead, :n]
        refs = np.bincount(table[table >= 0], minlength=c["pages"]).astype(np.int32)
        codes, scales = _pool(g, c["pages"], c["n_kv"], P, c["hd"], c["layers"])
        parents = np.where(r.rand(R) < 0.05, -1, np.sort(r.randint(0, max(1, R // 2), size=R) * 2 % R)).astype(np.int32)
        return {"case": c, "codes": codes, "scales": scales, "table": _dev(table), "lens": _dev(lens.astype(np.int32)),
                "refs": _dev(refs), "parents": _dev(parents), "n_new": _dev(n_new.astype(np.int32))}
    if k == "logits":
        # rows of a language model's logits: a broad bulk, some rows sharply peaked, the padding ids at -inf
        x = torch.randn((c["T"], c["V"]), device="cuda", generator=g)
        x *= torch.linspace(1, 4, c["T"], device="cuda")[:, None]
        x[:, torch.randint(c["V"], (8,), device="cuda", generator=g)] += 12
        x[:, c["V"] - c["V"] // 100:] = -math.inf
        x = x.to(torch.bfloat16) if c["bf16"] else x
        t = torch.randint(c["V"] - c["V"] // 100, (c["T"],), device="cuda", generator=g, dtype=torch.int32)
        return {"case": c, "logits": x, "targets": t}
    h = torch.randn((c["T"], c["H"]), device="cuda", generator=g)
    w = torch.empty((c["V"], c["H"]), dtype=torch.bfloat16, device="cuda")
    for part in w.split(16384):
        part.copy_(torch.randn(part.shape, device="cuda", generator=g).mul_(2.5 / math.sqrt(c["H"])))
    t = torch.randint(c["V"], (c["T"],), device="cuda", generator=g, dtype=torch.int32)
    return {"case": c, "h": h.to(torch.bfloat16), "w": w, "targets": t, "scale": 1.0}


# ------------------------------------------------------------------------------------------------ one pass
def run(state):
    return {"attend": _run_attend, "append": _run_append, "pages": _run_pages, "logits": _run_logits,
            "score": _run_score}[state["case"]["kind"]](state)


def _values(codes, scales):
    """Keys and values that the pages [n, 2, n_kv, page, hd] stand for, f32 [n, page, n_kv, hd]."""
    n, _, n_kv, page, hd = codes.shape
    x = codes.float() * scales[..., None, None]
    k = x[:, 0].transpose(1, 2)
    v = x[:, 1].reshape(n, n_kv, page // 4, hd, 4).transpose(3, 4).reshape(n, n_kv, page, hd).transpose(1, 2)
    return k, v


def _rows(pages, S):
    """[S * W, page, n_kv, hd] as [S, W * page, n_kv, hd]."""
    return pages.reshape(S, -1, *pages.shape[2:])


def _run_attend(s):
    if own:
        return _ops().attention_paged(s["q"], s["codes"], s["scales"], s["table"], s["lens"], cu_q=s["cu"],
                                      max_q=s["max_q"], max_len=s["max_len"], softmax_scale=s["softmax_scale"])
    q, S, n_kv = s["q"].float(), s["table"].shape[0], s["codes"].shape[2]
    T, n_q, hd = q.shape
    at = s["table"].clamp(min=0).long().reshape(-1)
    k, v = _values(s["codes"][at], s["scales"][at])
    k, v = _rows(k, S), _rows(v, S)  # [S, L, n_kv, hd]
    lens = s["lens"].long()
    cu = s["cu"].long() if s["cu"] is not None else torch.arange(S + 1, device=q.device)
    n_new = cu[1:] - cu[:-1]
    j = torch.arange(s["max_q"], device=q.device)
    pick = (cu[:-1, None] + j).clamp(max=max(T - 1, 0))  # [S, max_q]
    qs = q[pick].reshape(S, s["max_q"], n_kv, n_q // n_kv, hd).permute(0, 2, 1, 3, 4).flatten(2, 3)
    pos = lens[:, None] - n_new[:, None] + j  # a query's own position
    key = torch.arange(k.shape[1], device=q.device)
    see = (key <= pos[..., None]) & (key < lens[:, None, None])  # [S, max_q, L]
    x = (qs @ k.permute(0, 2, 3, 1)) * s["softmax_scale"]
    x = torch.where(see.repeat_interleave(n_q // n_kv, 1)[:, None], x, -math.inf)
    m = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(m == -math.inf, 0, m))
    z = p.sum(-1, keepdim=True)
    o = (p @ v.permute(0, 2, 1, 3)) / torch.where(z == 0, 1, z)
    lse = torch.where(z == 0, -math.inf, m + torch.log(z))
    group = (S, n_kv, s["max_q"], n_q // n_kv)
    o = o.reshape(*group, hd).permute(0, 2, 1, 3, 4).reshape(S * s["max_q"], n_q, hd)
    lse = lse.reshape(group).permute(0, 2, 1, 3).reshape(S * s["max_q"], n_q)
    tok = torch.arange(T, device=q.device)
    seq = torch.searchsorted(cu, tok, right=True) - 1
    back = seq * s["max_q"] + tok - cu[seq]
    return o[back].to(torch.bfloat16), lse[back]


def _run_append(s):
    if own:
        ops = _ops()
        ops.kv_append(s["k"], s["v"], s["codes"], s["scales"], s["table"], s["past"], cu_new=s["cu"],
                      max_new=s["max_new"])
        return ops.kv_read(s["codes"], s["scales"], s["table"], s["start"], s["count"], s["max_count"])
    codes, scales, table, past, cu = s["codes"], s["scales"], s["table"].long(), s["past"].long(), s["cu"].long()
    S, page = table.shape[0], codes.shape[3]
    row, slot = s["row"], s["slot"]
    at = table[row, slot]
    pos = slot[:, None] * page + torch.arange(page, device=row.device)  # [n, page]
    old = pos < past[row][:, None]
    new = ~old & (pos < (past + cu[1:] - cu[:-1])[row][:, None])
    tok = (cu[row][:, None] + pos - past[row][:, None]).clamp(0, max(s["k"].shape[0] - 1, 0))
    x = torch.stack([s["k"].float()[tok], s["v"].float()[tok]], 1).permute(0, 1, 3, 2, 4)  # [n, 2, n_kv, page, hd]
    on = new[:, None, None, :, None]
    x = torch.where(on, x, 0)
    was = torch.where(old.any(1)[:, None, None], scales[at], 0)
    now = torch.maximum(was, x.abs().amax((3, 4)) / torch.full((), 127.0, device=x.device))
    by = torch.where(now > 0, now, 1)[..., None, None]
    held = codes[at]  # [n, 2, n_kv, page, hd], the value plane in groups of four tokens
    kk, vv = held[:, 0], held[:, 1]
    vv = vv.reshape(*vv.shape[:2], page // 4, -1, 4).transpose(3, 4).reshape(vv.shape)
    held = torch.stack([kk, vv], 1)
    again = torch.round(held.float() * was[..., None, None] / by).to(torch.int8)
    fresh = torch.round(x / by).clamp(-127, 127).to(torch.int8)
    out = torch.where(on, fresh, torch.where(old[:, None, None, :, None], again, held))
    vv = out[:, 1].reshape(*kk.shape[:2], page // 4, 4, -1).transpose(3, 4).reshape(kk.shape)
    codes[at] = torch.stack([out[:, 0], vv], 1)
    scales[at] = now
    # read back
    want = s["start"].long()[:, None] + torch.arange(s["max_count"], device=row.device)
    inside = torch.arange(s["max_count"], device=row.device) < s["count"].long()[:, None]
    first = (s["start"].long() // page)[:, None] + torch.arange(-(-s["max_count"] // page) + 1, device=row.device)
    first = table[torch.arange(S, device=row.device)[:, None], first.clamp(max=table.shape[1] - 1)].clamp(min=0)
    k, v = _values(codes[first.reshape(-1)], scales[first.reshape(-1)])
    k, v = _rows(k, S), _rows(v, S)
    off = want - (s["start"].long() // page * page)[:, None]
    take = torch.arange(S, device=row.device)[:, None]
    zero = inside[..., None, None]
    return (torch.where(zero, k[take, off], 0).to(torch.bfloat16), torch.where(zero, v[take, off], 0).to(torch.bfloat16))


def _run_pages(s):
    c = s["case"]
    if own:
        ops = _ops()
        if c["action"] == "compact":
            table, refs, used = ops.kv_compact(s["codes"], s["scales"], s["table"], s["refs"])
            return {"table": table, "refs": refs, "used": used, "codes": s["codes"], "scales": s["scales"]}
        table, lens, refs = ops.kv_fork(s["codes"], s["scales"], s["table"], s["lens"], s["refs"], s["parents"])
        ops.kv_reserve(table, lens, refs, s["n_new"], c["page"])
        return {"table": table, "lens": lens, "refs": refs, "codes": s["codes"], "scales": s["scales"]}
    codes, scales, P = s["codes"], s["scales"], c["page"]
    pages, dev = codes.shape[1], codes.device
    ids = torch.arange(pages, device=dev)
    if c["action"] == "compact":
        live = s["refs"] > 0
        used = live.sum()
        moving = (live & (ids >= used)).nonzero().flatten()
        hole = (~live & (ids < used)).nonzero().flatten()
        to = ids.clone()
        to[moving] = hole
        codes[:, hole] = codes[:, moving]
        scales[:, hole] = scales[:, moving]
        refs = torch.where(ids < used, torch.zeros_like(s["refs"]).scatter_(0, to[live], s["refs"][live]), 0)
        table = torch.where(s["table"] >= 0, to[s["table"].clamp(min=0).long()], -1)
        return {"table": table.int(), "refs": refs.int(), "used": used.reshape(1).int(), "codes": codes, "scales": scales}
    par = s["parents"].long()
    R, W = par.shape[0], s["table"].shape[1]
    slot = torch.arange(W, device=dev)
    lens = torch.where(par >= 0, s["lens"].long()[par.clamp(min=0)], 0)
    n = (lens + P - 1) // P
    table = torch.where(slot < n[:, None], s["table"].long()[par.clamp(min=0)], -1)
    i = torch.arange(R, device=dev)
    again = ((par[:, None] == par) & (i < i[:, None])).any(1)  # an earlier row continues the same parent
    copy = again & (lens % P != 0)
    keeps = (table >= 0) & ~(copy[:, None] & (slot == n[:, None] - 1))
    refs = torch.zeros(pages, dtype=torch.long, device=dev).index_add_(0, table.clamp(min=0).flatten(), keeps.long().flatten())
    free = torch.argsort(refs > 0, stable=True)
    who = copy.nonzero().flatten()
    src, dst = table[who, n[who] - 1], free[:who.shape[0]]
    codes[:, dst] = codes[:, src]
    scales[:, dst] = scales[:, src]
    table[who, n[who] - 1] = dst
    refs[dst] = 1
    # the pages of the next tokens
    more = (lens + s["n_new"].long() + P - 1) // P
    wants = (slot >= n[:, None]) & (slot < more[:, None])
    free = torch.argsort(refs > 0, stable=True)
    rank = wants.flatten().cumsum(0).reshape(R, W) - 1
    table = torch.where(wants, free[rank.clamp(min=0)], table)
    refs = refs.index_add_(0, table.clamp(min=0).flatten(), wants.long().flatten())
    return {"table": table.int(), "lens": lens.int(), "refs": refs.int(), "codes": codes, "scales": scales}


def _stats(x, t):
    """(log-probability of t, entropy) of rows x, f32."""
    m = x.amax(-1, keepdim=True)
    u = x - m
    e = torch.exp(u)
    z = e.sum(-1)
    ue = torch.where(e > 0, u * e, 0).sum(-1)
    own_u = u.gather(1, t.long()[:, None])[:, 0]
    return own_u - torch.log(z), torch.log(z) - ue / z


def _run_logits(s):
    if own:
        return _ops().token_logprobs(s["logits"], s["targets"], top_k=s["case"]["k"])
    x, t, k = s["logits"].float(), s["targets"].long(), s["case"]["k"]
    lp, ent = _stats(x, t)
    mine = x.gather(1, t[:, None])
    rank = (x > mine).sum(-1).int() + 1
    # the lowest index first among equals: the largest of whole numbers that hold (value, V - index)
    key = (x + 0.0).view(torch.int32)
    key = torch.where(key < 0, key ^ 0x7FFFFFFF, key).long() * x.shape[1]
    idx = (key + torch.arange(x.shape[1] - 1, -1, -1, device=x.device)).topk(k, -1)[1]
    val = x.gather(1, idx)
    m = x.amax(-1, keepdim=True)
    z = torch.exp(x - m).sum(-1, keepdim=True)
    return lp, ent, rank, idx.int(), val - m - torch.log(z)


def _run_score(s):
    if own:
        return _ops().score_tokens(s["h"], s["w"], s["targets"], logit_scale=s["scale"])
    return _stats((s["h"].float() @ s["w"].float().T) * s["scale"], s["targets"])


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    c, k = case, case["kind"]
    if k in ("attend", "append"):
        row = 2 * c["n_kv"] * c["hd"]  # keys and values of a token
    if k == "attend":
        lens, n = _sizes(c)
        T, L = float(n.sum()), float(lens.sum())
        b = L * row + L / c["page"] * (2 * c["n_kv"] * 4 + 4) + T * c["n_q"] * (4 * c["hd"] + 4)
        return {"bytes": b, "flops": 4.0 * c["hd"] * c["n_q"] * float((n * np.maximum(0, lens - (n - 1) / 2)).sum())}
    if k == "append":
        past, new = _sizes(c)
        T = float(new.sum())
        back = T + float((past % c["page"]).sum())  # what is read again and written as bf16
        b = T * row * 3 + back * row * 3
        return {"bytes": float(b), "flops": 4.0 * T * row}
    if k == "pages":
        size = c["layers"] * 2 * c["n_kv"] * (c["page"] * c["hd"] + 4)
        moved = 0.45 * c["rows"] if c["action"] == "fork" else _movers(c)
        meta = 4 * (2 * c["rows"] * (-(-c["max_len"] // c["page"]) + 2) + 2 * c["pages"] + 3 * c["rows"])
        return {"bytes": float(2 * moved * size + meta), "flops": 0.0}
    if k == "logits":
        b = c["T"] * (c["V"] * (2 if c["bf16"] else 4) + 16 + 8 * c["k"])
        return {"bytes": float(b), "flops": 4.0 * c["T"] * c["V"]}
    b = 2 * (c["T"] + c["V"]) * c["H"] + 12 * c["T"]
    return {"bytes": float(b), "flops": 2.0 * c["T"] * c["V"] * c["H"]}


def _movers(c):
    """Live pages above the live count, when the live ones are spread evenly."""
    live = min(c["pages"], c["rows"] * 0.75 * c["max_len"] / c["page"] + c["rows"] / 2)
    return live * (c["pages"] - live) / c["pages"]


# ------------------------------------------------------------------------------------------------ 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return {"attend": _exact_attend, "append": _exact_append, "pages": _exact_pages, "logits": _exact_logits,
            "score": _exact_score}[case["kind"]](s)


def _planes(s, ids, layer=None):
    """One sequence's keys and values in 64 bits, [n * page, n_kv, hd], from its page ids."""
    codes, scales = s["codes"][ids].double(), s["scales"][ids].double()
    n, _, n_kv, page, hd = codes.shape
    k = torch.einsum("nhtd,nh->nthd", codes[:, 0], scales[:, 0]).reshape(n * page, n_kv, hd)
    v = torch.einsum("nhgdf,nh->ngfhd", codes[:, 1].reshape(n, n_kv, page // 4, hd, 4), scales[:, 1])
    return k, v.reshape(n * page, n_kv, hd)


def _exact_attend(s):
    q, page = s["q"].double(), s["codes"].shape[3]
    T, n_q, hd = q.shape
    n_kv = s["codes"].shape[2]
    lens = s["lens"].tolist()
    cu = s["cu"].tolist() if s["cu"] is not None else list(range(len(lens) + 1))
    out, lse = torch.zeros_like(q), torch.full((T, n_q), -math.inf, dtype=torch.float64, device=q.device)
    for i, n in enumerate(lens):
        a, b = cu[i], cu[i + 1]
        if n == 0 or a == b:
            continue
        k, v = _planes(s, s["table"][i, :-(-n // page)].long())
        for h in range(n_q):
            x = q[a:b, h] @ k[:n, h * n_kv // n_q].T * s["softmax_scale"]
            late = torch.arange(n, device=q.device) > torch.arange(n - (b - a), n, device=q.device)[:, None]
            x = x.masked_fill(late, -math.inf)
            lse[a:b, h] = torch.logsumexp(x, -1)
            out[a:b, h] = torch.softmax(x, -1) @ v[:n, h * n_kv // n_q]
    return out, lse


def _exact_append(s):
    codes, scales, page = s["codes"], s["scales"], s["codes"].shape[3]
    past, cu = s["past"].tolist(), s["cu"].tolist()
    count, start, table = s["count"].tolist(), s["start"].tolist(), s["table"].tolist()
    S, n_kv, hd = len(past), codes.shape[2], codes.shape[4]
    out = [torch.zeros((S, s["max_count"], n_kv, hd), dtype=torch.float64, device=codes.device) for _ in range(2)]
    for i in range(S):
        if cu[i] == cu[i + 1]:  # nothing new: the range reads as it was
            if count[i]:
                k, v = _planes(s, torch.tensor([table[i][start[i] // page]], device=codes.device))
                out[0][i, :count[i]], out[1][i, :count[i]] = k[:count[i]], v[:count[i]]
            continue
        ids = torch.tensor(table[i][start[i] // page:-(-(past[i] + cu[i + 1] - cu[i]) // page)], device=codes.device)
        had = past[i] - start[i]  # tokens of the first page that were there
        before = _planes(s, ids[:1]) if had else None
        for w, x in enumerate((s["k"], s["v"])):
            y = torch.zeros((len(ids) * page, n_kv, hd), dtype=torch.float64, device=codes.device)
            y[had:count[i]] = x[cu[i]:cu[i + 1]].double()
            y = y.reshape(len(ids), page, n_kv, hd)
            top = y.abs().amax((1, 3)) / 127
            if had:
                top[0] = torch.maximum(top[0], scales[ids[0], w].double())
                y[0, :had] = before[w][:had]
            by = torch.where(top > 0, top, 1)[:, None, :, None]
            y = (torch.round(y / by) * by).reshape(-1, n_kv, hd)
            out[w][i, :count[i]] = y[:count[i]]
    return out[0], out[1]


def _exact_pages(s):
    """The scales, moved by a walk over the rows on the host; ids and codes are whole numbers and have to be equal."""
    c, P = s["case"], s["case"]["page"]
    scales, refs = s["scales"].double(), s["refs"].tolist()
    if c["action"] == "compact":
        used = sum(n > 0 for n in refs)
        holes = [p for p in range(used) if refs[p] == 0]
        for p, q in zip(holes, [p for p in range(used, len(refs)) if refs[p] > 0]):
            scales[:, p] = scales[:, q]
        return {"table": None, "refs": None, "used": None, "codes": None, "scales": scales}
    table, lens, par = s["table"].tolist(), s["lens"].tolist(), s["parents"].tolist()
    listed_, seen, jobs = set(), set(), []
    for p in par:
        if p < 0:
            continue
        n = -(-lens[p] // P)
        part = lens[p] % P != 0 and p in seen
        listed_.update(table[p][:n - 1] if part else table[p][:n])
        if part:
            jobs.append(table[p][n - 1])
        seen.add(p)
    free = [p for p in range(len(refs)) if p not in listed_]
    for src, dst in zip(jobs, free):
        scales[:, dst] = s["scales"][:, src].double()
    return {"table": None, "lens": None, "refs": None, "codes": None, "scales": scales}


def _exact_logits(s):
    x, t, k = s["logits"], s["targets"].long(), s["case"]["k"]
    out = [[], [], []]
    for a in range(0, x.shape[0], 256):
        lp = torch.log_softmax(x[a:a + 256].double(), -1)
        out[0].append(lp.gather(1, t[a:a + 256, None])[:, 0])
        out[1].append(-(lp.exp() * torch.where(lp == -math.inf, 0, lp)).sum(-1))
        out[2].append(lp.topk(k, -1)[0] if k else lp[:, :0])
    return torch.cat(out[0]), torch.cat(out[1]), None, None, torch.cat(out[2])


def _exact_score(s):
    lp, ent, w = [], [], s["w"].double()
    for a in range(0, s["h"].shape[0], 1024):
        x = torch.log_softmax(s["h"][a:a + 1024].double() @ w.T * s["scale"], -1)
        lp.append(x.gather(1, s["targets"][a:a + 1024, None].long())[:, 0])
        ent.append(-(x.exp() * x).sum(-1))
    return torch.cat(lp), torch.cat(ent)
