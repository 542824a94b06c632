"""Plain implementations, in 64 bits on the CPU, of the operators over the 8-bit paged cache, and the inputs that
their tests share."""
import math

import numpy as np
import torch


def planes(codes, scales, ids):
    """Keys and values that pages `ids` of one layer stand for, f64 [len(ids) * page, n_kv, hd]."""
    c, s = codes[ids].double(), scales[ids].double()
    n, _, n_kv, page, hd = c.shape
    k = (c[:, 0] * s[:, 0, :, None, None]).permute(0, 2, 1, 3)
    v = c[:, 1].reshape(n, n_kv, page // 4, hd, 4).permute(0, 2, 4, 1, 3).reshape(n, page, n_kv, hd)
    return k.reshape(n * page, n_kv, hd), (v * s[:, 1, None, :, None]).reshape(n * page, n_kv, hd)


def attend(q, codes, scales, table, lens, cu, scale):
    """(out, lse, |values| weighted by the probabilities, bound of the scores' f32 error), all f64."""
    T, n_q, hd = q.shape
    page, n_kv = codes.shape[3], codes.shape[2]
    out, av = torch.zeros(T, n_q, hd, dtype=torch.float64), torch.zeros(T, n_q, hd, dtype=torch.float64)
    lse, err = torch.full((T, n_q), -math.inf, dtype=torch.float64), torch.zeros(T, n_q, dtype=torch.float64)
    for r, n in enumerate(lens):
        a, b = int(cu[r]), int(cu[r + 1])
        if n == 0 or a == b:
            continue
        k, v = planes(codes, scales, table[r, :-(-n // page)].long())
        for t in range(a, b):
            see = n - (b - a) + (t - a) + 1
            if see <= 0:
                continue
            for h in range(n_q):
                g = h // (n_q // n_kv)
                qq = q[t, h].double()
                x = k[:see, g] @ qq * scale
                p = torch.softmax(x, 0)
                out[t, h], av[t, h], lse[t, h] = p @ v[:see, g], p @ v[:see, g].abs(), torch.logsumexp(x, 0)
                # hd products summed in f32, then a few roundings of the scaled score and of the exponent
                err[t, h] = ((k[:see, g].abs() @ qq.abs()) * scale).max() * (hd + 8) * 2.0 ** -24
    return out, lse, av, err


def pool(pages, n_kv, page, hd, seed, layers=None):
    g = torch.Generator().manual_seed(seed)
    lead = (pages,) if layers is None else (layers, pages)
    codes = torch.randint(-127, 128, (*lead, 2, n_kv, page, hd), generator=g, dtype=torch.int8)
    scales = 0.005 + 0.02 * torch.rand((*lead, 2, n_kv), generator=g)
    return codes, scales


def tables(lens, page, pages, seed, width=None):
    r = np.random.RandomState(seed)
    ids, at = r.permutation(pages), 0
    need = [-(-int(n) // page) for n in lens]
    t = np.full((len(lens), width or max(1, max(need))), -1, np.int32)
    for i, n in enumerate(need):
        t[i, :n] = ids[at:at + n]
        at += n
    return torch.from_numpy(t)


def append(k, v, codes, scales, table, lens, cu):
    """The append's definition, in place on CPU tensors, in f32 as it is defined (each step rounded once)."""
    page, n_kv, hd = codes.shape[3], codes.shape[2], codes.shape[4]
    f = np.float32
    for r, n0 in enumerate(lens):
        n0, m = int(n0), int(cu[r + 1] - cu[r])
        for slot in range(n0 // page, -(-(n0 + m) // page) if m else 0):
            p = int(table[r, slot])
            lo, hi = slot * page, min((slot + 1) * page, n0 + m)
            old, new0 = max(0, n0 - lo), max(lo, n0)
            for w, x in enumerate((k, v)):
                for h in range(n_kv):
                    new = x[int(cu[r]) + new0 - n0:int(cu[r]) + hi - n0, h].float().numpy()
                    was = f(scales[p, w, h]) if old else f(0)
                    top = f(np.abs(new).max())
                    now = f(np.nan) if not np.isfinite(top) or np.isnan(was) else max(was, f(top / f(127)))
                    by = now if np.isfinite(now) and now > 0 else f(1)
                    rows = codes[p, w, h]
                    rows = (rows.reshape(page // 4, hd, 4).permute(0, 2, 1).reshape(page, hd) if w else rows).numpy().copy()
                    if np.isnan(now):
                        rows[:hi - lo] = 0
                    else:
                        if old and now != was:
                            rows[:old] = np.rint((rows[:old].astype(f) * was) / by).astype(np.int8)
                        rows[old:hi - lo] = np.clip(np.rint(new / by), -127, 127).astype(np.int8)
                    rows = torch.from_numpy(rows)
                    codes[p, w, h] = rows.reshape(page // 4, 4, hd).permute(0, 2, 1).reshape(page, hd) if w else rows
                    scales[p, w, h] = float(now)


def fork(codes, scales, table, lens, parents, pages):
    """New (table, lens, refs) by a walk over the rows; the pool in place."""
    page, width = codes.shape[4], table.shape[1]
    t = torch.full((len(parents), width), -1, dtype=torch.int32)
    ln, refs, seen, jobs = torch.zeros(len(parents), dtype=torch.int32), torch.zeros(pages, dtype=torch.int32), set(), []
    for i, p in enumerate(parents):
        p = int(p)
        if p < 0:
            continue
        n, ln[i] = -(-int(lens[p]) // page), lens[p]
        t[i, :n] = table[p, :n]
        if p in seen and int(lens[p]) % page:
            jobs.append((i, n - 1))
        seen.add(p)
        for j in range(n - 1 if (i, n - 1) in jobs else n):
            refs[t[i, j]] += 1
    free = [q for q in range(pages) if refs[q] == 0]
    for (i, j), q in zip(jobs, free):
        codes[:, q], scales[:, q] = codes[:, t[i, j]].clone(), scales[:, t[i, j]].clone()
        t[i, j], refs[q] = q, 1
    return t, ln, refs


def reserve(table, lens, refs, n_new, page):
    free = [q for q in range(len(refs)) if refs[q] == 0]
    for i in range(table.shape[0]):
        for j in range(int(lens[i]) // page, -(-(int(lens[i]) + int(n_new[i])) // page)):
            if table[i, j] < 0:
                table[i, j] = free.pop(0)
                refs[table[i, j]] = 1


def compact(codes, scales, table, refs):
    used = int((refs > 0).sum())
    holes, to = [p for p in range(used) if refs[p] == 0], {-1: -1}
    new = torch.zeros_like(refs)
    for p in range(len(refs)):
        if refs[p] > 0:
            to[p] = p if p < used else holes.pop(0)
            new[to[p]] = refs[p]
            if to[p] != p:
                codes[:, to[p]], scales[:, to[p]] = codes[:, p].clone(), scales[:, p].clone()
    return torch.tensor([[to[int(p)] for p in row] for row in table], dtype=torch.int32), new, used


def scores(x, targets, k):
    """(logprobs, entropy, ranks, top ids, top logprobs) of f64 rows, numbers before NaN, lower ids first."""
    x = x.double()
    T, V = x.shape
    out = [np.zeros(T), np.zeros(T), np.zeros(T, np.int64), np.zeros((T, k), np.int64), np.zeros((T, k))]
    for t in range(T):
        row = x[t].numpy()
        live = row[row != -np.inf]
        bad = np.isnan(row).any() or np.isposinf(row).any()
        m = live.max() if len(live) and not bad else 0.0
        z = np.exp(live - m).sum() if not bad else np.nan
        with np.errstate(invalid="ignore"):
            # (row - m) - ln z, so that rows of the type's lowest value do not lose ln z
            lp = np.where(row == -np.inf, -np.inf, row - m - np.log(z)) if len(live) else np.full(V, -np.inf)
            if bad:
                lp = np.full(V, np.nan)
            p = np.exp(lp)
            out[1][t] = np.nan if bad else -(p[p > 0] * lp[p > 0]).sum()
        g = int(targets[t])
        if 0 <= g < V:
            out[0][t] = lp[g]
            out[2][t] = 1 + ((row > row[g]) | (np.isnan(row[g]) & ~np.isnan(row))).sum()
        key = np.where(np.isnan(row), -np.inf, row)
        order = np.lexsort((np.arange(V), -key, np.isnan(row)))[:k]
        out[3][t], out[4][t] = order, lp[order]
    return out
