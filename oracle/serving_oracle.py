"""Plain restatement in numpy (64-bit) of the serving operators of include/wmi.h: wmi_paged_plan, wmi_paged_write,
wmi_paged_attention, wmi_sample_tokens. What tests/test_gpu_serving.py and tests/test_cpu_serving.py compare with, used there only."""
import numpy as np


def to_bf16(x):
    """float array -> bfloat16 bit patterns (uint16), round to nearest even; NaN stays NaN"""
    u = np.ascontiguousarray(x, np.float32).view(np.uint32)
    r = ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7FC0), r)


def from_bf16(b):
    return (np.asarray(b, np.uint16).astype(np.uint32) << 16).view(np.float32)


def plan(ctx, new, free, page, table, cap):
    """-> table, cu_q, kv_lens, slots, positions, counts"""
    table = table.copy()
    cols, cu, kv, slots, positions = table.shape[1], [0], [], [], []
    taken = bad = 0
    first_out = None
    for i, (c, n) in enumerate(zip(map(int, ctx), map(int, new))):
        if c < 0 or n < 0 or c + n > cols * page:
            bad += 1
            kv.append(0)
            cu.append(cu[-1])
            continue
        lo, hi = -(-c // page), -(-(c + n) // page)
        if first_out is None and (cu[-1] + n > cap or taken + hi - lo > len(free)):
            first_out = i
        if first_out is not None:
            kv.append(c)
            cu.append(cu[-1])
            continue
        for j in range(lo, hi):
            table[i, j] = free[taken]
            taken += 1
        for p in range(c, c + n):
            pg = int(table[i, p // page])
            slots.append(pg * page + p % page if pg >= 0 and pg * page + p % page < 2 ** 31 else -1)
            positions.append(p)
        kv.append(c + n)
        cu.append(cu[-1] + n)
    pad = cap - len(slots)
    i32 = lambda v: np.asarray(v, np.int32)
    return table, i32(cu), i32(kv), i32(slots + [-1] * pad), i32(positions + [0] * pad), i32([len(ctx) if first_out is None else first_out, cu[-1], taken, bad])


def attention(q, k, v, table, cu, kv_lens, page, scale, window=0):
    """q [rows][hq][d], k and v [pages][page][hkv][d] (float64 values of what the device holds). -> out, mass, reach:
    mass[row][hq][d] = sum_j p_j |v_j| (what a relative error of the probabilities can move), reach[row][hq] = the largest
    scale sum_d |q_d k_d| over the visible keys (what the rounding of a score is relative to)"""
    rows, hq, d = q.shape
    n_pages, hkv = k.shape[0], k.shape[2]
    out, mass, reach = np.full(q.shape, np.nan), np.zeros(q.shape), np.zeros((rows, hq))
    for i in range(len(kv_lens)):
        n = int(cu[i + 1] - cu[i])
        length = min(max(int(kv_lens[i]), 0), table.shape[1] * page)
        for t in range(n):
            pos = length - n + t
            js = np.arange(max(0, pos - window + 1) if window > 0 else 0, pos + 1)
            pg = table[i, js // page] if len(js) else js
            ok = (pg >= 0) & (pg < n_pages)
            js, pg = js[ok], pg[ok]
            r = int(cu[i]) + t
            if not len(js):
                out[r] = 0.0
                continue
            for h in range(hq):
                kk, vv = k[pg, js % page, h // (hq // hkv)], v[pg, js % page, h // (hq // hkv)]
                s = scale * (kk @ q[r, h])
                p = np.exp(s - s.max())
                p /= p.sum()
                out[r, h] = p @ vv
                mass[r, h] = p @ np.abs(vv)
                reach[r, h] = (abs(scale) * (np.abs(kk) @ np.abs(q[r, h]))).max()
    return out, mass, reach


def sample(x, uniform, temperature=None, top_k=None, top_p=None, min_p=None):
    """-> token, logprob, distance: how far (relative to the kept mass) the uniform number is from the next border of the draw or of
    top_p; a draw nearer than the arithmetic resolves may go either way"""
    rows, V = x.shape
    tok, lp = np.full(rows, -1, np.int32), np.full(rows, -np.inf)
    dist = np.full(rows, np.inf)
    for r in range(rows):
        row = np.where(np.isnan(x[r]), -np.inf, x[r].astype(np.float64))
        top = row.max()
        if top == -np.inf:
            continue
        t = 1.0 if temperature is None else float(temperature[r])
        drawn = t > 0
        t = t if drawn else 1.0
        with np.errstate(invalid="ignore", over="ignore"):
            e = np.where(row == top, 0.0, (row - top) / t)
        w = np.where(row == -np.inf, 0.0, np.exp(e))
        order = np.lexsort((np.arange(V), -row))
        order = order[row[order] > -np.inf]
        n = len(order) if drawn else 1
        if drawn and top_k is not None and top_k[r] > 0:
            n = min(n, int(top_k[r]))
        if drawn and top_p is not None and top_p[r] < 1:
            head = w[order[:n]]
            before = np.cumsum(head) - head
            lim = float(np.float32(top_p[r])) * head.sum()
            dist[r] = min(dist[r], np.abs(before[1:] - lim).min(initial=np.inf) / head.sum())
            n = max(1, int((before < lim).sum()))
        kept = order[:n]
        if drawn and min_p is not None and min_p[r] > 0:
            kept = kept[(w[kept] >= float(np.float32(min_p[r]))) | (kept == order[0])]
        kept = np.sort(kept)
        c = np.cumsum(w[kept])
        u = float(uniform[r])
        u = min(u, 1 - 2.0 ** -24) if u > 0 else 0.0
        target = u * c[-1]
        live = np.nonzero(w[kept] > 0)[0]
        j = min(int((c <= target).sum()), int(live[-1]))
        if drawn:
            dist[r] = min(dist[r], np.abs(c - target).min() / c[-1] if u > 0 else np.inf)
        tok[r] = kept[j]
        lp[r] = e[kept[j]] - np.log(w.sum())
    return tok, lp, dist
