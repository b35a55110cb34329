"""Cases of the serving operators (page plan, K/V write, attention over the paged cache, token draw): inputs, the operators'
plain forms in elementary torch operations, their 64-bit definitions, and the calls a program makes of the framework's own."""
import math
import random

import numpy as np
import torch

own = False

DEV = "cuda"
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
NEG = float("-inf")


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one decode step of a batch: 64 sequences of the decoder (text context 448 = 28 pages of 16), one new token each
        dict(name="plan_step", op="plan", n_seq=64, page=16, cols=28, new_lo=1, new_hi=1, long_share=0.0, full=0.85, spare=8),
        # the admission step of a busy server: thousands of requests, a fifth of them with a chunk of prompt, the rest one token
        dict(name="plan_admit", op="plan", n_seq=4096, page=64, cols=512, new_lo=1, new_hi=700, long_share=0.2, full=0.9, spare=100),
        # the same decode step's K and V into the decoder's head-major pages
        dict(name="write_step", op="write", n=64, pad=0, heads=20, dim=64, page=16, dtype="f16", head_major=True),
        # a chunk of prompts of many requests, padded at its end, into token-major pages
        dict(name="write_prompt", op="write", n=40000, pad=123, heads=8, dim=128, page=64, dtype="bf16", head_major=False),
        # the step of one clip's beams: five short sequences, as many key as query heads (latency)
        dict(name="attn_clip_step", op="attn", n_seq=5, new_lo=1, new_hi=1, ctx_lo=100, ctx_hi=440, hq=20, hkv=20, dim=64, page=16, window=0, dtype="f16", head_major=True),
        # a decode step of an ordinary batch with shared key heads and ragged lengths
        dict(name="attn_batch_step", op="attn", n_seq=64, new_lo=1, new_hi=1, ctx_lo=17, ctx_hi=8191, hq=32, hkv=8, dim=128, page=64, window=0, dtype="bf16", head_major=False),
        # a few very long sequences, one token each: the keys have to be split
        dict(name="attn_long_step", op="attn", n_seq=3, new_lo=1, new_hi=1, ctx_lo=90000, ctx_hi=131071, hq=32, hkv=8, dim=128, page=128, window=0, dtype="f16", head_major=False),
        # the prompt pass of a batch of clips with text context: up to half of the 448 positions
        dict(name="attn_prompt", op="attn", n_seq=64, new_lo=3, new_hi=224, ctx_lo=0, ctx_hi=0, hq=20, hkv=20, dim=64, page=16, window=0, dtype="f16", head_major=True),
        # chunks of new tokens over contexts that are cached already: the compute-bound end
        dict(name="attn_chunk", op="attn", n_seq=3, new_lo=3500, new_hi=4097, ctx_lo=20000, ctx_hi=28500, hq=32, hkv=8, dim=128, page=64, window=0, dtype="bf16", head_major=False),
        # the five draws of one clip's fallback at a temperature
        dict(name="sample_clip", op="sample", rows=5, vocab=51866, dtype="f32", mix="temperature", spread=3.0),
        # the draws of a whole batch, every filter in use somewhere
        dict(name="sample_batch", op="sample", rows=1024, vocab=51866, dtype="f32", mix="all", spread=2.0),
        # a wider vocabulary in 16 bits (many equal values)
        dict(name="sample_wide", op="sample", rows=48, vocab=131071, dtype="bf16", mix="all", spread=3.0),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["plan", "write", "attn", "attn", "attn", "sample", "sample"])
    if op == "plan":
        n = _log_int(rng, 1, 4096)
        cols = _log_int(rng, 4, 512)
        page = rng.choice([8, 16, 32, 64, 128])
        return dict(op=op, n_seq=n, page=page, cols=cols, new_lo=1, new_hi=_log_int(rng, 1, min(700, page * cols // 2)), long_share=rng.choice([0.0, 0.1, 0.2, 1.0]),
                    full=rng.uniform(0.2, 1.0), spare=rng.choice([0, 1, 8, 100, -max(1, n // 9)]))
    if op == "write":
        return dict(op=op, n=_log_int(rng, 1, 40000), pad=rng.choice([0, 0, 1, 37]), heads=rng.choice([1, 2, 5, 6, 8, 20]), dim=rng.choice([40, 64, 80, 128]),
                    page=rng.choice([8, 16, 32, 64, 128]), dtype=rng.choice(["f16", "bf16"]), head_major=rng.random() < 0.5)
    if op == "sample":
        vocab = _log_int(rng, 100, 131071)
        return dict(op=op, rows=_log_int(rng, 1, min(1024, 53000000 // vocab)), vocab=vocab, dtype=rng.choice(["f32", "f16", "bf16"]),
                    mix=rng.choice(["temperature", "top_k", "top_p", "min_p", "greedy", "all"]), spread=rng.choice([0.5, 2.0, 3.0, 6.0]))
    hkv = rng.choice([1, 2, 4, 8, 20])
    group = rng.choice([1, 1, 2, 3, 4, 5, 8]) if hkv <= 8 else 1
    dim = rng.choice([40, 64, 80, 128, 128])
    kind = rng.choice(["step", "few", "chunk"])
    n_seq = _log_int(rng, 1, 64)
    new_hi = {"step": 1, "few": rng.randint(2, 12), "chunk": _log_int(rng, 13, 4097)}[kind]
    ctx_hi = _log_int(rng, 1, 131071 if kind != "chunk" else 28500)
    c = dict(op=op, n_seq=max(1, min(n_seq, 12000 // new_hi)), new_lo=1, new_hi=new_hi, ctx_lo=rng.choice([0, ctx_hi // 2]), ctx_hi=ctx_hi, hq=hkv * group, hkv=hkv, dim=dim,
             page=rng.choice([8, 16, 32, 64, 128]), window=rng.choice([0, 0, 0, _log_int(rng, 1, 8192)]), dtype=rng.choice(["f16", "bf16"]),
             head_major=rng.random() < 0.3)
    # no dearer than the dearest listed one: keys' bytes and operations, from the longest lengths
    n, length = c["n_seq"], ctx_hi + new_hi
    while n > 1 and (4 * n * length * hkv * dim > 1.3e9 or 4 * n * new_hi * length * c["hq"] * dim > 5e12):
        n -= 1
    c["n_seq"] = n
    return c


# ------------------------------------------------------------------------------------------------ inputs
def _new_lengths(c):
    """fixed by the case, so that every seed's outputs have one shape"""
    r = random.Random("%s %d %d %d" % (c["op"], c["n_seq"], c["new_lo"], c["new_hi"]))
    share = c.get("long_share", 1.0)
    return [r.randint(c["new_lo"], c["new_hi"]) if r.random() < share else c["new_lo"] for _ in range(c["n_seq"])]


def _plan_lengths(c, r):
    room, new = c["page"] * c["cols"], _new_lengths(c)
    return [r.randint(0, max(0, min(int(room * c["full"]), room - k))) for k in new], new


def _attn_lengths(c, r):
    return [r.randint(c["ctx_lo"], c["ctx_hi"]) for _ in range(c["n_seq"])], _new_lengths(c)


def _pages(n, page):
    return (n + page - 1) // page


def _cache(n_pages, c, gen):
    """[n_pages + 1][page][heads][dim] views of K and V; the last page takes what padded rows write in the plain form"""
    h = c.get("heads") or c["hkv"]
    shape = (n_pages + 1, h, c["page"], c["dim"]) if c["head_major"] else (n_pages + 1, c["page"], h, c["dim"])
    out = []
    for _ in range(2):
        t = torch.empty(shape, dtype=DTYPES[c["dtype"]], device=DEV).normal_(generator=gen)
        out.append(t.transpose(1, 2) if c["head_major"] else t)
    return out


def prepare(case, seed):
    c, r = case, random.Random(seed * 1000003 + 17)
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
    s = {"case": c}
    if c["op"] == "plan":
        ctx, new = _plan_lengths(c, r)
        P = c["page"]
        used = [_pages(k, P) for k in ctx]
        need = sum(_pages(a + b, P) for a, b in zip(ctx, new)) - sum(used)
        n_free = max(0, need + c["spare"])
        ids = torch.randperm(sum(used) + n_free, generator=gen, device=DEV).to(torch.int32)
        flat = torch.full((c["n_seq"], c["cols"]), -1, dtype=torch.int32, device=DEV)
        u = i32(used)
        flat[torch.arange(c["cols"], device=DEV)[None, :] < u[:, None]] = ids[: sum(used)]
        cap = sum(new) + c["n_seq"] % 7
        s.update(ctx=i32(ctx), new=i32(new), free=ids[sum(used):].contiguous(), table=flat, cap=cap)
        bufs = [torch.empty(n, dtype=torch.int32, device=DEV) for n in (c["n_seq"] + 1, c["n_seq"], cap, cap, 4)]
        s["bufs"] = bufs
        if own:
            from handy_amd import serving
            s["plan"] = serving.PagePlan(*bufs)
        return s
    if c["op"] == "write":
        P, n = c["page"], c["n"]
        n_pages = _pages(n, P) + 3
        k, v = _cache(n_pages, c, gen)
        slots = torch.randperm(n_pages, generator=gen, device=DEV)[: _pages(n, P)]
        slots = (slots[:, None] * P + torch.arange(P, device=DEV)[None, :]).reshape(-1)[:n]
        slots = torch.cat([slots, torch.full((c["pad"],), -1, device=DEV)]).to(torch.int32)
        rows = n + c["pad"]
        # K and V of the new tokens as a fused projection leaves them: parts of one row
        qkv = torch.empty((rows, 3, c["heads"], c["dim"]), dtype=DTYPES[c["dtype"]], device=DEV).normal_(generator=gen)
        s.update(k_all=k, v_all=v, k_new=qkv[:, 1], v_new=qkv[:, 2], slots=slots, n_pages=n_pages)
        if own:
            from handy_amd import serving
            s["cache"] = serving.PagedCache(k[:n_pages], v[:n_pages])
        return s
    if c["op"] == "attn":
        ctx, new = _attn_lengths(c, r)
        P = c["page"]
        lens = [a + b for a, b in zip(ctx, new)]
        used = [_pages(k, P) for k in lens]
        n_pages = sum(used) + 2
        k, v = _cache(n_pages, c, gen)
        cols = max(used)
        table = torch.full((c["n_seq"], cols), -1, dtype=torch.int32, device=DEV)
        table[torch.arange(cols, device=DEV)[None, :] < i32(used)[:, None]] = torch.randperm(n_pages, generator=gen, device=DEV)[: sum(used)].to(torch.int32)
        n = sum(new)
        q = torch.empty((n, c["hq"], c["dim"]), dtype=DTYPES[c["dtype"]], device=DEV).normal_(generator=gen)
        q *= torch.linspace(0.5, 2.0, c["hq"], device=DEV).to(q.dtype)[None, :, None]         # heads of flat and of sharp attention
        cu = np.concatenate([[0], np.cumsum(new)]).tolist()
        s.update(q=q, k=k[:n_pages], v=v[:n_pages], table=table, cu=i32(cu), kv_lens=i32(lens), new=new, lens=lens, scale=1.0 / math.sqrt(c["dim"]),
                 out=torch.empty_like(q))
        if own:
            from handy_amd import serving
            s["cache"] = serving.PagedCache(s["k"], s["v"])
            need = serving.paged_attention_workspace(s["cache"], n, c["hq"], c["n_seq"], max(new), max(lens))
            s["ws"] = torch.empty(max(need, 16), dtype=torch.uint8, device=DEV)
        return s
    rows, V = c["rows"], c["vocab"]
    x = torch.empty((rows, V), dtype=torch.float32, device=DEV).normal_(generator=gen) * c["spread"]
    peak = torch.randint(0, V, (rows, 4), generator=gen, device=DEV)                          # a few likely tokens a row, as a model's logits have
    x.scatter_add_(1, peak, torch.rand((rows, 4), generator=gen, device=DEV) * 9.0)
    x[:, torch.randint(0, V, (V // 50,), generator=gen, device=DEV)] = NEG                    # suppressed tokens
    T = torch.rand(rows, generator=gen, device=DEV) * 0.9 + 0.2
    k = torch.randint(1, min(V, 200) + 1, (rows,), generator=gen, device=DEV).to(torch.int32)
    p = torch.rand(rows, generator=gen, device=DEV) * 0.6 + 0.4
    m = torch.rand(rows, generator=gen, device=DEV) * 0.1
    if c["mix"] == "all":
        which = torch.randint(0, 8, (rows,), generator=gen, device=DEV)
        k = torch.where(which % 2 == 1, k, torch.zeros_like(k))
        p = torch.where(which // 2 % 2 == 1, p, torch.ones_like(p))
        m = torch.where(which // 4 == 1, m, torch.zeros_like(m))
        T = torch.where(torch.rand(rows, generator=gen, device=DEV) < 0.1, torch.zeros_like(T), T)
    elif c["mix"] == "greedy":
        T = torch.zeros_like(T)
    use = {"temperature": "", "greedy": "", "top_k": "k", "top_p": "p", "min_p": "m", "all": "kpm"}[c["mix"]]
    s.update(logits=x.to(DTYPES[c["dtype"]]), uniform=torch.rand(rows, generator=gen, device=DEV), temperature=T, top_k=k if "k" in use else None,
             top_p=p if "p" in use else None, min_p=m if "m" in use else None, token=torch.empty(rows, dtype=torch.int32, device=DEV),
             logprob=torch.empty(rows, dtype=torch.float32, device=DEV))
    return s


# ------------------------------------------------------------------------------------------------ plain forms
def _plan_plain(s):
    c = s["case"]
    P, cols, cap, B = c["page"], c["cols"], s["cap"], c["n_seq"]
    ctx, new, free, table = s["ctx"].long(), s["new"].long(), s["free"], s["table"]
    n_free = free.numel()
    valid = (ctx >= 0) & (new >= 0) & (ctx + new <= cols * P)
    n = torch.where(valid, new, 0)
    first = (ctx + P - 1) // P
    need = torch.where(valid, (ctx + new + P - 1) // P - first, 0)
    fits = (torch.cumsum(n, 0) <= cap) & (torch.cumsum(need, 0) <= n_free)
    admitted = torch.cumprod(fits.long(), 0)
    n, need = n * admitted, need * admitted
    cu = torch.cat([torch.zeros_like(n[:1]), torch.cumsum(n, 0)])
    off = torch.cumsum(need, 0) - need
    rel = torch.arange(cols, device=DEV)[None, :] - first[:, None]
    if n_free:
        fresh = free[(off[:, None] + rel).clamp(0, n_free - 1)]
        table.copy_(torch.where((rel >= 0) & (rel < need[:, None]), fresh, table))
    tok = torch.arange(cap, device=DEV)
    seq = torch.searchsorted(cu[1:], tok, right=True).clamp(max=B - 1)
    pos = ctx[seq] + tok - cu[seq]
    live = tok < cu[-1]
    page = table[seq, (pos // P).clamp(0, cols - 1)].long()
    slots = torch.where(live & (page >= 0), page * P + pos % P, -1)
    counts = torch.stack([admitted.sum(), cu[-1], need.sum(), (~valid).sum()])
    i32 = lambda t: t.to(torch.int32)
    return table, i32(cu), i32(torch.where(valid, ctx + n, 0)), i32(slots), i32(torch.where(live, pos, 0)), i32(counts)


def _write_plain(s):
    P, n_pages = s["case"]["page"], s["n_pages"]
    slot = s["slots"].long()
    slot = torch.where((slot >= 0) & (slot < n_pages * P), slot, n_pages * P)
    s["k_all"][slot // P, slot % P] = s["k_new"]
    s["v_all"][slot // P, slot % P] = s["v_new"]
    return s["k_all"][:n_pages], s["v_all"][:n_pages]


def _softmax_pv(sc, mask, v):
    """sc [..., rows, keys], mask broadcast to it, v [..., keys, dim] -> rows without a key give 0"""
    sc = torch.where(mask, sc, NEG)
    m = sc.amax(-1, keepdim=True)
    p = torch.exp(sc - torch.where(m == NEG, 0.0, m))
    return torch.matmul(p, v) / p.sum(-1, keepdim=True).clamp(min=1e-30)


def _attn_plain(s):
    c = s["case"]
    P, W, hkv, D = c["page"], c["window"], c["hkv"], c["dim"]
    g = c["hq"] // hkv
    n_pages = s["k"].shape[0]
    q, out = s["q"], s["out"]
    if c["new_hi"] == 1:                                       # one token a request: batches of requests, padded to their longest
        order = list(range(c["n_seq"]))
        step = max(1, 400000 // max(s["lens"]))
        for a in range(0, len(order), step):
            ids = order[a:a + step]
            L = max(s["lens"][i] for i in ids)
            tb = s["table"][a:a + step, :_pages(L, P)].long()
            ok = ((tb >= 0) & (tb < n_pages)).repeat_interleave(P, 1)[:, :L]
            pos = s["kv_lens"][a:a + step].long()[:, None] - 1
            j = torch.arange(L, device=DEV)[None, :]
            ok = ok & (j <= pos)
            if W:
                ok = ok & (j > pos - W)
            tb = tb.clamp(0, n_pages - 1)
            k = s["k"][tb].reshape(len(ids), -1, hkv, D)[:, :L].float().permute(0, 2, 3, 1)
            v = s["v"][tb].reshape(len(ids), -1, hkv, D)[:, :L].float().permute(0, 2, 1, 3)
            qq = q[a:a + step].float().reshape(len(ids), hkv, g, D)
            o = _softmax_pv(torch.matmul(qq, k.contiguous()) * s["scale"], ok[:, None, None, :], v.contiguous())
            out[a:a + step] = o.reshape(len(ids), c["hq"], D).to(out.dtype)
        return out
    q0 = 0
    for i, (n, L) in enumerate(zip(s["new"], s["lens"])):
        tb = s["table"][i, :_pages(L, P)].long()
        ok = ((tb >= 0) & (tb < n_pages)).repeat_interleave(P)[:L]
        tb = tb.clamp(0, n_pages - 1)
        k = s["k"][tb].reshape(-1, hkv, D)[:L].float().permute(1, 2, 0).contiguous()
        v = s["v"][tb].reshape(-1, hkv, D)[:L].float().permute(1, 0, 2).contiguous()
        for a in range(0, n, 512):
            b = min(n, a + 512)
            hi = L - n + b
            qq = q[q0 + a:q0 + b].float().reshape(b - a, hkv, g, D).permute(1, 2, 0, 3).reshape(hkv, g * (b - a), D)
            pos = L - n + torch.arange(a, b, device=DEV)[:, None]
            j = torch.arange(hi, device=DEV)[None, :]
            mask = (j <= pos) & ok[None, :hi]
            if W:
                mask = mask & (j > pos - W)
            o = _softmax_pv(torch.matmul(qq, k[:, :, :hi]) * s["scale"], mask.repeat(g, 1)[None], v[:, :hi])
            out[q0 + a:q0 + b] = o.reshape(hkv, g, b - a, D).permute(2, 0, 1, 3).reshape(b - a, c["hq"], D).to(out.dtype)
        q0 += n
    return out


def _sample_plain(s):
    x = s["logits"].double()                                   # 64 bits: a draw near a border must not move
    x = torch.where(torch.isnan(x), NEG, x)
    rows, V = x.shape
    T = s["temperature"].double()[:, None]
    drawn = T > 0
    T = torch.where(drawn, T, 1.0)
    top = x.amax(1, keepdim=True)
    w = torch.where(x == top, 1.0, torch.exp((x - top) / T))
    w = torch.where(x == NEG, 0.0, w)
    z = w.sum(1, keepdim=True)
    xs, idx = torch.sort(x, dim=1, descending=True, stable=True)
    ws = w.gather(1, idx)
    rank = torch.arange(V, device=DEV)[None, :]
    keep = xs > NEG
    if s["top_k"] is not None:
        k = s["top_k"].long()[:, None]
        keep = keep & ((rank < k) | (k <= 0))
    if s["top_p"] is not None:
        p = s["top_p"].double()[:, None]
        head = torch.where(keep, ws, 0.0)
        before = torch.cumsum(head, 1) - head
        keep = keep & ((before < p * head.sum(1, keepdim=True)) | ~(p < 1.0))
    if s["min_p"] is not None:
        m = s["min_p"].double()[:, None]
        keep = keep & ((ws >= m) | ~(m > 0.0))
    keep = keep | ((rank == 0) & (xs > NEG))
    keep = keep & (drawn | (rank == 0))
    kept = torch.zeros_like(keep).scatter_(1, idx, keep)
    c = torch.cumsum(torch.where(kept, w, 0.0), 1)
    target = s["uniform"].double()[:, None].clamp(0.0, 1.0) * c[:, -1:]
    last = torch.where(kept & (w > 0), torch.arange(V, device=DEV)[None, :], -1).amax(1)
    token = torch.minimum((c <= target).sum(1), last)
    lp = (x.gather(1, token.clamp(min=0)[:, None]) - top) / T
    lp = torch.where(x.gather(1, token.clamp(min=0)[:, None]) == top, 0.0, lp) - torch.log(z)
    lp = torch.where(token[:, None] >= 0, lp, NEG)
    return token.to(torch.int32), lp[:, 0].float()


def run(state):
    s, c = state, state["case"]
    if not own:
        return {"plan": _plan_plain, "write": _write_plain, "attn": _attn_plain, "sample": _sample_plain}[c["op"]](s)
    from handy_amd import serving
    st = torch.cuda.current_stream().cuda_stream
    if c["op"] == "plan":
        plan = serving.plan_pages(s["ctx"], s["new"], s["free"], s["table"], c["page"], s["plan"], stream=st)
        return s["table"], plan.cu_q, plan.kv_lens, plan.slots, plan.positions, plan.counts
    if c["op"] == "write":
        serving.write_kv(s["cache"], s["k_new"], s["v_new"], s["slots"], stream=st)
        return s["k_all"][:s["n_pages"]], s["v_all"][:s["n_pages"]]
    if c["op"] == "attn":
        return serving.paged_attention(s["q"], s["cache"], s["table"], s["cu"], s["kv_lens"], max(s["new"]), max(s["lens"]), s["out"], scale=s["scale"],
                                       window=c["window"], workspace=s["ws"], stream=st)
    serving.sample_tokens(s["logits"], s["uniform"], s["token"], logprob=s["logprob"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"],
                          min_p=s["min_p"], stream=st)
    return s["token"], s["logprob"]


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def _visible(c, ctx, new):
    """sum over queries of visible keys, and over requests of keys any query sees"""
    W, pairs, keys = c["window"], 0, 0
    for a, n in zip(ctx, new):
        if W:
            pairs += sum(min(a + t + 1, W) for t in range(n))
            keys += min(a + n, W + n - 1)
        else:
            pairs += n * a + n * (n + 1) // 2
            keys += a + n
    return pairs, keys


def work(case):
    c = case
    r = random.Random(17)                                       # lengths of a typical seed
    if c["op"] == "plan":
        ctx, new = _plan_lengths(c, r)
        fresh = sum(_pages(a + b, c["page"]) - _pages(a, c["page"]) for a, b in zip(ctx, new))
        return {"bytes": 8 * c["n_seq"] + 8 * fresh + 8 * c["n_seq"] + 8 * (sum(new) + c["n_seq"] % 7) + 4 * c["n_seq"], "flops": 0}
    if c["op"] == "write":
        return {"bytes": 8 * c["n"] * c["heads"] * c["dim"] + 4 * (c["n"] + c["pad"]), "flops": 0}
    if c["op"] == "attn":
        ctx, new = _attn_lengths(c, r)
        pairs, keys = _visible(c, ctx, new)
        return {"bytes": 4 * keys * c["hkv"] * c["dim"] + 4 * sum(new) * c["hq"] * c["dim"] + 4 * keys // c["page"], "flops": 4 * pairs * c["hq"] * c["dim"]}
    size = 4 if c["dtype"] == "f32" else 2
    return {"bytes": c["rows"] * (c["vocab"] * size + 28), "flops": 0}


# ------------------------------------------------------------------------------------------------ definitions in 64 bits
def _exact_attn(case, s):
    c = case
    P, W, D = c["page"], c["window"], c["dim"]
    g = c["hq"] // c["hkv"]
    out = torch.zeros((s["q"].shape[0], c["hq"], D), dtype=torch.float64, device=DEV)
    q0 = 0
    for i, (n, L) in enumerate(zip(s["new"], s["lens"])):
        j = torch.arange(L, device=DEV)
        page = s["table"][i].long()[j // P]
        for h in range(c["hkv"]):
            k, v = s["k"][page, j % P, h].double(), s["v"][page, j % P, h].double()
            for hq in range(h * g, (h + 1) * g):
                for a in range(0, n, 2048):
                    b = min(n, a + 2048)
                    pos = L - n + torch.arange(a, b, device=DEV)
                    sc = torch.mm(s["q"][q0 + a:q0 + b, hq].double(), k.t().contiguous()) * s["scale"]
                    hide = j[None, :] > pos[:, None]
                    if W:
                        hide = hide | (j[None, :] <= pos[:, None] - W)
                    e = torch.softmax(sc.masked_fill_(hide, NEG), dim=1)
                    out[q0 + a:q0 + b, hq] = torch.mm(e, v)
        q0 += n
    return out


def _exact_sample(case, s):
    x = s["logits"].double().cpu().numpy()
    host = lambda t: None if t is None else t.double().cpu().numpy()
    T, k, p, m, u = (host(s[n]) for n in ("temperature", "top_k", "top_p", "min_p", "uniform"))
    tok, lp = np.empty(len(x), np.int32), np.empty(len(x))
    for r, row in enumerate(x):
        live = np.nonzero(row > -np.inf)[0]
        t = T[r] if T[r] > 0 else 1.0
        w = np.exp((row[live] - row[live].max()) / t)
        lp_all = (row[live] - row[live].max()) / t - math.log(w.sum())
        order = np.argsort(-row[live], kind="stable")
        n = len(order)
        if not T[r] > 0:
            n = 1
        else:
            if k is not None and k[r] > 0:
                n = min(n, int(k[r]))
            if p is not None and p[r] < 1:
                cum = np.concatenate([[0.0], np.cumsum(w[order[:n]])])
                n = max(1, int(np.searchsorted(cum[:-1], p[r] * cum[-1], side="left")))
            if m is not None and m[r] > 0:
                n = min(n, max(1, int((w >= m[r]).sum())))
        kept = np.sort(order[:n])
        cum = np.cumsum(w[kept])
        at = kept[min(int(np.searchsorted(cum, u[r] * cum[-1], side="right")), n - 1)]
        tok[r], lp[r] = live[at], lp_all[at]
    return torch.from_numpy(tok).to(DEV), torch.from_numpy(lp).to(DEV)


def _exact_plan(case, s):
    P, cols, cap = case["page"], case["cols"], s["cap"]
    ctx, new, free = s["ctx"].tolist(), s["new"].tolist(), s["free"].tolist()
    table = s["table"].cpu().numpy().copy()
    cu, kv, slots, positions, taken, admitted, stop = [0], [], [], [], 0, 0, False
    for i, (a, n) in enumerate(zip(ctx, new)):
        first, end = -(-a // P), -(-(a + n) // P)
        stop = stop or cu[-1] + n > cap or taken + end - first > len(free)
        if stop:
            cu.append(cu[-1])
            kv.append(a)
            continue
        table[i, first:end] = free[taken:taken + end - first]
        taken += end - first
        admitted += 1
        cu.append(cu[-1] + n)
        kv.append(a + n)
        at = np.arange(a, a + n)
        positions.append(at)
        slots.append(table[i, at // P].astype(np.int64) * P + at % P)
    n = cu[-1]
    tail = np.zeros(cap - n, np.int64)
    i32 = lambda v: torch.tensor(np.asarray(v), dtype=torch.int32, device=DEV)
    return i32(table), i32(cu), i32(kv), i32(np.concatenate(slots + [tail - 1])), i32(np.concatenate(positions + [tail])), i32([admitted, n, taken, 0])


def _exact_write(case, s):
    """every slot of the cache asks for the row that names it"""
    P, n_pages = case["page"], s["n_pages"]
    row = torch.full((n_pages * P + 1,), -1, device=DEV)
    row[s["slots"].long()] = torch.arange(s["slots"].numel(), device=DEV)       # padding (-1) lands on the entry past the last slot
    row = row[:-1].reshape(n_pages, P)
    pick = lambda new, old: torch.where((row >= 0)[:, :, None, None], new[row.clamp(min=0)], old[:n_pages]).double()
    return pick(s["k_new"], s["k_all"]), pick(s["v_new"], s["v_all"])


def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    return {"attn": _exact_attn, "sample": _exact_sample, "plan": _exact_plan, "write": _exact_write}[case["op"]](case, s)
