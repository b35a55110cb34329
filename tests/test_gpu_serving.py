"""GPU tests of the serving operators (handy_amd/serving.py over wmi_paged_plan, wmi_paged_write, wmi_paged_attention and
wmi_sample_tokens) against the 64-bit restatement in oracle/serving_oracle.py. Device memory comes from the library's own
runtime (no torch)."""
import ctypes as C
import os
import sys

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, ROOT)
from handy_amd import serving as sv           # noqa: E402
from handy_amd import whisper_rs as wr        # noqa: E402
from oracle import serving_oracle as so       # noqa: E402

pytestmark = pytest.mark.gpu

HALF_STEP = {"float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}        # a rounding to the type, relative


def dev(a, dtype=None):
    return sv.DeviceArray.from_numpy(a, dtype)


def host_form(x, dtype):
    return so.to_bf16(x) if dtype == "bfloat16" else x.astype(np.float16 if dtype == "float16" else np.float32)


def values(h, dtype):
    return (so.from_bf16(h) if dtype == "bfloat16" else h).astype(np.float64)


# ------------------------------------------------------------------------------------------------ plan
def run_plan(ctx, new, free, page, table, cap, stride=None, stream=0):
    n, cols = table.shape
    full = np.full((n, stride or cols), -7, np.int32)
    full[:, :cols] = table
    td = dev(full)
    view = td.view((n, cols), (full.shape[1], 1)) if stride else td
    out = sv.PagePlan(*(dev(np.full(k, -99, np.int32)) for k in (n + 1, n, cap, cap, 4)))
    sv.plan_pages(dev(np.asarray(ctx, np.int32)), dev(np.asarray(new, np.int32)), dev(np.asarray(free, np.int32)), view, page, out, stream=stream)
    if stream:
        assert wr.load_library().wmi_dev_stream_sync(stream) == 0
    got = td.numpy()
    assert (got[:, cols:] == -7).all()
    return (got[:, :cols],) + tuple(b.numpy() for b in out)


def plan_case(rng, n, page, cols, new_hi, spare, cap_short=0):
    room = page * cols
    new = rng.integers(0, new_hi + 1, n)
    ctx = np.array([rng.integers(0, max(room - k, 0) + 1) for k in new])
    used = -(-ctx // page)
    need = int((-(-(ctx + new) // page) - used).sum())
    ids = rng.permutation(int(used.sum()) + max(need + spare, 0)).astype(np.int32)
    table = np.full((n, cols), -1, np.int32)
    at = 0
    for i, u in enumerate(used):
        table[i, :u] = ids[at:at + u]
        at += u
    return ctx, new, ids[at:], page, table, max(int(new.sum()) - cap_short, 0)


@pytest.mark.parametrize("n,page,cols,new_hi,spare,short", [
    (1, 16, 28, 1, 3, 0), (1, 1, 7, 3, 0, 0), (64, 16, 28, 1, 8, 0), (65, 8, 12, 40, 0, 0), (300, 64, 16, 200, -5, 0), (300, 16, 40, 90, 4, 777),
    (1025, 32, 9, 33, 2, 0), (4096, 64, 20, 70, -900, 0), (16384, 16, 3, 5, 10, 3), (7, 1024, 2, 2000, 1, 0), (5, 16, 28, 0, 0, 0)])
def test_plan_matches_restatement(n, page, cols, new_hi, spare, short):
    rng = np.random.default_rng(n * 131 + page)
    case = plan_case(rng, n, page, cols, new_hi, spare, short)
    ref = so.plan(*case)
    got = run_plan(*case, stride=cols + 3)
    for name, g, r in zip(("table", "cu_q", "kv_lens", "slots", "positions", "counts"), got, ref):
        assert np.array_equal(g, r), name


def test_plan_odd_lengths_and_edges():
    """Negative lengths, lengths past the table row, sums beyond 32 bits, a table entry that names no page, room for no row, no
    request at all, a free list that ends with the last page, and a repeat of the call on its own result."""
    page, cols = 16, 4
    table = np.array([[3, -1, -1, -1], [5, 6, -1, -1], [-1, -1, -1, -1], [0, 1, 2, 7], [-1, -1, -1, -1], [9, -1, -1, -1]], np.int32)
    big = 2 ** 31 - 1
    ctx, new = [10, 20, -4, 64, big, 7], [9, 30, 3, 0, big, 60]
    for cap in (0, 5, 9, 38, 39, 99, 400):
        for n_free in (0, 1, 2, 3, 4, 10):
            free = np.arange(20, 20 + n_free, dtype=np.int32)
            ref = so.plan(ctx, new, free, page, table, cap)
            for g, r in zip(run_plan(ctx, new, free, page, table, cap), ref):
                assert np.array_equal(g, r), (cap, n_free)
    ctx, new = [30], [4]                                          # the cached tail lies on a page the table does not name
    table = np.array([[2, -1, -1, -1]], np.int32)
    ref = so.plan(ctx, new, [8], page, table, 6)
    got = run_plan(ctx, new, [8], page, table, 6)
    assert ref[3].tolist() == [-1, -1, 8 * 16, 8 * 16 + 1, -1, -1]
    for g, r in zip(got, ref):
        assert np.array_equal(g, r)
    again = run_plan(ctx, new, [8], page, got[0], 6)
    for g, r in zip(again, ref):
        assert np.array_equal(g, r)
    assert [x.tolist() for x in run_plan([], [], [], page, np.zeros((0, 4), np.int32), 3)[1:]] == [[0], [], [-1] * 3, [0] * 3, [0] * 4]
    table = np.array([[0, -1, -1, -1]], np.int32)                 # a page whose slots pass 31 bits
    for g, r in zip(run_plan([1], [40], [2 ** 27, 2 ** 31 - 1], page, table, 64), so.plan([1], [40], [2 ** 27, 2 ** 31 - 1], page, table, 64)):
        assert np.array_equal(g, r)


# ------------------------------------------------------------------------------------------------ cache and write
def make_cache(rng, n_pages, page, heads, dim, dtype, head_major=False, fill=None, pad=0):
    """-> PagedCache, host values [pages][page][heads][dim] of K and V, the two base arrays"""
    arrays, hosts, bases = [], [], []
    for _ in range(2):
        h = host_form(rng.standard_normal((n_pages, page, heads, dim)), dtype) if fill is None else host_form(np.full((n_pages, page, heads, dim), fill), dtype)
        hosts.append(h)
        inner = np.moveaxis(h, 2, 1) if head_major else h
        if pad:
            inner = np.concatenate([inner, np.zeros(inner.shape[:-1] + (pad,), inner.dtype)], axis=-1)
        base = dev(inner, dtype)
        bases.append(base)
        shape, st = base.shape, base.stride()
        view = base.view(shape[:3] + (dim,), st) if pad else base
        arrays.append(view.permute(0, 2, 1, 3) if head_major else view)
    return sv.PagedCache(*arrays), hosts, bases


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("n,page,heads,dim,head_major", [(1, 16, 20, 64, True), (64, 16, 20, 64, True), (333, 8, 2, 40, False), (257, 1, 3, 7, False), (1000, 64, 8, 128, False), (5, 32, 1, 1, True)])
def test_write_matches_restatement(dtype, n, page, heads, dim, head_major):
    rng = np.random.default_rng(n + dim)
    n_pages = -(-n // page) + 2
    cache, hosts, bases = make_cache(rng, n_pages, page, heads, dim, dtype, head_major)
    slots = rng.permutation(n_pages * page)[:n].astype(np.int32)
    slots[rng.random(n) < 0.2] = rng.choice([-1, -(2 ** 31), n_pages * page, 2 ** 31 - 1])
    qkv = host_form(rng.standard_normal((n, 3, heads, dim)), dtype)
    qd = dev(qkv, dtype)
    part = lambda i: qd.view((n, heads, dim), (3 * heads * dim, dim, 1), i * heads * dim)
    sv.write_kv(cache, part(1), part(2), dev(slots))
    for which, (host, base) in enumerate(zip(hosts, bases)):
        ref = host.copy()
        for r, s in enumerate(slots):
            if 0 <= s < n_pages * page:
                ref[s // page, s % page] = qkv[r, 1 + which]
        got = base.numpy()
        assert np.array_equal(np.moveaxis(got, 1, 2) if head_major else got, ref)


# ------------------------------------------------------------------------------------------------ attention
def attn_setup(seed, dtype, lens, news, hkv, group, dim, page, head_major=False, spread=1.0, cols=None, fill=None, pad=0):
    rng = np.random.default_rng(seed)
    used = [-(-max(L, 0) // page) for L in lens]
    n_pages = sum(used) + 2
    cache, hosts, bases = make_cache(rng, n_pages, page, hkv, dim, dtype, head_major, fill=fill, pad=pad)
    cols = cols or max(max(used), 1)
    table = np.full((len(lens), cols), -1, np.int32)
    ids = rng.permutation(n_pages)
    at = 0
    for i, u in enumerate(used):
        table[i, :u] = ids[at:at + u]
        at += u
    rows = int(sum(news))
    q = host_form(rng.standard_normal((rows, hkv * group, dim)) * spread, dtype)
    cu = np.concatenate([[0], np.cumsum(news)]).astype(np.int32)
    return cache, hosts, bases, table, q, cu, np.asarray(lens, np.int32)


def run_attn(cache, table, q, cu, lens, dtype, max_new, max_kv, window=0, scale=None, stream=0, extra_rows=0, ws_fill=0xFF):
    rows, hq, dim = q.shape
    qd = dev(q, dtype)
    out = dev(np.full((rows + extra_rows, hq, dim), 0x1234, np.uint16).view(np.float16) if dtype == "float16" else np.full((rows + extra_rows, hq, dim), 0x1234, np.uint16), dtype)
    if extra_rows:
        qd = dev(np.concatenate([q, np.zeros((extra_rows, hq, dim), q.dtype)]), dtype)
    need = sv.paged_attention_workspace(cache, rows + extra_rows, hq, len(lens), max_new, max_kv)
    ws = dev(np.full(need, ws_fill, np.uint8)) if need else None
    sv.paged_attention(qd, cache, dev(table), dev(cu), dev(lens), max_new, max_kv, out, scale=scale, window=window, workspace=ws, stream=stream)
    if stream:
        assert wr.load_library().wmi_dev_stream_sync(stream) == 0
    got = out.numpy()
    if extra_rows:
        assert (got[rows:].view(np.uint16) == 0x1234).all(), "rows behind the last request were written"
    return got[:rows]


def check_attn(got, dtype, q, hosts, table, cu, lens, page, scale, window=0, what=""):
    """Bound per element, from the arithmetic: the output's rounding to the type (half a step of its value); the probabilities'
    rounding to the type (half a step, on both the numerator and, at most, its sum: relative to sum p|v|); the scores' 32-bit
    products and sums, (dim + 8) 2^-24 of sum |q k|, twice (the key's own and the maximum's), through the exponential; the
    32-bit sums over the keys, n 2^-24; 2^-20 for the exponentials."""
    ref, mass, reach = so.attention(values(q, dtype), values(hosts[0], dtype), values(hosts[1], dtype), table, cu, lens, page, scale, window)
    half, n = HALF_STEP[dtype], max([int(x) for x in lens] + [1])
    rel = 2 * half + 2 * (q.shape[2] + 8) * 2.0 ** -24 * reach[:, :, None] + 2 * n * 2.0 ** -24 + 2.0 ** -20
    tiny = 2.0 ** -24 if dtype == "float16" else 2.0 ** -126        # below the normal numbers a rounding is absolute
    tol = half * np.abs(ref) + rel * mass * 1.01 + tiny
    g = values(got, dtype)
    assert np.isfinite(g).all(), what
    bad = np.abs(g - ref) > tol
    assert not bad.any(), (what, float((np.abs(g - ref) / tol).max()), np.argwhere(bad)[:4].tolist())


ATTN = [
    # lens, news, hkv, group, dim, page, window
    ([1], [1], 1, 1, 64, 16, 0),
    ([5, 1, 31, 200], [1, 1, 1, 1], 2, 4, 128, 16, 0),
    ([440, 17, 16, 1, 300], [1] * 5, 20, 1, 64, 16, 0),
    ([1000, 2047, 33], [1] * 3, 2, 8, 128, 64, 0),
    ([777, 64], [2, 3], 2, 5, 80, 8, 0),
    ([224, 100, 3, 64, 65], [224, 100, 3, 64, 65], 3, 1, 64, 16, 0),
    ([500, 130, 260], [200, 1, 129], 2, 4, 128, 64, 0),
    ([300, 40, 333], [77, 40, 1], 1, 7, 40, 32, 0),
    ([600, 90], [150, 90], 2, 2, 128, 16, 50),
    ([900, 31, 500], [1, 1, 1], 2, 3, 64, 32, 100),
    ([130, 0, 7], [130, 0, 0], 1, 3, 72, 1, 1),
    ([50, 3, 0, 64], [50, 9, 4, 70], 2, 2, 64, 16, 0),        # more new tokens than keys: their first rows see nothing
    ([257], [257], 1, 33, 128, 128, 0),                        # a group larger than a tile's rows
    ([4500], [1], 1, 1, 128, 1024, 0),
]


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("case", range(len(ATTN)))
def test_attention_matches_restatement(case, dtype):
    lens, news, hkv, group, dim, page, window = ATTN[case]
    cache, hosts, bases, table, q, cu, kv = attn_setup(case, dtype, lens, news, hkv, group, dim, page, head_major=case % 2 == 0, spread=1.5)
    got = run_attn(cache, table, q, cu, kv, dtype, max(news), max(lens), window=window, extra_rows=3)
    check_attn(got, dtype, q, hosts, table, cu, kv, page, dim ** -0.5, window, str(case))


@pytest.mark.parametrize("max_new,max_kv", [(0, 0), (1, 1), (500, 10 ** 6), (1, 2 ** 31 - 1)])
def test_attention_hints_do_not_matter(max_new, max_kv):
    lens, news = [700, 90, 1, 350], [1, 90, 1, 40]
    cache, hosts, _, table, q, cu, kv = attn_setup(5, "bfloat16", lens, news, 2, 4, 128, 16)
    got = run_attn(cache, table, q, cu, kv, "bfloat16", max_new, max_kv)
    check_attn(got, "bfloat16", q, hosts, table, cu, kv, 16, 128 ** -0.5)


@pytest.mark.parametrize("news", [[1, 1, 1], [40, 70, 9]])
def test_attention_ignores_what_no_row_sees(news):
    """Unused slots and unused pages hold NaN and infinity (stale memory does): nothing of them may reach a result, and neither may
    pages that the table names wrongly (negative, past the cache)."""
    dtype, page, lens = "float16", 16, [203, 150, 77]
    cache, hosts, bases, table, q, cu, kv = attn_setup(9, dtype, lens, news, 2, 2, 64, page)
    seen = np.zeros(hosts[0].shape[:2], bool)
    for i, L in enumerate(lens):
        for j in range(L):
            seen[table[i, j // page], j % page] = True
    for host, base, junk in zip(hosts, bases, (np.float16(np.inf), np.float16(np.nan))):
        host[~seen] = junk
        assert wr.load_library().wmi_dev_upload(base.data_ptr(), host.ctypes.data, host.nbytes) == 0
    wrong = table.copy()
    wrong[0, 3], wrong[1, 0], wrong[1, 5], wrong[2, 1] = -1, hosts[0].shape[0], 2 ** 31 - 1, -(2 ** 31)
    clean = [np.where(seen[:, :, None, None], h, np.float16(0)) for h in hosts]
    for tb in (table, wrong):
        got = run_attn(cache, tb, q, cu, kv, dtype, max(news), max(lens))
        check_attn(got, dtype, q, clean, tb, cu, kv, page, 64 ** -0.5)
        got = run_attn(cache, tb, q, cu, kv, dtype, max(news), max(lens), window=20)
        check_attn(got, dtype, q, clean, tb, cu, kv, page, 64 ** -0.5, 20)


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
def test_attention_wide_scores_and_strided_operands(dtype):
    """Scores of a few hundred (one key takes everything), a scale of its own, rows of a fused projection as q, a padded cache."""
    rng = np.random.default_rng(3)
    lens, news, hkv, group, dim, page = [90, 300, 64], [90, 2, 1], 2, 2, 64, 16
    cache, hosts, _, table, q, cu, kv = attn_setup(4, dtype, lens, news, hkv, group, dim, page, spread=30.0, pad=8)
    rows, hq = q.shape[:2]
    wide = np.zeros((rows, 2 * hq * dim + 16), q.dtype)
    wide[:, 8:8 + hq * dim] = q.reshape(rows, -1)
    qd = dev(wide, dtype).view((rows, hq, dim), (wide.shape[1], dim, 1), 8)
    od = dev(np.zeros_like(wide), dtype)
    out = od.view((rows, hq, dim), (wide.shape[1], dim, 1), 8)
    need = sv.paged_attention_workspace(cache, rows, hq, len(lens), max(news), max(lens))
    ws = dev(np.full(need, 0xFF, np.uint8)) if need else None
    sv.paged_attention(qd, cache, dev(table), dev(cu), dev(kv), max(news), max(lens), out, scale=0.4, workspace=ws)
    check_attn(out.numpy(), dtype, q, hosts, table, cu, kv, page, 0.4)
    full = od.numpy()
    assert not full[:, :8].any() and not full[:, 8 + hq * dim:].any()
    del rng


# ------------------------------------------------------------------------------------------------ sample
def run_sample(x, dtype, u, T=None, k=None, p=None, m=None, stride=None, stream=0, logprob=True):
    rows, V = x.shape
    full = x
    if stride:
        full = np.full((rows, stride), 60000 if dtype != "bfloat16" else so.to_bf16(np.float32(60000)), x.dtype)
        full[:, :V] = x
    ld = dev(full, dtype)
    if stride:
        ld = ld.view((rows, V), (stride, 1))
    tok, lp = dev(np.full(rows, -99, np.int32)), dev(np.full(rows, 99, np.float32)) if logprob else None
    f32 = lambda a: None if a is None else dev(np.asarray(a, np.float32))
    sv.sample_tokens(ld, f32(u), tok, logprob=lp, temperature=f32(T), top_k=None if k is None else dev(np.asarray(k, np.int32)), top_p=f32(p), min_p=f32(m), stream=stream)
    if stream:
        assert wr.load_library().wmi_dev_stream_sync(stream) == 0
    return tok.numpy(), lp.numpy() if logprob else None


def check_sample(x, dtype, u, T=None, k=None, p=None, m=None, what="", **kw):
    """Tokens equal the restatement's wherever the uniform number is not within 1e-9 of a border (the weights are held in 2^-45ths of
    the largest, up to 2^18 of them); logprob within its rounding to 32 bits, 2^-24 of its value, and 1e-9."""
    f = lambda a: None if a is None else np.asarray(a, np.float32)
    tok, lp = run_sample(x, dtype, u, T, k, p, m, **kw)
    ref, rlp, dist = so.sample(values(x, dtype) if dtype != "float32" else x, f(u), f(T), k, f(p), f(m))
    clear = dist > 1e-9
    assert (~clear).sum() <= max(1, len(clear) // 4), what
    assert np.array_equal(tok[clear], ref[clear]), (what, np.argwhere(tok != ref)[:5].tolist(), tok[tok != ref][:5], ref[tok != ref][:5])
    same = clear & np.isfinite(rlp)
    assert (np.abs(lp[same] - rlp[same]) <= 2.0 ** -24 * np.abs(rlp[same]) + 1e-9).all(), what
    assert np.array_equal(np.isneginf(lp[clear]), np.isneginf(rlp[clear])), what


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("rows,V,stride", [(1, 1, None), (3, 2, 5), (7, 100, None), (5, 51866, 51872), (33, 4097, None), (2, 131071, None), (1, 262144, None)])
def test_sample_matches_restatement(dtype, rows, V, stride):
    rng = np.random.default_rng(V + rows)
    for spread in (0.3, 3.0, 12.0):
        x = rng.standard_normal((rows, V)) * spread
        x[:, rng.integers(0, V, V // 40)] = -np.inf
        x = host_form(x, dtype)
        u = rng.random(rows).astype(np.float32)
        T = rng.uniform(0.1, 1.5, rows)
        k, p, m = rng.integers(1, max(2, min(V, 300)), rows), rng.uniform(0.05, 0.999, rows), rng.uniform(0.0, 0.3, rows)
        for kk in (None, k):
            for pp in (None, p):
                for mm in (None, m):
                    check_sample(x, dtype, u, T, kk, pp, mm, (spread, kk is not None, pp is not None, mm is not None), stride=stride)
        check_sample(x, dtype, u, np.zeros(rows), k, p, m, "greedy", stride=stride)
        check_sample(x, dtype, u, None, None, p, None, "no temperature")


def test_sample_parameters_at_their_ends():
    rng = np.random.default_rng(8)
    V = 700
    x = (rng.standard_normal((9, V)) * 3).astype(np.float32)
    for u in (0.0, 1.0 - 2.0 ** -24, 1.0, 0.5):
        uu = np.full(9, u, np.float32)
        check_sample(x, "float32", uu, what=("u", u))
        check_sample(x, "float32", uu, np.full(9, 0.7), [0, -5, 1, 2, V - 1, V, V + 1, 2 ** 31 - 1, -(2 ** 31)], what=("k", u))
        check_sample(x, "float32", uu, np.full(9, 0.7), None, [0.0, -1.0, 1.0, 2.0, np.inf, np.nan, 1e-30, 1 - 2.0 ** -24, 0.5], what=("p", u))
        check_sample(x, "float32", uu, np.full(9, 0.7), None, None, [0.0, -1.0, 1.0, 2.0, np.inf, np.nan, 1e-30, 1 - 2.0 ** -24, 0.5], what=("m", u))
        check_sample(x, "float32", uu, [0.0, -1.0, np.nan, 1e-30, 1e-45, 1e30, np.inf, 1.0, 0.01], what=("T", u))
    tok, _ = run_sample(x, "float32", np.full(9, np.nan), np.full(9, 0.7))      # a uniform number that is none counts as 0
    assert np.array_equal(tok, run_sample(x, "float32", np.zeros(9), np.full(9, 0.7))[0])
    tok, lp = run_sample(x, "float32", np.full(9, 0.3), logprob=False)
    assert lp is None and np.array_equal(tok, so.sample(x, np.full(9, 0.3, np.float32))[0])


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
def test_sample_ties_infinities_and_nothing_to_draw(dtype):
    rng = np.random.default_rng(2)
    V = 3001
    rows = [np.zeros(V), np.full(V, -np.inf), np.full(V, np.nan), rng.integers(-2, 3, V) * 1.0, np.where(np.arange(V) % 7 == 3, np.inf, 1.0),
            np.where(np.arange(V) == 2900, 5.0, -np.inf), np.where(rng.random(V) < 0.5, np.nan, rng.standard_normal(V)), np.where(np.arange(V) % 2 == 0, -0.0, 0.0),
            np.where(np.arange(V) == 17, 60000.0, rng.standard_normal(V)), np.where(rng.random(V) < 0.3, -60000.0, 1.0)]
    x = host_form(np.stack(rows), dtype)
    n = len(rows)
    for i in range(6):
        u = rng.random(n).astype(np.float32)
        check_sample(x, dtype, u, what=i)
        check_sample(x, dtype, u, np.full(n, 0.5), rng.integers(1, V, n), what=("k", i))
        check_sample(x, dtype, u, np.full(n, 0.5), rng.integers(1, V, n), rng.uniform(0.1, 0.9, n), what=("kp", i))
        check_sample(x, dtype, u, np.full(n, 0.5), rng.integers(1, 40, n), rng.uniform(0.1, 0.9, n), rng.uniform(0, 1, n), what=("kpm", i))
        check_sample(x, dtype, u, np.zeros(n), what=("greedy", i))


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("rows,V", [(6, 40000), (6, 5000), (257, 17000)])
def test_sample_cuts_inside_a_crowd(dtype, rows, V):
    """Nearly all entries within a few hundredths, one well above: the cut of top-k or top-p lies among thousands of entries that the
    bins from the largest value down do not tell apart. At positive and negative values, with min_p bounds that leave the crowd in (too
    many for a list), out, or in part."""
    rng = np.random.default_rng(V)
    for shift, gap in ((3.0, 6.0), (-3.0, 6.0), (-0.01, 1.0)):
        x = shift + 0.01 * rng.standard_normal((rows, V))
        x[np.arange(rows), rng.integers(0, V, rows)] = shift + gap
        x = host_form(x, dtype)
        u = rng.random(rows).astype(np.float32)
        k, p = rng.integers(V // 10, V, rows), rng.uniform(0.1, 0.95, rows)
        edge = np.exp(-gap) * rng.uniform(0.98, 1.02, rows)             # weights of the crowd
        for kk, pp, mm in ((k, None, None), (None, p, None), (k, p, None), (None, p, edge), (k, None, edge), (k, p, edge), (None, p, np.full(rows, 0.9 * np.exp(-gap))),
                           (None, p, np.full(rows, 0.9)), (None, p, np.full(rows, 1 / 2048)), (np.full(rows, 7), p, np.full(rows, 0.5))):
            check_sample(x, dtype, u, None, kk, pp, mm, (shift, gap, kk is not None, pp is not None, mm is not None))


def test_sample_does_not_depend_on_the_rows_beside():
    rng = np.random.default_rng(12)
    x = (rng.standard_normal((300, 5003)) * 2).astype(np.float32)
    u, T, k, p = rng.random(300), rng.uniform(0.3, 1.2, 300), rng.integers(0, 90, 300), rng.uniform(0.5, 1.1, 300)
    tok, lp = run_sample(x, "float32", u, T, k, p)
    for a, b in ((0, 1), (5, 9), (17, 300)):
        t2, l2 = run_sample(x[a:b], "float32", u[a:b], T[a:b], k[a:b], p[a:b])
        assert np.array_equal(t2, tok[a:b]) and np.array_equal(l2, lp[a:b])


# ------------------------------------------------------------------------------------------------ the four together, streams, graphs
def loop_arrays(rng, dtype, n_seq, page, hkv, group, dim, V, steps):
    cols = 12
    cache, hosts, bases = make_cache(rng, n_seq * cols, page, hkv, dim, dtype)
    return cache, hosts, bases, cols


def test_decode_loop_plan_write_attend_draw():
    """Five steps of a batch as a server runs them -- a prompt chunk, then one token each, one request a step behind -- with every
    operator's result checked and fed to the next, on a stream of the caller's."""
    L = wr.load_library()
    rng = np.random.default_rng(77)
    dtype, n_seq, page, hkv, group, dim, V = "float16", 6, 16, 2, 3, 64, 1000
    cache, hosts, bases, cols = loop_arrays(rng, dtype, n_seq, page, hkv, group, dim, V, 5)
    table = np.full((n_seq, cols), -1, np.int32)
    free = rng.permutation(n_seq * cols).astype(np.int32)
    stream = L.wmi_dev_stream_create()
    assert stream
    ctx = np.zeros(n_seq, np.int32)
    kept = [hosts[0].copy(), hosts[1].copy()]
    for step in range(5):
        new = rng.integers(3, 50, n_seq) if step == 0 else np.ones(n_seq, np.int64)
        if step == 1:
            new[2] = 0
        cap = int(new.sum()) + 2
        ref = so.plan(ctx, new, free, page, table, cap)
        td, out = dev(table), sv.PagePlan.allocate(n_seq, cap)
        sv.plan_pages(dev(ctx), dev(new.astype(np.int32)), dev(free), td, page, out, stream=stream)
        k_new, v_new = (host_form(rng.standard_normal((cap, hkv, dim)), dtype) for _ in range(2))
        kd, vd = dev(k_new, dtype), dev(v_new, dtype)
        sv.write_kv(cache, kd, vd, out.slots, stream=stream)
        q = host_form(rng.standard_normal((cap, hkv * group, dim)), dtype)
        qd, od = dev(q, dtype), dev(np.zeros_like(q), dtype)
        need = sv.paged_attention_workspace(cache, cap, hkv * group, n_seq, int(new.max()), int((ctx + new).max()))
        ws = dev(np.zeros(max(need, 1), np.uint8))
        sv.paged_attention(qd, cache, td, out.cu_q, out.kv_lens, int(new.max()), int((ctx + new).max()), od, workspace=ws, stream=stream)
        x, u = (rng.standard_normal((n_seq, V)) * 3).astype(np.float32), rng.random(n_seq).astype(np.float32)
        xd, ud, tok = dev(x), dev(u), dev(np.zeros(n_seq, np.int32))
        T = dev(np.full(n_seq, 0.8, np.float32))
        sv.sample_tokens(xd, ud, tok, temperature=T, stream=stream)
        assert L.wmi_dev_stream_sync(stream) == 0
        for g, r in zip((td,) + tuple(out), ref):
            assert np.array_equal(g.numpy(), r), step
        for r, s in enumerate(ref[3]):
            if s >= 0:
                kept[0][s // page, s % page], kept[1][s // page, s % page] = k_new[r], v_new[r]
        for b, h in zip(bases, kept):
            assert np.array_equal(b.numpy(), h)
        rows = int(ref[1][-1])
        check_attn(od.numpy()[:rows], dtype, q[:rows], kept, ref[0], ref[1], ref[2], page, dim ** -0.5, what=step)
        assert not od.numpy()[rows:].any()
        assert np.array_equal(tok.numpy(), so.sample(x, u, np.full(n_seq, 0.8, np.float32))[0])
        table, free, ctx = ref[0], free[ref[5][2]:], ref[2]
    L.wmi_dev_stream_destroy(stream)


def test_captured_step_replays_like_the_eager_one():
    """Plan, write, attention and draw captured once and replayed over changing inputs in the same buffers."""
    L = wr.load_library()
    for f in ("hipStreamBeginCapture", "hipStreamEndCapture", "hipGraphInstantiate", "hipGraphLaunch", "hipGraphExecDestroy", "hipGraphDestroy"):
        getattr(L, f).restype = C.c_int                            # the runtime the library is linked against, found through it
    rng = np.random.default_rng(5)
    dtype, n_seq, page, hkv, group, dim, V, cols = "bfloat16", 4, 16, 2, 4, 128, 3000, 40
    cache, hosts, bases = make_cache(rng, n_seq * cols, page, hkv, dim, dtype)
    cap = n_seq
    ctx, new, free, td = (dev(np.zeros(n, np.int32)) for n in (n_seq, n_seq, n_seq, (n_seq, cols)))
    out = sv.PagePlan.allocate(n_seq, cap)
    kd, vd = (dev(np.zeros((cap, hkv, dim), np.uint16), dtype) for _ in range(2))
    qd, od = (dev(np.zeros((cap, hkv * group, dim), np.uint16), dtype) for _ in range(2))
    xd, ud, tok, lp = dev(np.zeros((n_seq, V), np.float32)), dev(np.zeros(n_seq, np.float32)), dev(np.zeros(n_seq, np.int32)), dev(np.zeros(n_seq, np.float32))
    T, p = dev(np.full(n_seq, 0.9, np.float32)), dev(np.full(n_seq, 0.8, np.float32))
    need = sv.paged_attention_workspace(cache, cap, hkv * group, n_seq, 1, page * cols)
    ws = dev(np.zeros(max(need, 1), np.uint8))
    stream = L.wmi_dev_stream_create()

    def step():
        sv.plan_pages(ctx, new, free, td, page, out, stream=stream)
        sv.write_kv(cache, kd, vd, out.slots, stream=stream)
        sv.paged_attention(qd, cache, td, out.cu_q, out.kv_lens, 1, page * cols, od, workspace=ws, stream=stream)
        sv.sample_tokens(xd, ud, tok, logprob=lp, temperature=T, top_p=p, stream=stream)

    def put(d, a):
        a = np.ascontiguousarray(a)
        assert L.wmi_dev_upload(d.data_ptr(), a.ctypes.data, a.nbytes) == 0

    step()
    assert L.wmi_dev_stream_sync(stream) == 0
    graph, ex = C.c_void_p(), C.c_void_p()
    assert L.hipStreamBeginCapture(C.c_void_p(stream), 2) == 0      # relaxed mode
    step()
    assert L.hipStreamEndCapture(C.c_void_p(stream), C.byref(graph)) == 0 and graph.value
    assert L.hipGraphInstantiate(C.byref(ex), graph, None, None, C.c_size_t(0)) == 0
    pages = rng.permutation(n_seq * cols).astype(np.int32)
    for i, lens in enumerate(([3, 100, 31, 600], [1, 1, 1, 1], [600, 17, 16, 333], [50, 0, 200, 15])):
        c = np.maximum(np.asarray(lens) - 1, 0).astype(np.int32)
        n = (np.asarray(lens) > 0).astype(np.int32)
        table = np.full((n_seq, cols), -1, np.int32)
        for s in range(n_seq):
            u = -(-int(c[s]) // page)
            table[s, :u] = pages[s * cols:s * cols + u]
        fr = np.array([pages[s * cols + cols - 1] for s in range(n_seq)], np.int32)
        ref = so.plan(c, n, fr, page, table, cap)
        hk, hv, hq = (host_form(rng.standard_normal(s), dtype) for s in ((cap, hkv, dim), (cap, hkv, dim), (cap, hkv * group, dim)))
        x, u = (rng.standard_normal((n_seq, V)) * 2).astype(np.float32), rng.random(n_seq).astype(np.float32)
        for d, a in ((ctx, c), (new, n), (free, fr), (td, table), (kd, hk), (vd, hv), (qd, hq), (xd, x), (ud, u)):
            put(d, a)
        assert L.wmi_dev_sync() == 0
        assert L.hipGraphLaunch(ex, C.c_void_p(stream)) == 0
        assert L.wmi_dev_stream_sync(stream) == 0
        for r, s in enumerate(ref[3]):
            if s >= 0:
                hosts[0][s // page, s % page], hosts[1][s // page, s % page] = hk[r], hv[r]
        for g, r in zip((td,) + tuple(out), ref):
            assert np.array_equal(g.numpy(), r), i
        for b, h in zip(bases, hosts):
            assert np.array_equal(b.numpy(), h)
        rows = int(ref[1][-1])
        check_attn(od.numpy()[:rows], dtype, hq[:rows], hosts, ref[0], ref[1], ref[2], page, dim ** -0.5, what=i)
        got, glp = tok.numpy(), lp.numpy()
        eager, elp = run_sample(x, "float32", u, np.full(n_seq, 0.9), None, np.full(n_seq, 0.8))
        assert np.array_equal(got, eager) and np.array_equal(glp, elp)
    assert L.hipGraphExecDestroy(ex) == 0 and L.hipGraphDestroy(graph) == 0
    L.wmi_dev_stream_destroy(stream)


def test_host_memory_is_refused_and_nothing_runs():
    """A host pointer among the arguments is an error, not a fault: the entry asks the runtime whose memory each buffer is."""
    L = wr.load_library()
    host = np.zeros(4096, np.int32)
    x, u, tok = dev(np.zeros((2, 50), np.float32)), dev(np.zeros(2, np.float32)), dev(np.full(2, -9, np.int32))
    assert L.wmi_sample_tokens(host.ctypes.data, 2, 50, 2, 50, u.data_ptr(), None, None, None, None, tok.data_ptr(), None, None) == -1
    assert L.wmi_sample_tokens(x.data_ptr(), 2, 50, 2, 50, host.ctypes.data, None, None, None, None, tok.data_ptr(), None, None) == -1
    assert L.wmi_sample_tokens(x.data_ptr(), 2, 50, 2, 50, u.data_ptr(), host.ctypes.data, None, None, None, tok.data_ptr(), None, None) == -1
    assert (tok.numpy() == -9).all()
    cache, _, bases = make_cache(np.random.default_rng(0), 4, 16, 2, 64, "float16")
    kv = dev(np.ones((3, 2, 64), np.float16))
    before = bases[0].numpy()
    assert L.wmi_paged_write(cache.ref, kv.data_ptr(), 128, 64, kv.data_ptr(), 128, 64, host.ctypes.data, 3, None) == -1
    assert np.array_equal(bases[0].numpy(), before)
    assert L.wmi_sample_tokens(x.data_ptr(), 2, 50, 2, 50, u.data_ptr(), None, None, None, None, tok.data_ptr(), None, None) == 0      # and the next call runs
    assert L.wmi_dev_sync() == 0 and (tok.numpy() == 0).all()


@pytest.mark.parametrize("head_major", [False, True])
def test_offsets_past_32_bits_in_a_long_cache(head_major):
    """A cache of more than 2^32 elements (9.7 GB each of K and V): pages at its end are written and read, nothing at their offsets
    modulo 2^31 or 2^32."""
    dtype, page, hkv, dim, n_pages = "float16", 16, 8, 128, 296000
    per = page * hkv * dim
    assert n_pages * per > 2 ** 32 + 2 ** 28
    bases = [sv.DeviceArray((n_pages, page, hkv, dim), dtype) for _ in range(2)]
    strides = (per, dim, page * dim, 1) if head_major else (per, hkv * dim, dim, 1)
    cache = sv.PagedCache(*(b.view((n_pages, page, hkv, dim), strides) for b in bases))
    rng = np.random.default_rng(2)
    L, lens = wr.load_library(), [150, 31]
    pages = np.array([n_pages - 1 - 3 * i for i in range(12)], np.int32)
    table = np.full((2, 10), -1, np.int32)
    table[0], table[1, :2] = pages[:10], pages[10:]
    low = sorted({(int(p) * per) % m // per + d for p in pages for m in (2 ** 31, 2 ** 32) for d in (0, 1)})       # what a 32-bit offset would hit
    zeros = np.zeros(per, np.float16)
    for b in bases:
        for p in low + pages.tolist():
            assert L.wmi_dev_upload(b.data_ptr() + p * per * 2, zeros.ctypes.data, zeros.nbytes) == 0
    new = [rng.standard_normal((sum(lens), hkv, dim)).astype(np.float16) for _ in range(2)]
    slots = np.concatenate([[table[i, j // page] * page + j % page for j in range(n)] for i, n in enumerate(lens)]).astype(np.int32)
    sv.write_kv(cache, dev(new[0]), dev(new[1]), dev(slots))
    got = np.empty(per, np.float16)
    for which, b in enumerate(bases):
        for p in low:
            assert L.wmi_dev_download(got.ctypes.data, b.data_ptr() + p * per * 2, got.nbytes) == 0 and not got.any(), p
    hosts = [np.zeros((n_pages - int(pages.min()), page, hkv, dim), np.float16) for _ in range(2)]
    for h, x in zip(hosts, new):
        h[(slots // page) - int(pages.min()), slots % page] = x
    small = np.where(table >= 0, table - pages.min(), -1)
    for news in ([1, 1], [70, 31]):
        q = (rng.standard_normal((sum(news), hkv * 2, dim))).astype(np.float16)
        cu = np.concatenate([[0], np.cumsum(news)]).astype(np.int32)
        out = run_attn(cache, table, q, cu, np.array(lens, np.int32), dtype, max(news), max(lens))
        check_attn(out, dtype, q, hosts, small, cu, lens, page, dim ** -0.5, what=str(news))
    for b in bases:
        b.free()


def test_calls_on_two_streams_at_once():
    """Attention and draws enqueued on two streams without waiting, a workspace each: the results of the calls made one at a time."""
    L, dtype = wr.load_library(), "bfloat16"
    rng = np.random.default_rng(8)
    streams = [L.wmi_dev_stream_create() for _ in range(2)]
    jobs = []
    for seed, lens, news in ((31, [9000, 20], [1, 1]), (32, [5000, 700], [60, 200])):
        cache, hosts, bases, table, q, cu, kv = attn_setup(seed, dtype, lens, news, 2, 4, 128, 16)
        need = sv.paged_attention_workspace(cache, q.shape[0], q.shape[1], 2, max(news), max(lens))
        assert need > 0
        ref = run_attn(cache, table, q, cu, kv, dtype, max(news), max(lens))
        x, u = dev((rng.standard_normal((40, 20011)) * 2).astype(np.float32)), dev(rng.random(40).astype(np.float32))
        p, t0, t1 = dev(np.full(40, 0.9, np.float32)), dev(np.zeros(40, np.int32)), dev(np.zeros(40, np.int32))
        sv.sample_tokens(x, u, t0, top_p=p)
        jobs.append((cache, bases, dev(q, dtype), dev(table), dev(cu), dev(kv), max(news), max(lens), dev(np.zeros(q.shape, np.uint16), dtype), dev(np.full(need, 0xFF, np.uint8)), ref, x, u, p, t0, t1))
    assert L.wmi_dev_sync() == 0
    for _ in range(10):
        for s, (cache, _, q, table, cu, kv, mn, mk, out, ws, _, x, u, p, _, t1) in zip(streams, jobs):
            sv.paged_attention(q, cache, table, cu, kv, mn, mk, out, workspace=ws, stream=s)
            sv.sample_tokens(x, u, t1, top_p=p, stream=s)
    for s in streams:
        assert L.wmi_dev_stream_sync(s) == 0
    for j in jobs:
        assert np.array_equal(j[8].numpy(), j[10]) and np.array_equal(j[15].numpy(), j[14].numpy())
    for s in streams:
        L.wmi_dev_stream_destroy(s)


# ------------------------------------------------------------------------------------------------ attention: long tails
@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("n,dim,page", [(131071, 64, 64), (40000, 128, 16)])
@pytest.mark.parametrize("new,sink", [(1, "first"), (1, "last"), (40, "first")])
def test_attention_keeps_a_long_tail_behind_one_key(dtype, n, dim, page, new, sink):
    """One key whose score is far above all others' and whose V is 0: the result is the others', each a tiny weight. Bound: check_attn's, plus
    what a 16-bit probability below its normal numbers loses, half a step of 2^-24 against the 2^11 that the largest of a row is held at
    (float16; bfloat16 has no such numbers here), for every key: n 2^-36 of the largest |v|."""
    rng = np.random.default_rng(n + dim)
    n_pages = -(-n // page)
    at = 0 if sink == "first" else n - 1
    for gap in (15.0, 16.0, 17.0, 17.4, 19.0):
        k = 0.02 * rng.standard_normal((n_pages * page, 1, dim))
        v = rng.uniform(0.5, 1.5, (n_pages * page, 1, dim))
        k[at], v[at] = gap / dim ** 0.5, 0.0
        hosts = [host_form(x.reshape(n_pages, page, 1, dim), dtype) for x in (k, v)]
        cache = sv.PagedCache(*(dev(h, dtype) for h in hosts))
        table, cu, kv = np.arange(n_pages, dtype=np.int32)[None], np.array([0, new], np.int32), np.array([n], np.int32)
        q = host_form(np.ones((new, 2, dim)), dtype)
        ref, mass, reach = so.attention(values(q, dtype), values(hosts[0], dtype), values(hosts[1], dtype), table, cu, kv, page, dim ** -0.5)
        half = HALF_STEP[dtype]
        rel = 2 * half + 2 * (dim + 8) * 2.0 ** -24 * reach[:, :, None] + 2 * n * 2.0 ** -24 + 2.0 ** -20
        tol = half * np.abs(ref) + rel * mass * 1.01 + (2.0 ** -24 + n * 2.0 ** -36 * 1.5 if dtype == "float16" else 2.0 ** -126)
        for hint in (n, 1):                                        # keys split over workgroups, and all of them in one
            got = values(run_attn(cache, table, q, cu, kv, dtype, new, hint), dtype)
            assert (np.abs(got - ref) <= tol).all(), (gap, hint, float((np.abs(got - ref) / tol).max()), got.flat[0], ref.flat[0])


# ------------------------------------------------------------------------------------------------ plan: the largest row count
def test_plan_of_two_to_the_31_rows():
    """n_rows_cap = 2^31 - 1, the largest the entry takes (8.6 GB each of slots and positions): the rows at both ends are planned, and what lies in
    front of the two arrays and behind them is left alone."""
    L, cap, guard = wr.load_library(), 2 ** 31 - 1, 4096
    arrays = [sv.DeviceArray(cap + 2 * guard, "int32") for _ in range(2)]
    mark = np.full(guard, 0x5A5A5A5A, np.int32)
    for a in arrays:
        for at in (0, guard + cap):
            assert L.wmi_dev_upload(a.data_ptr() + 4 * at, mark.ctypes.data, mark.nbytes) == 0
    ctx, new, free, page, cols = [5, 30], [40, 1], np.arange(7, 17, dtype=np.int32), 16, 4
    table = np.array([[0, -1, -1, -1], [1, 2, -1, -1]], np.int32)
    out = sv.PagePlan(dev(np.zeros(3, np.int32)), dev(np.zeros(2, np.int32)), arrays[0].view((cap,), (1,), guard), arrays[1].view((cap,), (1,), guard), dev(np.zeros(4, np.int32)))
    td = dev(table)
    sv.plan_pages(dev(np.array(ctx, np.int32)), dev(np.array(new, np.int32)), dev(free), td, page, out)
    assert L.wmi_dev_sync() == 0
    ref = so.plan(ctx, new, free, page, table, 4096)
    for g, r in zip((td, out.cu_q, out.kv_lens, out.counts), (ref[0], ref[1], ref[2], ref[5])):
        assert np.array_equal(g.numpy(), r)
    got = np.empty(4096, np.int32)
    for a, first, rest in zip(arrays, ref[3:5], (-1, 0)):
        for at in (0, 2 ** 30, cap - 4096):
            assert L.wmi_dev_download(got.ctypes.data, a.data_ptr() + 4 * (guard + at), got.nbytes) == 0
            assert np.array_equal(got, first if at == 0 else np.full(4096, rest)), at
        for at in (0, guard + cap):
            assert L.wmi_dev_download(got.ctypes.data, a.data_ptr() + 4 * at, got.nbytes) == 0 and np.array_equal(got, mark), at
        a.free()


# ------------------------------------------------------------------------------------------------ attention: huge scores
@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("dim,page", [(64, 16), (128, 64), (40, 4)])
@pytest.mark.parametrize("new", [1, 70])
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_attention_of_scores_of_any_finite_size(dtype, dim, page, new, sign):
    """Scores up to 2^33 (float16) and 2^100 (bfloat16), positive and negative: every key is a multiple of one vector, the largest multiple
    takes everything, and keys with the same one -- in different tiles, waves and parts -- share it evenly. (The gap to the next multiple, a
    two-thousandth of the score, is far above the 2^-24 a score is off by.) Bound: the output's rounding and the probabilities', half a step each."""
    rng = np.random.default_rng(dim + new)
    n, top = 3000, 2000 if dtype == "float16" else 250
    n_pages = -(-n // page)
    step, hot = (16.0, 4096.0) if dtype == "float16" else (2.0 ** 40, 2.0 ** 46)
    mult = rng.integers(top // 2, top - 1, n_pages * page) if sign > 0 else rng.integers(3, top // 2, n_pages * page)
    best = rng.permutation(n - new)[:9]
    mult[best] = top if sign > 0 else 2
    k = np.broadcast_to((mult * step)[:, None, None], (n_pages * page, 1, dim))
    v = rng.uniform(0.5, 1.5, (n_pages * page, 1, dim))
    hosts = [host_form(x.reshape(n_pages, page, 1, dim), dtype) for x in (k, v)]
    assert np.array_equal(values(hosts[0], dtype).reshape(-1, dim)[:, 0], mult * step)
    q = host_form(np.broadcast_to(hot * (1 + rng.integers(0, 100, (new, 3, 1)) / 128), (new, 3, dim)), dtype)
    cache = sv.PagedCache(*(dev(h, dtype) for h in hosts))
    table, cu, kv = np.arange(n_pages, dtype=np.int32)[None], np.array([0, new], np.int32), np.array([n], np.int32)
    ref = values(hosts[1], dtype).reshape(-1, dim)[best].mean(0)
    for hint in (n, 1):                                            # keys split over workgroups, and all of them in one
        got = values(run_attn(cache, table, q, cu, kv, dtype, new, hint, scale=sign), dtype)
        assert np.isfinite(got).all(), hint
        assert (np.abs(got - ref) <= 3.01 * HALF_STEP[dtype] * np.abs(ref)).all(), (hint, float(np.abs(got / ref - 1).max()))


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("dim,page", [(64, 16), (128, 64), (40, 4)])
@pytest.mark.parametrize("new", [1, 60])
def test_attention_over_one_key_is_its_value(dtype, dim, page, new):
    """A row that sees one key gives that key's V to the bit (its weight is 1), and so does one whose other keys are far below it."""
    lens = [1, 60, 200]
    news = [min(new, L) for L in lens]
    cache, hosts, bases, table, q, cu, kv = attn_setup(2, dtype, lens, news, 2, 3, dim, page)
    got = run_attn(cache, table, q, cu, kv, dtype, max(news), max(lens), window=1)
    rows = [(i, L - n + t) for i, (L, n) in enumerate(zip(lens, news)) for t in range(n)]
    own = np.stack([hosts[1][table[i, p // page], p % page] for i, p in rows])
    assert np.array_equal(got, np.repeat(own, 3, axis=1))
    first = run_attn(cache, table, q, cu, kv, dtype, max(news), max(lens))
    at = [r for r, (_, p) in enumerate(rows) if p == 0]
    assert at and np.array_equal(first[at], np.repeat(own[at], 3, axis=1))
    k = values(hosts[0], dtype)                                    # every key but the first of its request 100 nats below it
    k[:] = -50.0 / dim ** 0.5
    for i in range(len(lens)):
        k[table[i, 0], 0] *= -1.0
    upload(bases[0], host_form(k, dtype), dtype)
    got = run_attn(cache, table, host_form(np.ones(q.shape), dtype), cu, kv, dtype, max(news), max(lens))
    assert np.array_equal(got, np.repeat(np.stack([hosts[1][table[i, 0], 0] for i, _ in rows]), 3, axis=1))


# ------------------------------------------------------------------------------------------------ attention: infinite keys
@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("dim,page", [(40, 16), (64, 16), (80, 64), (128, 32), (72, 2)])
@pytest.mark.parametrize("new", [1, 50])
def test_attention_of_keys_at_minus_infinity(dtype, dim, page, new):
    """Keys with an infinite element (in the first dims, in the last) that make the score minus infinity have weight 0, whatever the head's dim:
    the result is the other keys'."""
    rng = np.random.default_rng(dim + new)
    n = 700
    n_pages = -(-n // page)
    k, v = (rng.standard_normal((n_pages * page, 2, dim)) for _ in range(2))
    q = rng.standard_normal((new, 4, dim))
    q[:, :, 0], q[:, :, -1] = np.abs(q[:, :, 0]) + 0.1, np.abs(q[:, :, -1]) + 0.1
    gone = rng.random(n_pages * page) < 0.3
    gone[0] = False
    keep = [host_form(x.reshape(n_pages, page, 2, dim), dtype) for x in (k, v)]
    k[gone & (np.arange(len(gone)) % 2 == 0), :, 0] = -np.inf
    k[gone & (np.arange(len(gone)) % 2 == 1), :, -1] = -np.inf
    cache = sv.PagedCache(dev(host_form(k.reshape(n_pages, page, 2, dim), dtype), dtype), dev(keep[1], dtype))
    table, cu, kv = np.arange(n_pages, dtype=np.int32)[None], np.array([0, new], np.int32), np.array([n], np.int32)
    q = host_form(q, dtype)
    got = run_attn(cache, table, q, cu, kv, dtype, new, n)
    # the restatement over one page a key, the gone ones' page absent
    one = [h.reshape(n_pages * page, 1, 2, dim) for h in keep]
    check_attn(got, dtype, q, one, np.where(gone, -1, np.arange(n_pages * page))[None], cu, kv, 1, dim ** -0.5, what=(dim, new))


@pytest.mark.parametrize("news", [[4, 1, 9], [90, 7, 300]])
@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 5, 40, 2, 1])
def test_attention_windows_as_long_as_they_come_and_more_rows_than_keys(news, window):
    """A window of 2^31 - 1 as "no limit", with requests that bring more new tokens than they have keys: their first rows, at positions in front
    of the keys, give zeros, the others see what they see."""
    lens = [2, 0, 5] if max(news) < 10 else [60, 3, 250]
    cache, hosts, _, table, q, cu, kv = attn_setup(7, "bfloat16", lens, news, 2, 3, 64, 16)
    got = run_attn(cache, table, q, cu, kv, "bfloat16", max(news), max(lens), window=window, extra_rows=2)
    check_attn(got, "bfloat16", q, hosts, table, cu, kv, 16, 64 ** -0.5, window, (news, window))


def test_draws_into_the_parameters_own_arrays():
    """token in place of top_k, logprob in place of the uniform numbers or the temperatures: the results of separate arrays."""
    rng = np.random.default_rng(4)
    for rows, V in ((700, 300), (300, 20000), (9, 30000)):
        x, u = (rng.standard_normal((rows, V)) * 3).astype(np.float32), rng.random(rows).astype(np.float32)
        x[rows // 2] = -np.inf
        T, k = rng.uniform(0.3, 1.2, rows).astype(np.float32), rng.integers(1, 50, rows).astype(np.int32)
        tok, lp = run_sample(x, "float32", u, T, k)
        for place in ("u", "T"):
            ud, Td, kd = dev(u), dev(T), dev(k)
            sv.sample_tokens(dev(x), ud, kd, logprob=ud if place == "u" else Td, temperature=Td, top_k=kd)
            assert np.array_equal(kd.numpy(), tok) and np.array_equal((ud if place == "u" else Td).numpy(), lp)


@pytest.mark.parametrize("dim,page", [(64, 16), (128, 64), (40, 4)])
@pytest.mark.parametrize("new,hint", [(1, 0), (1, 1), (60, 0), (60, 1)])
def test_attention_of_the_largest_values(dim, page, new, hint):
    """float16 values of 65504 and -65504, the largest there are: a mean of them is one of them, not infinity, whatever the weights' roundings add up
    to. Bound: the weights' rounding, half a step each."""
    rng = np.random.default_rng(dim)
    lens = [3, 2, 700, 17, 1, 5]
    news = [min(new, L) for L in lens]
    cache, hosts, _, table, q, cu, kv = attn_setup(11, "float16", lens, news, 2, 2, dim, page)
    big = np.where(np.arange(dim) % 2 == 0, 65504.0, -65504.0)
    hosts[1] = np.broadcast_to(big, hosts[1].shape).astype(np.float16)
    cache = sv.PagedCache(cache.k, dev(hosts[1], "float16"))
    got = values(run_attn(cache, table, q, cu, kv, "float16", max(news), max(lens) if hint == 0 else hint), "float16")
    assert np.isfinite(got).all()
    assert (np.abs(got - big) <= 65504 * 2.0 ** -10).all()
    del rng


# ------------------------------------------------------------------------------------------------ errors of others
def test_an_earlier_calls_error_is_not_taken_for_this_ones():
    """An error that some other call left with the runtime: the operators run, succeed, and leave it to whoever asks for it."""
    L = wr.load_library()
    for f in ("hipSetDevice", "hipGetLastError", "hipPeekAtLastError"):
        getattr(L, f).restype = C.c_int                            # the runtime the library is linked against, found through it
    cache, hosts, _, table, q, cu, kv = attn_setup(3, "float16", [20, 5], [1, 1], 2, 1, 64, 16)
    x, u, tok = dev(np.eye(2, 50, 7, dtype=np.float32) * 50), dev(np.full(2, 0.5, np.float32)), dev(np.full(2, -9, np.int32))
    rows, slots = dev(np.ones((2, 2, 64), np.float16)), dev(np.full(2, -1, np.int32))
    out = sv.PagePlan.allocate(2, 4)
    plan_in = [dev(np.array(v, np.int32)) for v in ([3, 4], [1, 1], [9])]
    td, qd, od, cud, kvd = dev(table), dev(q, "float16"), dev(np.zeros_like(q), "float16"), dev(cu), dev(kv)
    calls = [lambda: sv.plan_pages(*plan_in, td, 16, out), lambda: sv.write_kv(cache, rows, rows, slots), lambda: sv.sample_tokens(x, u, tok),
             lambda: sv.paged_attention(qd, cache, td, cud, kvd, 1, 20, od)]
    for call in calls:
        assert L.hipSetDevice(4096) != 0                           # no such device: an error, and nothing else
        err = L.hipPeekAtLastError()
        assert err != 0
        call()
        assert L.hipPeekAtLastError() == err and L.hipGetLastError() == err and L.hipGetLastError() == 0
    assert L.wmi_dev_sync() == 0
    assert tok.numpy().tolist() == [7, 8]
    check_attn(od.numpy(), "float16", q, hosts, table, cu, kv, 16, 64 ** -0.5)


# ------------------------------------------------------------------------------------------------ attention: every kernel's holes and masks
def upload(base, host, dtype):
    a = np.ascontiguousarray(host)
    assert wr.load_library().wmi_dev_upload(base.data_ptr(), a.ctypes.data, a.nbytes) == 0


def junk_of(dtype):
    return (np.float16(np.inf), np.float16(np.nan)) if dtype == "float16" else (np.uint16(0x7F80), np.uint16(0x7FC0))


KERNELS = [([1, 1, 1], None), ([5, 1, 3], None), ([40, 70, 9], None), ([40, 70, 9], 0)]      # new tokens, max_kv hint: step, step or chunk, chunk of 4 waves, of 8 (dims above 64)


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("dim", [40, 64, 80, 128])
@pytest.mark.parametrize("page", [1, 8, 16, 64])
def test_attention_of_every_kernel_ignores_what_no_row_sees(dtype, dim, page):
    """Stale memory (NaN, infinity) in unused slots and pages, and table entries that name no page, at every head dim, page size and type, for
    the step kernel and both chunk kernels, with and without a window."""
    lens = [203, 150, 77]
    for news, hint in KERNELS:
        cache, hosts, bases, table, q, cu, kv = attn_setup(dim + page, dtype, lens, news, 2, 4, dim, page)
        seen = np.zeros(hosts[0].shape[:2], bool)
        for i, L in enumerate(lens):
            seen[table[i, np.arange(L) // page], np.arange(L) % page] = True
        clean = [np.where(seen[:, :, None, None], h, np.zeros((), h.dtype)) for h in hosts]
        wrong = table.copy()
        last = [(L - 1) // page for L in lens]
        wrong[0, last[0] // 3], wrong[1, 0], wrong[1, last[1] // 2], wrong[2, last[2]] = -1, hosts[0].shape[0], 2 ** 31 - 1, -(2 ** 31)
        for junk in (junk_of(dtype), junk_of(dtype)[::-1]):
            for h, base, j in zip(hosts, bases, junk):
                h[~seen] = j
                upload(base, h, dtype)
            for tb in (table, wrong):
                for window in (0, 20):
                    got = run_attn(cache, tb, q, cu, kv, dtype, max(news), max(lens) if hint is None else hint, window=window)
                    check_attn(got, dtype, q, clean, tb, cu, kv, page, dim ** -0.5, window, (news, hint, window))


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("dim,page", [(40, 8), (64, 16), (80, 1), (128, 64), (128, 2)])
def test_attention_of_every_kernel_keeps_a_bad_value_to_the_rows_that_see_it(dtype, dim, page):
    """NaN and infinity in the V of a key that some rows of a tile see and others, masked by position or window, do not: the others' results are
    those of a finite value there."""
    lens = [203, 150, 77]
    for news, hint in KERNELS[1:]:
        cache, hosts, bases, table, q, cu, kv = attn_setup(dim + page, dtype, lens, news, 2, 4, dim, page)
        at = [L - n // 2 - 1 for L, n in zip(lens, news)]          # seen by the later half of the request's new tokens, up to the window's length on
        for window in (0, 11):
            pos = np.concatenate([L - n + np.arange(n) for L, n in zip(lens, news)])
            bad = np.repeat(at, news)
            sees = (pos >= bad) & ((pos < bad + window) if window else True)
            for junk in junk_of(dtype):
                spoiled = hosts[1].copy()
                for i, j in enumerate(at):
                    spoiled[table[i, j // page], j % page] = junk
                upload(bases[1], spoiled, dtype)
                got = run_attn(cache, table, q, cu, kv, dtype, max(news), max(lens) if hint is None else hint, window=window)
                ref = got.copy()
                zero = hosts[1].copy()
                for i, j in enumerate(at):
                    zero[table[i, j // page], j % page] = 0
                upload(bases[1], zero, dtype)
                plain = run_attn(cache, table, q, cu, kv, dtype, max(news), max(lens) if hint is None else hint, window=window)
                check_attn(plain, dtype, q, [hosts[0], zero], table, cu, kv, page, dim ** -0.5, window, (news, hint, window))
                assert np.array_equal(ref[~sees], plain[~sees]), (news, hint, window)
                assert sees.any() and not np.isfinite(values(ref, dtype)[sees]).any(), (news, hint, window)


WIDE = [
    # lens, news, hkv, group, dim, page, window: 256 packed rows and more, for the eight-wave chunk kernel
    ([500, 130, 260], [200, 1, 129], 2, 4, 128, 64, 0),
    ([600, 90, 333], [150, 90, 7], 2, 2, 128, 16, 50),
    ([300, 5, 0, 140], [100, 5, 0, 140], 1, 3, 96, 8, 0),
    ([300, 64, 421], [60, 64, 200], 2, 5, 72, 32, 33),
    ([257], [257], 1, 33, 128, 128, 0),
    ([90, 200], [120, 300], 1, 7, 80, 4, 100),                 # more new tokens than keys
]


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("case", range(len(WIDE)))
@pytest.mark.parametrize("max_kv", [0, 9000])
def test_attention_on_eight_waves_matches_restatement(case, dtype, max_kv):
    lens, news, hkv, group, dim, page, window = WIDE[case]
    cache, hosts, bases, table, q, cu, kv = attn_setup(case, dtype, lens, news, hkv, group, dim, page, head_major=case % 2 == 0, spread=1.5)
    assert dim > 64 and max(news) * group >= 256
    got = run_attn(cache, table, q, cu, kv, dtype, max(news), max_kv, window=window, extra_rows=3)
    check_attn(got, dtype, q, hosts, table, cu, kv, page, dim ** -0.5, window, str(case))
