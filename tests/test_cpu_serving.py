"""Refusals of the serving operators that need no GPU: the C entries check sizes, types, alignment and pointers before they touch the
device, the Python layer checks shapes before it calls them. Plus the restatement's own sanity."""
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


class Fake:
    """Something that looks like a device array and owns no memory (the entries must refuse before they would use it)."""

    def __init__(self, shape, dtype, strides=None, ptr=0x10000):
        self.shape, self.dtype, self._p = tuple(shape), dtype, ptr
        self._s = tuple(strides) if strides is not None else sv._contiguous(self.shape)

    def data_ptr(self): return self._p
    def stride(self): return self._s
    def numel(self): return int(np.prod(self.shape))


P = 0x10000         # a non-null, aligned address that is no device memory


def cache_struct(**kw):
    c = dict(k=P, v=P, dtype=0, n_pages=8, page_tokens=16, n_kv_heads=2, head_dim=64, page_stride=2048, token_stride=128, head_stride=64)
    c.update(kw)
    return wr.wmi_paged_cache(*[c[n] for n, _ in wr.wmi_paged_cache._fields_])


def attn_struct(**kw):
    a = dict(q=P, out=P, block_table=P, cu_q=P, kv_lens=P, q_row_stride=256, q_head_stride=64, out_row_stride=256, out_head_stride=64, table_stride=8, table_cols=8,
             n_rows=3, n_seq=3, n_q_heads=4, window=0, max_new=1, max_kv=100, scale=0.125)
    a.update(kw)
    return wr.wmi_paged_attn(*[a[n] for n, _ in wr.wmi_paged_attn._fields_])


def test_attention_entry_refuses():
    L = wr.load_library()
    call = lambda c, a: L.wmi_paged_attention(C.byref(c), C.byref(a), None, 0, None)
    for bad in (dict(k=None), dict(v=None), dict(dtype=2), dict(dtype=-1), dict(n_pages=0), dict(n_kv_heads=0), dict(head_dim=0), dict(page_stride=-8), dict(k=P + 2), dict(v=P + 8),
                dict(token_stride=100), dict(head_stride=4)):
        assert call(cache_struct(**bad), attn_struct()) == -1, bad
    for bad in (dict(page_tokens=0), dict(page_tokens=12), dict(page_tokens=2048), dict(page_tokens=-16), dict(head_dim=60), dict(head_dim=136), dict(n_pages=2 ** 30)):
        assert call(cache_struct(**bad), attn_struct()) == -3, bad
    for bad in (dict(q=None), dict(out=None), dict(block_table=None), dict(cu_q=None), dict(kv_lens=None), dict(n_q_heads=3), dict(n_q_heads=0), dict(n_rows=-1), dict(n_seq=-1),
                dict(table_cols=-1), dict(table_stride=7), dict(window=-1), dict(max_new=-1), dict(max_kv=-2), dict(scale=float("nan")), dict(scale=float("inf")), dict(q=P + 4), dict(out=P + 2),
                dict(q_row_stride=-256), dict(out_head_stride=-64), dict(q_head_stride=63), dict(out_row_stride=255)):
        assert call(cache_struct(), attn_struct(**bad)) == -1, bad
    assert call(cache_struct(n_kv_heads=1), attn_struct(n_q_heads=129)) == -3
    assert L.wmi_paged_attention(None, C.byref(attn_struct()), None, 0, None) == -1
    assert L.wmi_paged_attention(C.byref(cache_struct()), None, None, 0, None) == -1
    assert call(cache_struct(), attn_struct(n_rows=0)) == 0 and call(cache_struct(), attn_struct(n_seq=0)) == 0      # nothing to do
    assert L.wmi_paged_attention_workspace(C.byref(cache_struct(head_dim=60)), C.byref(attn_struct())) == -3
    assert L.wmi_paged_attention_workspace(C.byref(cache_struct()), C.byref(attn_struct(q=None, out=None))) >= 0      # sizes only


def test_plan_write_sample_entries_refuse():
    L = wr.load_library()
    def plan(**kw):
        a = dict(ctx=P, new=P, n_seq=3, free=P, n_free=2, page=16, table=P, cols=4, stride=4, cu=P, kv=P, slots=P, pos=P, cap=5, counts=P)
        a.update(kw)
        return L.wmi_paged_plan(a["ctx"], a["new"], a["n_seq"], a["free"], a["n_free"], a["page"], a["table"], a["cols"], a["stride"], a["cu"], a["kv"], a["slots"], a["pos"], a["cap"],
                                a["counts"], None)
    for bad in (dict(ctx=None), dict(new=None), dict(free=None), dict(table=None), dict(cu=None), dict(kv=None), dict(slots=None), dict(pos=None), dict(counts=None), dict(n_seq=-1),
                dict(n_free=-1), dict(cols=-1), dict(cap=-1), dict(stride=3)):
        assert plan(**bad) == -1, bad
    for bad in (dict(page=0), dict(page=24), dict(page=4096), dict(n_seq=16385), dict(cols=2 ** 27, stride=2 ** 27)):
        assert plan(**bad) == -3, bad
    write = lambda c, n=3, k=P, v=P, s=P, row=128: L.wmi_paged_write(C.byref(c), k, row, 64, v, row, 64, s, n, None)
    assert write(cache_struct(), n=-1) == -1 and write(cache_struct(), k=None) == -1 and write(cache_struct(), v=None) == -1 and write(cache_struct(), s=None) == -1
    assert write(cache_struct(), row=-128) == -1 and write(cache_struct(dtype=2)) == -1 and write(cache_struct(page_tokens=3)) == -3 and write(cache_struct(), n=0) == 0
    def sample(**kw):
        a = dict(x=P, dt=2, stride=50, rows=2, V=50, u=P, tok=P)
        a.update(kw)
        return L.wmi_sample_tokens(a["x"], a["dt"], a["stride"], a["rows"], a["V"], a["u"], None, None, None, None, a["tok"], None, None)
    for bad in (dict(x=None), dict(u=None), dict(tok=None), dict(dt=3), dict(dt=-1), dict(rows=-1), dict(V=0), dict(stride=-1), dict(x=P + 2)):
        assert sample(**bad) == -1, bad
    assert sample(V=262145, stride=262145) == -3 and sample(rows=0) == 0


def test_python_layer_refuses_wrong_shapes_and_types():
    kv = lambda **kw: Fake(kw.get("shape", (8, 16, 2, 64)), kw.get("dtype", "float16"), kw.get("strides"))
    cache = sv.PagedCache(kv(), kv())
    for k, v in ((kv(dtype="float32"), kv(dtype="float32")), (kv(), kv(dtype="bfloat16")), (kv(), kv(shape=(8, 16, 2, 72))), (kv(shape=(8, 16, 128)), kv(shape=(8, 16, 128))),
                 (kv(), kv(strides=(2048, 64, 1024, 1))), (kv(strides=(2048, 128, 1, 2)), kv(strides=(2048, 128, 1, 2)))):
        with pytest.raises(ValueError):
            sv.PagedCache(k, v)
    i32 = lambda *s: Fake(s, "int32")
    good = dict(q=Fake((5, 4, 64), "float16"), block_table=i32(3, 8), cu_q=i32(4), kv_lens=i32(3), out=Fake((5, 4, 64), "float16"))
    for bad in (dict(q=Fake((5, 4, 72), "float16")), dict(q=Fake((5, 4, 64), "bfloat16")), dict(out=Fake((4, 4, 64), "float16")), dict(block_table=i32(2, 8)),
                dict(block_table=Fake((3, 8), "int64")), dict(cu_q=i32(3)), dict(kv_lens=Fake((3,), "float32")), dict(out=Fake((5, 4, 64), "float16", (256, 1, 4))),
                dict(q=Fake((5, 3, 64), "float16"), out=Fake((5, 3, 64), "float16"))):
        a = {**good, **bad}
        with pytest.raises(ValueError):
            sv.paged_attention(a["q"], cache, a["block_table"], a["cu_q"], a["kv_lens"], 1, 100, a["out"])
    with pytest.raises(ValueError):
        sv.paged_attention(good["q"], cache, good["block_table"], good["cu_q"], good["kv_lens"], 1, 100, good["out"], workspace=Fake((64,), "float32"))
    new = Fake((3, 2, 64), "float16")
    for a in ((Fake((3, 2, 72), "float16"), new, i32(3)), (new, Fake((2, 2, 64), "float16"), i32(3)), (new, new, i32(2)), (new, new, Fake((3,), "int64")), (Fake((3, 2, 64), "bfloat16"), new, i32(3))):
        with pytest.raises(ValueError):
            sv.write_kv(cache, *a)
    plan = sv.PagePlan(i32(4), i32(3), i32(9), i32(9), i32(4))
    for a in ((i32(3), i32(2), i32(5), i32(3, 4)), (i32(4), i32(3), i32(5), i32(3, 4)), (i32(3), i32(3), i32(5), i32(2, 4)), (i32(3), i32(3), Fake((5,), "int64"), i32(3, 4)),
              (i32(3), i32(3), i32(5), Fake((3, 4), "int32", (8, 2)))):
        with pytest.raises(ValueError):
            sv.plan_pages(*a, 16, plan)
    for bad in ((i32(3), i32(3), i32(9), i32(9), i32(4)), (i32(4), i32(3), i32(9), i32(8), i32(4)), (i32(4), i32(3), i32(9), i32(9), i32(3)), (Fake((4,), "int64"), i32(3), i32(9), i32(9), i32(4))):
        with pytest.raises(ValueError):
            sv.PagePlan(*bad)
    x, u, t = Fake((2, 50), "float32"), Fake((2,), "float32"), i32(2)
    for a, kw in (((Fake((2, 50), "float64"), u, t), {}), ((Fake((100,), "float32"), u, t), {}), ((x, Fake((1,), "float32"), t), {}), ((x, u, Fake((2,), "int64")), {}),
                  ((x, u, t), dict(top_k=Fake((2,), "float32"))), ((x, u, t), dict(temperature=i32(2))), ((x, u, t), dict(logprob=Fake((2,), "float16"))),
                  ((Fake((2, 50), "float32", (1, 2)), u, t), {})):
        with pytest.raises(ValueError):
            sv.sample_tokens(*a, **kw)


def test_restatement_on_cases_worked_by_hand():
    t, cu, kv, slots, pos, counts = so.plan([3, 4], [2, 5], [9, 8, 7], 4, np.array([[1, -1, -1], [0, -1, -1]], np.int32), 8)
    assert t.tolist() == [[1, 9, -1], [0, 8, 7]] and cu.tolist() == [0, 2, 7] and kv.tolist() == [5, 9]
    assert slots.tolist() == [7, 36, 32, 33, 34, 35, 28, -1] and pos.tolist() == [3, 4, 4, 5, 6, 7, 8, 0] and counts.tolist() == [2, 7, 3, 0]
    x = np.log(np.array([[0.1, 0.4, 0.2, 0.3]]))
    at = lambda u, **kw: int(so.sample(x, np.array([u], np.float32), **kw)[0][0])
    assert [at(u) for u in (0.0, 0.09, 0.11, 0.49, 0.51, 0.69, 0.71, 0.999)] == [0, 0, 1, 1, 2, 2, 3, 3]
    assert [at(u, top_k=[2]) for u in (0.0, 0.57, 0.58)] == [1, 1, 3]                 # 0.4 and 0.3 in the vocabulary's order: border 4/7
    assert [at(u, top_p=[0.75]) for u in (0.4, 0.5, 0.7)] == [1, 2, 3]                # 0.4 + 0.3 < 0.75: three are kept
    assert at(0.99, min_p=[0.6]) == 3 and at(0.99, min_p=[0.8]) == 1 and at(0.3, temperature=[0.0]) == 1
    k = np.zeros((1, 4, 1, 2)); v = np.arange(8.0).reshape(1, 4, 1, 2)
    out, _, _ = so.attention(np.zeros((2, 1, 2)), k, v, np.array([[0]]), [0, 2], [3], 4, 1.0)
    assert out[:, 0].tolist() == [[1.0, 2.0], [2.0, 3.0]]                             # means of the first two and three values


def test_plan_and_write_refuse_shared_memory():
    """Outputs that overlap an input or each other (workgroups read the lengths while others write), and one place for K and V."""
    L = wr.load_library()
    names = ["ctx", "new", "free", "table", "cu", "kv", "slots", "pos", "counts"]
    def plan(**kw):
        a = dict(zip(names, (0x10000 * (i + 1) for i in range(9))))
        a.update(kw)
        return L.wmi_paged_plan(a["ctx"], a["new"], 3, a["free"], 2, 16, a["table"], 4, 5, a["cu"], a["kv"], a["slots"], a["pos"], 6, a["counts"], None)
    base = dict(zip(names, (0x10000 * (i + 1) for i in range(9))))
    size = dict(ctx=3, new=3, free=2, table=14, cu=4, kv=3, slots=6, pos=6, counts=4)
    for out in names[3:]:
        for other in names:
            if other == out:
                continue
            for at in (base[other], base[other] + 4 * (size[other] - 1), base[other] - 4 * (size[out] - 1)):      # equal, and by one entry at either end
                assert plan(**{out: at}) == -1, (out, other)
    assert L.wmi_paged_write(C.byref(cache_struct(k=P, v=P)), 0x20000, 128, 64, 0x30000, 128, 64, 0x40000, 3, None) == -1
    assert L.wmi_paged_write(C.byref(cache_struct(k=P, v=P)), 0x20000, 128, 64, 0x20000, 256, 64, 0x40000, 3, None) == -1


def test_numbers_out_of_range_are_value_errors():
    cache = sv.PagedCache(Fake((8, 16, 2, 64), "float16"), Fake((8, 16, 2, 64), "float16"))
    i32 = lambda *s: Fake(s, "int32")
    q, out = Fake((5, 4, 64), "float16"), Fake((5, 4, 64), "float16")
    for kw in (dict(window=2 ** 31), dict(window=-2 ** 40), dict(scale=1e300), dict(window=1.5)):
        with pytest.raises(ValueError):
            sv.paged_attention(q, cache, i32(3, 8), i32(4), i32(3), 1, 100, out, **kw)
    with pytest.raises(ValueError):
        sv.paged_attention(q, cache, i32(3, 8), i32(4), i32(3), 1, 2 ** 33, out)


def test_tables_whose_rows_share_memory_are_refused():
    """A table expanded from one row (stride 0) or with overlapping rows owns fewer entries than rows times columns: no stride of the library's
    own choice may reach past them. A single row's stride does not matter."""
    cache = sv.PagedCache(Fake((8, 16, 2, 64), "float16"), Fake((8, 16, 2, 64), "float16"))
    i32 = lambda *s: Fake(s, "int32")
    plan = sv.PagePlan(i32(4), i32(3), i32(9), i32(9), i32(4))
    for stride in (0, 1, 7):
        table = Fake((3, 8), "int32", (stride, 1))
        with pytest.raises(ValueError, match="share memory"):
            sv._table(table, 3)
        with pytest.raises(ValueError, match="share memory"):
            sv.plan_pages(i32(3), i32(3), i32(5), table, 16, plan)
        with pytest.raises(ValueError, match="share memory"):
            sv.paged_attention(Fake((5, 4, 64), "float16"), cache, table, i32(4), i32(3), 1, 100, Fake((5, 4, 64), "float16", ptr=0x90000))
        assert sv._table(Fake((1, 8), "int32", (stride, 1)), 1) == (0x10000, 8, 8)
    assert sv._table(Fake((3, 8), "int32", (11, 1)), 3) == (0x10000, 11, 8)
    assert sv._table(Fake((3, 0), "int32", (0, 1)), 3)[1:] == (0, 0)


def test_attention_refuses_tables_of_more_keys_than_its_numbers_hold():
    """Key numbers are 32-bit and run a few tiles past the last one: table_cols * page_tokens is at most 2^31 - 256, in the workspace call too."""
    L = wr.load_library()
    for page, cols, rc in ((16, 2 ** 27 - 16, -1), (16, 2 ** 27 - 15, -3), (16, 2 ** 31 - 1, -3), (1, 2 ** 31 - 256, -1), (1, 2 ** 31 - 255, -3), (1024, 2 ** 21 - 1, -1), (1024, 2 ** 21, -3)):
        c, a = cache_struct(page_tokens=page), attn_struct(table_cols=cols, table_stride=cols)
        assert L.wmi_paged_attention(C.byref(c), C.byref(a), None, 0, None) in ((rc, -4) if rc == -1 else (rc,)), (page, cols)      # (-1: no device memory; -4: no GPU at all)
        assert (L.wmi_paged_attention_workspace(C.byref(c), C.byref(a)) >= 0) == (rc == -1)


def test_workspace_sizes_need_no_cache_memory():
    """The workspace call looks at sizes only: a caller may size its memory before it allocates the cache. The calls that use the cache refuse."""
    L = wr.load_library()
    a = attn_struct(q=None, out=None, block_table=None, cu_q=None, kv_lens=None, n_rows=1, n_seq=1, max_kv=100000, table_cols=8000, table_stride=8000)
    need = L.wmi_paged_attention_workspace(C.byref(cache_struct()), C.byref(a))
    assert need > 0
    for kw in (dict(k=None), dict(v=None), dict(k=None, v=None)):
        assert L.wmi_paged_attention_workspace(C.byref(cache_struct(**kw)), C.byref(a)) == need
        assert L.wmi_paged_attention(C.byref(cache_struct(**kw)), C.byref(attn_struct()), None, 0, None) == -1
        assert L.wmi_paged_write(C.byref(cache_struct(**kw)), P, 128, 64, P, 128, 64, P, 3, None) == -1


def test_views_stay_inside_their_array():
    """DeviceArray.view: neither end may lie outside the memory, for views of views too."""
    base = sv.DeviceArray((1,), "int32", _base=Fake((100,), "int32"))          # (stands for an allocation: the checks look at shapes only)
    base._base, base.shape, base._strides = None, (100,), (1,)
    for shape, strides, offset in (((4,), (1,), -1), ((4,), (1,), -100), ((4,), (1,), 97), ((1,), (1,), 100), ((2, 3), (50, 26), 0), ((2,), (-1,), 5)):
        with pytest.raises(ValueError):
            base.view(shape, strides, offset)
    inner = base.view((10,), (1,), 20)
    assert inner._offset == 20 and inner.view((5,), (1,), -20)._offset == 0    # a view's offset counts from the view, the memory is the array's
    with pytest.raises(ValueError):
        inner.view((5,), (1,), -21)
    with pytest.raises(ValueError):
        base.view((0, 4), (4, 1), -8)
    assert base.view((0, 4), (4, 1), 100).shape == (0, 4)


def test_attention_refuses_an_output_that_shares_memory():
    """out (and the workspace) may share no element with what the kernels read, nor out's rows with each other. Layouts that interleave without
    meeting are taken. Told from the codes without a GPU: -1 for the arguments, -4 for a call whose arguments are in order."""
    L = wr.load_library()
    A, far = 0x100000, dict(q=0x1000000, out=0x2000000, block_table=0x3000000, cu_q=0x3100000, kv_lens=0x3200000)
    cache = cache_struct(k=0x4000000, v=0x5000000)
    base = dict(far, n_rows=6, n_seq=3, n_q_heads=4, q_row_stride=256, q_head_stride=64, out_row_stride=256, out_head_stride=64, max_new=2)

    def call(ws=None, ws_bytes=0, **kw):
        return L.wmi_paged_attention(C.byref(cache), C.byref(attn_struct(**{**base, **kw})), ws, ws_bytes, None)
    if call() != -4:
        pytest.skip("a GPU is present: these addresses are refused as no memory of it")

    def refused(**kw):
        rc = call(**kw)
        assert rc in (-1, -4), rc
        return rc == -1
    for other, size in (("q", 6 * 256 * 2), ("block_table", 3 * 8 * 4), ("cu_q", 16), ("kv_lens", 12)):
        at, end = base[other], base[other] + size
        for out in (at, (end - 1) // 16 * 16, at - (5 * 256 + 3 * 64 + 64) * 2 + 16):
            assert refused(out=out), (other, hex(out))
        assert not refused(out=(end + 15) // 16 * 16) and not refused(out=at - 6 * 256 * 2), other
    for at in (cache.k, cache.v):
        assert refused(out=at) and refused(out=at + 8 * 2048 * 2 - 16) and not refused(out=at + 8 * 2048 * 2)
    both = dict(q_row_stride=1024, out_row_stride=1024)           # parts of one buffer's rows
    assert not refused(q=A, out=A + 512, **both) and not refused(q=A + 512, out=A, **both) and refused(q=A, out=A + 496, **both) and refused(q=A, out=A, **both)
    heads = dict(q_row_stride=512, out_row_stride=512, q_head_stride=128, out_head_stride=128)      # every other head of one buffer
    assert not refused(q=A, out=A + 128, **heads) and refused(q=A, out=A + 112, **heads) and refused(q=A, out=A + 256, **heads) and refused(q=A, out=A + 1024, **heads)
    for kw in (dict(out_row_stride=0), dict(out_head_stride=0), dict(out_head_stride=56), dict(out_row_stride=248), dict(out_row_stride=64)):
        assert refused(**kw), kw
    assert not refused(out_row_stride=64, out_head_stride=6 * 64)                                  # heads outermost
    assert not refused(n_rows=1, out_row_stride=0) and refused(n_rows=2, out_row_stride=0)
    assert not refused(q_row_stride=0) and not refused(q_head_stride=0)                            # queries may share memory: they are read
    long = dict(n_rows=3, n_seq=3, max_new=1, max_kv=100000, table_cols=8000, table_stride=8000)
    need = L.wmi_paged_attention_workspace(C.byref(cache), C.byref(attn_struct(**{**base, **long})))
    assert need > 0
    for name in ("q", "out", "block_table", "cu_q", "kv_lens"):
        assert refused(ws=base[name], ws_bytes=need, **long) and refused(ws=base[name] // 16 * 16 - (need - 1) // 16 * 16, ws_bytes=need, **long), name
    assert refused(ws=cache.k, ws_bytes=need, **long) and refused(ws=cache.v, ws_bytes=need, **long) and not refused(ws=0x6000000, ws_bytes=need, **long)


def test_sizes_that_do_not_fit_are_value_errors_too():
    """Whole numbers past 32 bits are errors in every call, not what their low bits say."""
    cache = sv.PagedCache(Fake((8, 16, 2, 64), "float16"), Fake((8, 16, 2, 64), "float16"))
    i32 = lambda *s: Fake(s, "int32")
    plan = sv.PagePlan(i32(4), i32(3), i32(9), i32(9), i32(4))
    for page in (2 ** 32 + 16, -2 ** 32 + 16, 16.5):
        with pytest.raises(ValueError):
            sv.plan_pages(i32(3), i32(3), i32(5), i32(3, 4), page, plan)
    for kw in (dict(n_rows=2 ** 32 + 1), dict(n_q_heads=2 ** 32 + 2), dict(n_seq=2 ** 32 + 1), dict(max_new=2 ** 32), dict(max_kv=2 ** 40)):
        with pytest.raises(ValueError):
            sv.paged_attention_workspace(cache, **{**dict(n_rows=1, n_q_heads=2, n_seq=1, max_new=1, max_kv=9), **kw})
    with pytest.raises(ValueError):
        sv.PagedCache(Fake((2 ** 32 + 8, 16, 2, 64), "float16"), Fake((2 ** 32 + 8, 16, 2, 64), "float16"))
    with pytest.raises(ValueError):
        sv.sample_tokens(Fake((2 ** 32 + 1, 50), "float32"), Fake((2 ** 32 + 1,), "float32"), i32(2 ** 32 + 1))
    with pytest.raises(ValueError):
        sv.write_kv(cache, Fake((2 ** 32 + 1, 2, 64), "float16"), Fake((2 ** 32 + 1, 2, 64), "float16"), i32(2 ** 32 + 1))


def test_split_calls_stay_within_a_grid():
    """The join of split keys has a workgroup of 256 threads for each row and query head, and a grid holds 2^32 threads: calls of 2^24 pairs and more
    (rows reserved far beyond the tokens that max_new and n_seq speak of) are not split and need no workspace."""
    L = wr.load_library()
    need = lambda rows: L.wmi_paged_attention_workspace(C.byref(cache_struct()), C.byref(attn_struct(n_rows=rows, n_seq=4, max_new=1, max_kv=10 ** 6)))
    assert need(2 ** 22 - 1) > 0 and need(2 ** 22) == 0 and need(2 ** 28 - 1) == 0


def test_draws_refuse_outputs_that_share_memory():
    """token and logprob may take the place of a parameter array entry by entry (a row reads its own before it writes), and share memory with
    nothing else. Told from the codes without a GPU: -1 for the arguments, -4 for a call whose arguments are in order."""
    L = wr.load_library()
    base = dict(x=0x1000000, u=0x2000000, T=0x2100000, k=0x2200000, p=0x2300000, m=0x2400000, tok=0x2500000, lp=0x2600000)

    def call(rows=5, V=50, stride=64, **kw):
        a = {**base, **kw}
        return L.wmi_sample_tokens(a["x"], 2, stride, rows, V, a["u"], a["T"], a["k"], a["p"], a["m"], a["tok"], a["lp"], None)
    if call() != -4:
        pytest.skip("a GPU is present: these addresses are refused as no memory of it")
    for out in ("tok", "lp"):
        for name in ("u", "T", "k", "p", "m"):
            assert call(**{out: base[name]}) == -4 and call(**{out: base[name] + 4}) == -1 and call(**{out: base[name] - 16}) == -1 and call(**{out: base[name] + 20}) == -4, (out, name)
        end = base["x"] + (4 * 64 + 50) * 4
        assert call(**{out: base["x"]}) == -1 and call(**{out: end - 4}) == -1 and call(**{out: end}) == -4 and call(**{out: base["x"] - 20}) == -4
        assert call(rows=1, stride=0, **{out: base["x"] + 50 * 4}) == -4 and call(rows=3, stride=0, **{out: base["x"] + 49 * 4}) == -1
    for d in (0, 4, -16):
        assert call(lp=base["tok"] + d) == -1
    assert call(lp=base["tok"] + 20) == -4 and call(lp=None, T=None, k=None, p=None, m=None) == -4


def test_draws_of_more_rows_than_a_grid_holds_are_refused():
    """A row is a workgroup of 256 threads (vocabularies up to 16384) to 1024, and a grid holds 2^32 threads."""
    L = wr.load_library()
    call = lambda rows, V: L.wmi_sample_tokens(P, 0, V, rows, V, 1 << 50, None, None, None, None, 1 << 51, None, None)
    for V, most in ((1, 2 ** 24), (16384, 2 ** 24), (16385, 2 ** 23), (131072, 2 ** 23), (131073, 2 ** 22)):
        assert call(most, V) == -3 and call(2 ** 31 - 1, V) == -3, V
        assert call(most - 1, V) in (-1, -4), V                    # (no GPU, or no memory of it)
