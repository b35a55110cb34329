// Serving operators around a paged K/V cache, for gfx950: block tables and slot maps from request lengths, the new tokens' K and
// V into their slots, and attention of a chunk of new tokens (or one token) over the cache.
#include "kernels.h"
#include "serving_host.h"

namespace wmi {

// ------------------------------------------------------------------------------------------ plan
// Request i has c cached and n new tokens. It needs ceil((c + n) / P) - ceil(c / P) fresh pages; the exclusive prefix sums of the
// new tokens and of the needs give its first row and its first entry in the free list. Requests are admitted in order up to the
// first (F) whose inclusive sums pass the row capacity or the free list.
// Every workgroup takes the whole prefix sum by itself (thousands of lengths, a few KB out of the L2: about 2 us) and keeps it in
// the LDS, so that rows and pages are then looked up by binary search there and the plan is one launch: bound by latency.
constexpr int kPlanMaxSeq = 16384;           // two 4-byte sums a request in 160 KB of LDS
constexpr int kPlanThreads = 1024;

struct PlanArgs {
    const int *ctx, *fresh, *free_pages;
    int *table, *cu, *kv, *slots, *positions, *counts;
    long table_stride;
    int n_seq, n_free, lp, cols, cap;
};

__global__ __launch_bounds__(kPlanThreads) void paged_plan_kernel(PlanArgs a) {
    extern __shared__ int plan_lds[];
    int *tok = plan_lds, *pag = plan_lds + a.n_seq + 1;      // exclusive prefix sums of admitted rows and pages
    __shared__ long long sh_n[16], sh_p[16];
    __shared__ int sh_first, sh_bad, sh_tok, sh_pag;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n_wave = blockDim.x >> 6;
    const int P = 1 << a.lp, B = a.n_seq, per = (B + (int)blockDim.x - 1) / (int)blockDim.x, i0 = min(B, tid * per), i1 = min(B, i0 + per);
    const long long room = (long long)a.cols << a.lp;
    auto lengths = [&](int i, long long &n, long long &need) {
        const long long c = a.ctx[i], m = a.fresh[i];
        const bool ok = c >= 0 && m >= 0 && c + m <= room;
        n = ok ? m : 0;
        need = ok ? ((c + m + P - 1) >> a.lp) - ((c + P - 1) >> a.lp) : 0;
        return ok;
    };
    if (tid == 0) { sh_first = B; sh_bad = 0; sh_tok = 0; sh_pag = 0; }
    long long sn = 0, sp = 0;                                // this thread's run of requests
    int bad = 0;
    for (int i = i0; i < i1; i++) { long long n, p; if (!lengths(i, n, p)) bad++; sn += n; sp += p; }
    long long xn = sn, xp = sp;                              // inclusive over the wave
    for (int o = 1; o < 64; o <<= 1) { const long long yn = __shfl_up(xn, o), yp = __shfl_up(xp, o); if (lane >= o) { xn += yn; xp += yp; } }
    if (lane == 63) { sh_n[wave] = xn; sh_p[wave] = xp; }
    __syncthreads();
    long long bn = xn - sn, bp = xp - sp;                    // exclusive over the workgroup
    for (int w = 0; w < n_wave; w++) if (w < wave) { bn += sh_n[w]; bp += sh_p[w]; }
    if (bad) atomicAdd(&sh_bad, bad);
    long long rn = bn, rp = bp;
    for (int i = i0; i < i1; i++) {
        long long n, p;
        lengths(i, n, p);
        if (rn + n > a.cap || rp + p > a.n_free) { atomicMin(&sh_first, i); break; }
        tok[i] = (int)rn; pag[i] = (int)rp;
        rn += n; rp += p;
    }
    __syncthreads();
    const int F = sh_first;
    if (i0 < i1 && F >= i0 && F < i1) {                      // the thread that met F: its sums are what is admitted in all
        long long tn = bn, tp = bp;
        for (int i = i0; i < F; i++) { long long n, p; lengths(i, n, p); tn += n; tp += p; }
        sh_tok = (int)tn; sh_pag = (int)tp;
    } else if (F == B && i1 == B && i0 < i1) {               // everything is admitted: the last run's end
        sh_tok = (int)rn; sh_pag = (int)rp;
    }
    __syncthreads();
    const int n_tok = sh_tok, n_pag = sh_pag;
    for (int i = F + tid; i <= B; i += blockDim.x) { tok[i] = n_tok; pag[i] = n_pag; }
    __syncthreads();

    const int gtid = blockIdx.x * blockDim.x + tid, gsize = gridDim.x * blockDim.x;
    // the last request whose sum is <= x among those that own anything: upper bound minus one
    auto owner = [&](const int *s, int x) { int lo = 0, hi = B; while (lo < hi) { const int m = (lo + hi) >> 1; if (s[m + 1] <= x) lo = m + 1; else hi = m; } return lo; };
    for (int x = gtid; x < n_pag; x += gsize) {
        const int i = owner(pag, x);
        a.table[i * a.table_stride + ((a.ctx[i] + P - 1) >> a.lp) + (x - pag[i])] = a.free_pages[x];
    }
    for (int x = gtid; x < a.cap; x += gsize) {
        int slot = -1, pos = 0;
        if (x < n_tok) {
            const int i = owner(tok, x), c = a.ctx[i], first = (c + P - 1) >> a.lp;
            pos = c + (x - tok[i]);
            const int col = pos >> a.lp;
            const long page = col >= first ? a.free_pages[pag[i] + col - first] : a.table[i * a.table_stride + col];   // fresh entries may still be on their way
            const long long sl = ((long long)page << a.lp) + (pos & (P - 1));
            if (page >= 0 && sl <= 0x7fffffff) slot = (int)sl;
        }
        a.slots[x] = slot;
        a.positions[x] = pos;
    }
    for (int i = gtid; i <= B; i += gsize) {
        a.cu[i] = tok[i];
        if (i < B) { long long n, p; const bool ok = lengths(i, n, p); a.kv[i] = ok ? a.ctx[i] + (i < F ? (int)n : 0) : 0; }
    }
    if (gtid == 0) { a.counts[0] = F; a.counts[1] = n_tok; a.counts[2] = n_pag; a.counts[3] = sh_bad; }
}

// ------------------------------------------------------------------------------------------ write
// cache[slot[r]] = new[r] for K and V; a row whose slot lies outside the cache is skipped. A thread moves VEC elements of K and
// of V: bound by HBM.
struct WriteArgs {
    const char *kn, *vn;
    char *kc, *vc;
    const int *slots;
    long kn_row, kn_head, vn_row, vn_head, page, token, head;   // strides in bytes
    long n_slots, total;
    int lp, heads, chunks;                                       // chunks of VEC elements in a head
};
template <class T>
__global__ __launch_bounds__(256) void paged_write_kernel(WriteArgs a) {
    for (long i = blockIdx.x * 256L + threadIdx.x; i < a.total; i += gridDim.x * 256L) {
        const int per_row = a.heads * a.chunks;
        const long r = i / per_row;
        const int j = (int)(i - r * per_row), h = j / a.chunks, c = j - h * a.chunks;
        const int slot = a.slots[r];
        if (slot < 0 || slot >= a.n_slots) continue;
        const long dst = (long)(slot >> a.lp) * a.page + (long)(slot & ((1 << a.lp) - 1)) * a.token + h * a.head + c * (long)sizeof(T);
        *(T *)(a.kc + dst) = *(const T *)(a.kn + r * a.kn_row + h * a.kn_head + c * (long)sizeof(T));
        *(T *)(a.vc + dst) = *(const T *)(a.vn + r * a.vn_row + h * a.vn_head + c * (long)sizeof(T));
    }
}

// ------------------------------------------------------------------------------------------ attention
// One workgroup per (row, query head): 8 or 16 lanes share a key (8 dims each), every lane group keeps its own running maximum,
// sum and accumulator over the keys it visits, and the groups are merged at the end.
template <class T> struct Vec8;
template <> struct Vec8<f16> { typedef f16x8 type; };
typedef __bf16 bf16;
typedef bf16 bf16x8 __attribute__((ext_vector_type(8)));
template <> struct Vec8<bf16> { typedef bf16x8 type; };

template <class T, int LPK>       // LPK lanes a key
__global__ __launch_bounds__(256) void paged_attention_kernel(PagedAttn a) {
    typedef typename Vec8<T>::type V8;
    constexpr int KPW = 64 / LPK;
    __shared__ float red[4][LPK][10];
    const int row = blockIdx.x, hq = blockIdx.y, tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, grp = lane / LPK, e = (lane % LPK) * 8;
    int lo = 0, hi = a.n_seq;                                 // the request of this row
    while (lo < hi) { const int m = (lo + hi) >> 1; if (a.cu[m + 1] <= row) lo = m + 1; else hi = m; }
    if (lo >= a.n_seq || row < a.cu[lo]) return;              // rows behind the last request stay as they are
    const int i = lo, n = a.cu[i + 1] - a.cu[i];
    const int L = min(max(a.kv_lens[i], 0), (int)min((long)a.cols << a.lp, 0x7fffffffL));
    const int pos = L - n + (row - a.cu[i]);
    const int k0 = a.window > 0 ? max(0, pos - a.window + 1) : 0;
    const int h = hq / a.group;
    const bool on = e < a.dim;
    const T *kc = (const T *)a.k + h * a.head_stride + e, *vc = (const T *)a.v + h * a.head_stride + e;
    float q[8], acc[8], m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int t = 0; t < 8; t++) { q[t] = 0.0f; acc[t] = 0.0f; }
    if (on) { const V8 x = *(const V8 *)((const T *)a.q + row * a.q_row + hq * a.q_head + e);
#pragma unroll
        for (int t = 0; t < 8; t++) q[t] = (float)x[t] * a.scale; }
    for (int j = k0 + wave * KPW + grp; j <= pos; j += 4 * KPW) {
        const int page = a.table[i * a.table_stride + (j >> a.lp)];
        if (page < 0 || page >= a.n_pages) continue;
        const long off = page * a.page_stride + (long)(j & ((1 << a.lp) - 1)) * a.token_stride;
        float d = 0.0f;
        V8 vx = {};
        if (on) {
            const V8 kx = *(const V8 *)(kc + off);
            vx = *(const V8 *)(vc + off);
#pragma unroll
            for (int t = 0; t < 8; t++) d = __builtin_fmaf(q[t], (float)kx[t], d);
        }
#pragma unroll
        for (int o = 1; o < LPK; o <<= 1) d += __shfl_xor(d, o);
        const float mn = fmaxf(m, d), al = m == -INFINITY ? 0.0f : __expf(m - mn), p = __expf(d - mn);
        l = l * al + p;
#pragma unroll
        for (int t = 0; t < 8; t++) acc[t] = acc[t] * al + p * (float)vx[t];
        m = mn;
    }
    for (int o = LPK; o < 64; o <<= 1) {
        const float om = __shfl_xor(m, o), ol = __shfl_xor(l, o), mn = fmaxf(m, om);
        const float fa = m == -INFINITY ? 0.0f : __expf(m - mn), fb = om == -INFINITY ? 0.0f : __expf(om - mn);
        l = l * fa + ol * fb;
#pragma unroll
        for (int t = 0; t < 8; t++) { const float oa = __shfl_xor(acc[t], o); acc[t] = acc[t] * fa + oa * fb; }
        m = mn;
    }
    if (grp == 0) { red[wave][lane][0] = m; red[wave][lane][1] = l;
#pragma unroll
        for (int t = 0; t < 8; t++) red[wave][lane][2 + t] = acc[t]; }
    __syncthreads();
    if (tid < LPK && on) {
        float mn = -INFINITY, ls = 0.0f, o[8] = {};
        for (int w = 0; w < 4; w++) mn = fmaxf(mn, red[w][tid][0]);
        for (int w = 0; w < 4; w++) {
            const float f = red[w][tid][0] == -INFINITY ? 0.0f : __expf(red[w][tid][0] - mn);
            ls += red[w][tid][1] * f;
#pragma unroll
            for (int t = 0; t < 8; t++) o[t] += red[w][tid][2 + t] * f;
        }
        const float inv = ls > 0.0f ? 1.0f / ls : 0.0f;      // a row that sees nothing gives zeros
        V8 y;
#pragma unroll
        for (int t = 0; t < 8; t++) y[t] = (T)(o[t] * inv);
        *(V8 *)((T *)a.out + row * a.o_row + hq * a.o_head + e) = y;
    }
}

size_t paged_attention_workspace(const PagedAttn &) { return 0; }

bool paged_attention(const PagedAttn &a, void *, hipStream_t st) {
    const dim3 grid(a.n_rows, a.hkv * a.group);
    if (a.dtype == WMI_F16) {
        if (a.dim <= 64) hipLaunchKernelGGL((paged_attention_kernel<f16, 8>), grid, dim3(256), 0, st, a);
        else hipLaunchKernelGGL((paged_attention_kernel<f16, 16>), grid, dim3(256), 0, st, a);
    } else {
        if (a.dim <= 64) hipLaunchKernelGGL((paged_attention_kernel<bf16, 8>), grid, dim3(256), 0, st, a);
        else hipLaunchKernelGGL((paged_attention_kernel<bf16, 16>), grid, dim3(256), 0, st, a);
    }
    return hipGetLastError() == hipSuccess;
}

namespace {

int log2_of(int x) { int l = 0; while ((1 << l) < x) l++; return l; }
bool power_of_two(int x) { return x > 0 && !(x & (x - 1)); }

// what every entry asks of a cache description; 0, -1 or -3
int check_cache(const wmi_paged_cache *c) {
    if (!c || !c->k || !c->v || c->n_pages < 1 || c->n_kv_heads < 1 || c->head_dim < 1) return -1;
    if (c->dtype != WMI_F16 && c->dtype != WMI_BF16) return -1;
    if (c->page_stride < 0 || c->token_stride < 0 || c->head_stride < 0) return -1;
    if (!power_of_two(c->page_tokens) || c->page_tokens > 1024 || (long long)c->n_pages * c->page_tokens > 0x7fffffffLL) return -3;
    return 0;
}
bool aligned16(const void *p) { return ((uintptr_t)p & 15) == 0; }

// the description in the kernels' terms, checked; 0, -1 or -3
int fill_attn(const wmi_paged_cache *c, const wmi_paged_attn *p, PagedAttn &a) {
    const int rc = check_cache(c);
    if (rc) return rc;
    if (!p || p->n_rows < 0 || p->n_seq < 0 || p->n_q_heads < 1 || p->n_q_heads % c->n_kv_heads || p->table_cols < 0 || p->window < 0 || p->max_new < 0 || p->max_kv < 0) return -1;
    if (!(p->scale == p->scale) || p->scale - p->scale != 0.0f) return -1;          // NaN or infinite
    if (c->head_dim % 8 || c->head_dim > 128 || p->n_q_heads / c->n_kv_heads > 128 || c->n_kv_heads > 65535) return -3;
    a.k = c->k; a.v = c->v; a.dtype = c->dtype; a.n_pages = c->n_pages; a.lp = log2_of(c->page_tokens); a.hkv = c->n_kv_heads; a.dim = c->head_dim;
    a.page_stride = c->page_stride; a.token_stride = c->token_stride; a.head_stride = c->head_stride;
    a.group = p->n_q_heads / c->n_kv_heads; a.n_rows = p->n_rows; a.n_seq = p->n_seq; a.cols = p->table_cols; a.table_stride = p->table_stride;
    a.q_row = p->q_row_stride; a.q_head = p->q_head_stride; a.o_row = p->out_row_stride; a.o_head = p->out_head_stride;
    a.window = p->window; a.max_new = p->max_new < p->n_rows ? p->max_new : p->n_rows; a.max_kv = p->max_kv; a.scale = p->scale;
    a.q = p->q; a.out = p->out; a.table = p->block_table; a.cu = p->cu_q; a.kv_lens = p->kv_lens;
    return 0;
}

}  // namespace
}  // namespace wmi

using namespace wmi;

extern "C" {

WHISPER_API int wmi_paged_plan(const int *ctx_lens, const int *new_lens, int n_seq, const int *free_pages, int n_free, int page_tokens, int *block_table,
                               int table_cols, long long table_stride, int *cu_q, int *kv_lens, int *slots, int *positions, int n_rows_cap, int *counts, void *stream) {
    if (n_seq < 0 || n_free < 0 || table_cols < 0 || table_stride < table_cols || n_rows_cap < 0 || !cu_q || !counts) return -1;
    if (n_seq > 0 && (!ctx_lens || !new_lens || !kv_lens)) return -1;
    if ((n_seq > 0 && table_cols > 0 && !block_table) || (n_free > 0 && !free_pages) || (n_rows_cap > 0 && (!slots || !positions))) return -1;
    if (!power_of_two(page_tokens) || page_tokens > 1024 || n_seq > kPlanMaxSeq || (long long)table_cols * page_tokens > 0x7fffffffLL) return -3;
    hipStream_t st = (hipStream_t)stream;
    const ServeCall call(st);
    if (!call.ok()) return -4;
    if (!call.own(cu_q, counts) || (n_seq > 0 && !call.own(ctx_lens, new_lens, kv_lens)) || (n_seq > 0 && table_cols > 0 && !call.owns(block_table)) ||
        (n_free > 0 && !call.owns(free_pages)) || (n_rows_cap > 0 && !call.own(slots, positions))) return -1;
    PlanArgs a{ctx_lens, new_lens, free_pages, block_table, cu_q, kv_lens, slots, positions, counts, (long)table_stride, n_seq, n_free, log2_of(page_tokens), table_cols, n_rows_cap};
    const size_t lds = 2 * sizeof(int) * ((size_t)n_seq + 1);
    if (lds > 48 * 1024 && hipFuncSetAttribute((const void *)paged_plan_kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds) != hipSuccess) { (void)hipGetLastError(); return -4; }
    // rows beyond a few thousand are spread over workgroups, one a CU at most (each repeats the prefix sum)
    const int want = (n_rows_cap + 4095) / 4096, groups = want < 1 ? 1 : want > 256 ? 256 : want;
    hipLaunchKernelGGL(paged_plan_kernel, dim3(groups), dim3(kPlanThreads), lds, st, a);
    return serve_done();
}

WHISPER_API int wmi_paged_write(const wmi_paged_cache *cache, const void *k_new, long long k_row_stride, long long k_head_stride, const void *v_new,
                                long long v_row_stride, long long v_head_stride, const int *slots, int n_rows, void *stream) {
    const int rc = check_cache(cache);
    if (rc) return rc;
    if (n_rows < 0 || (n_rows > 0 && (!k_new || !v_new || !slots)) || k_row_stride < 0 || k_head_stride < 0 || v_row_stride < 0 || v_head_stride < 0) return -1;
    if (n_rows == 0) return 0;
    hipStream_t st = (hipStream_t)stream;
    const ServeCall call(st);
    if (!call.ok()) return -4;
    if (!call.own(cache->k, cache->v, k_new, v_new, slots)) return -1;
    const long long all = cache->page_stride | cache->token_stride | cache->head_stride | k_row_stride | k_head_stride | v_row_stride | v_head_stride | cache->head_dim;
    const bool wide = all % 8 == 0 && aligned16(cache->k) && aligned16(cache->v) && aligned16(k_new) && aligned16(v_new);
    if (((uintptr_t)cache->k | (uintptr_t)cache->v | (uintptr_t)k_new | (uintptr_t)v_new) & 1) return -1;
    const int vec = wide ? 8 : 1, chunks = cache->head_dim / vec;
    if ((long long)cache->n_kv_heads * chunks > 0x7fffffffLL) return -3;
    WriteArgs a{(const char *)k_new, (const char *)v_new, (char *)cache->k, (char *)cache->v, slots, (long)k_row_stride * 2, (long)k_head_stride * 2, (long)v_row_stride * 2,
                (long)v_head_stride * 2, (long)cache->page_stride * 2, (long)cache->token_stride * 2, (long)cache->head_stride * 2,
                (long)cache->n_pages * cache->page_tokens, (long)n_rows * cache->n_kv_heads * chunks, log2_of(cache->page_tokens), cache->n_kv_heads, chunks};
    const long want = (a.total + 255) / 256;
    const unsigned blocks = (unsigned)(want > 65536 ? 65536 : want);
    if (wide) hipLaunchKernelGGL(paged_write_kernel<f32x4>, dim3(blocks), dim3(256), 0, st, a);
    else hipLaunchKernelGGL(paged_write_kernel<unsigned short>, dim3(blocks), dim3(256), 0, st, a);
    return serve_done();
}

WHISPER_API long long wmi_paged_attention_workspace(const wmi_paged_cache *cache, const wmi_paged_attn *args) {
    PagedAttn a;
    const int rc = fill_attn(cache, args, a);
    return rc ? rc : (long long)paged_attention_workspace(a);
}

WHISPER_API int wmi_paged_attention(const wmi_paged_cache *cache, const wmi_paged_attn *args, void *workspace, size_t workspace_bytes, void *stream) {
    PagedAttn a;
    const int rc = fill_attn(cache, args, a);
    if (rc) return rc;
    if (a.n_rows == 0 || a.n_seq == 0) return 0;
    if (!a.q || !a.out || !a.cu || !a.kv_lens || (a.cols > 0 && !a.table) || a.table_stride < a.cols) return -1;
    const long long all = a.page_stride | a.token_stride | a.head_stride | a.q_row | a.q_head | a.o_row | a.o_head;
    if (all % 8 || a.q_row < 0 || a.q_head < 0 || a.o_row < 0 || a.o_head < 0 || !aligned16(a.k) || !aligned16(a.v) || !aligned16(a.q) || !aligned16(a.out)) return -1;
    hipStream_t st = (hipStream_t)stream;
    const ServeCall call(st);
    if (!call.ok()) return -4;
    if (!call.own(a.k, a.v, a.q, (const void *)a.out, (const void *)a.cu, (const void *)a.kv_lens) || (a.cols > 0 && !call.owns(a.table))) return -1;
    const size_t need = paged_attention_workspace(a);
    if (need > workspace_bytes) return -2;
    if (need > 0 && (!aligned16(workspace) || !call.owns(workspace))) return -1;
    return paged_attention(a, workspace, st) ? 0 : -4;
}

}  // extern "C"
