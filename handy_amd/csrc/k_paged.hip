// Serving operators around a paged K/V cache, for gfx950: block tables and slot maps from request lengths, the new tokens' K and
// V into their slots, and attention of a chunk of new tokens (or one token) over the cache.
#include "kernels.h"
#include "serving_host.h"
#include <type_traits>

namespace wmi {

// ------------------------------------------------------------------------------------------ plan
// Request i has c cached and n new tokens. It needs ceil((c + n) / P) - ceil(c / P) fresh pages; the exclusive prefix sums of the
// new tokens and of the needs give its first row and its first entry in the free list. Requests are admitted in order up to the
// first (F) whose inclusive sums pass the row capacity or the free list.
// Every workgroup takes the whole prefix sum by itself (thousands of lengths, a few KB out of the L2: about 2 us) and keeps it in
// the LDS, so that rows and pages are then looked up by binary search there and the plan is one launch. Bound by latency: the lengths,
// the search (12 LDS reads for 4096 requests) and a row's table entry come one after the other; 5 us for 64 requests, 12 us for 4096
// with 290 000 rows.
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

    const unsigned gtid = blockIdx.x * blockDim.x + tid, gsize = gridDim.x * blockDim.x;        // (unsigned: a stride past the last of 2^31 - 1 rows must not wrap)
    // the last request whose sum is <= x among those that own anything: upper bound minus one
    auto owner = [&](const int *s, int x) { int lo = 0, hi = B; while (lo < hi) { const int m = (lo + hi) >> 1; if (s[m + 1] <= x) lo = m + 1; else hi = m; } return lo; };
    for (unsigned w = gtid; w < (unsigned)n_pag; w += gsize) {
        const int x = (int)w, i = owner(pag, x);
        a.table[i * a.table_stride + ((a.ctx[i] + P - 1) >> a.lp) + (x - pag[i])] = a.free_pages[x];
    }
    for (unsigned w = gtid; w < (unsigned)a.cap; w += gsize) {
        const int x = (int)w;
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
    for (int i = (int)gtid; i <= B; i += (int)gsize) {
        a.cu[i] = tok[i];
        if (i < B) { long long n, p; const bool ok = lengths(i, n, p); a.kv[i] = ok ? a.ctx[i] + (i < F ? (int)n : 0) : 0; }
    }
    if (gtid == 0) { a.counts[0] = F; a.counts[1] = n_tok; a.counts[2] = n_pag; a.counts[3] = sh_bad; }
}

// ------------------------------------------------------------------------------------------ write
// cache[slot[r]] = new[r] for K and V; a row whose slot lies outside the cache is skipped. A thread moves VEC elements of K and
// of V: bound by HBM (40 000 rows of 8 heads x 128, bf16: 54 us, 6.0 TB/s read and written).
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
// softmax(scale q K^T) V with the running maximum and sum of an online softmax. Both kernels compute, on MFMA,
//   S^T = K Q^T     K rows as the A operand, so that a lane holds scores of ONE query row (its column)
//   O^T += V^T P^T  P^T goes from the score registers straight into the B operand; V^T is read out of the row-major V tile with the
//                   LDS transpose load (4 keys of one dim a lane), in the key order the score registers hold
// The query rows of a request's tokens and of the heads that share a key head are packed into one list, row r = token * group +
// head, so that every K and V byte is read once for all of them.
//   paged_step_kernel    up to 16 packed rows (single tokens): bound by HBM. Each wave streams its own 16-key tiles. 64 requests of up
//                        to 8192 keys, 32/8 heads x 128, bf16, with the join: 190 - 209 us, 5.5 - 6.0 TB/s; 3 of 90 000 - 131 000 keys, f16:
//                        208 - 234 us, 6.2 - 6.9 TB/s (ranges over sessions; a pure read stream reaches 7.2).
//   paged_chunk_kernel   128 or 256 packed rows a workgroup, 64-key tiles shared by its waves. Three chunks of about 3800 tokens behind
//                        20 000 - 28 500 cached ones, 32/8 heads x 128, bf16: 4.9 - 5.7 ms, 940 - 1090 TFLOP/s; bound by issue: the matrix
//                        pipes are busy 43 % of the CU cycles, the vector instructions between two products (exponentials, conversions, the
//                        running maximum) fill the rest. Prompts of up to 224 tokens, 64 x 20 heads x 64, f16: 32 us, bound by the chain
//                        lengths - table - keys - two to four tiles in each short-lived workgroup.
// The keys of a tile of rows may be split over workgroups; paged_join_kernel adds the parts up.
// A probability is 2^(score c - m), c = |scale| log2(e). Its row's reference m is set by a largest score so far, whose own probability is 2^kBias
// then, and moves only when a score passes it by more than kMove (in powers of two), so that the accumulators are rescaled rarely instead of
// every tile. Probabilities are rounded to the cache's type for the product with V, their sums are of the unrounded ones (sums of the
// rounded ones: the same error, chunks 8 % slower). kBias puts f16's range above 1 to use: no probability reaches 2^16, and weights
// down to 2^-25 of the largest keep 11 bits, those down to 2^-36 fewer (with kBias 0 a long tail behind one key 17 nats above it came out 44 %
// too large). bf16 holds 8 bits whatever the size.
// (Chunks of 4096, f16, 128 dims: 5.82 ms with kMove + kBias = 4 + 11, 5.74 with 8 + 7, 5.90 with 2 + 13; single tokens and 64 dims do not tell
// them apart.)
typedef __bf16 bf16;
typedef bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef unsigned short u16x4 __attribute__((ext_vector_type(4)));
typedef unsigned short u16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

template <class T> struct Mma;
template <> struct Mma<f16> {
    typedef f16x8 V8; typedef f16x4 V4;
    static constexpr unsigned short kExp = 0x7c00, kOne = 0x3c00, kSign = 0x8000;
    static constexpr float kMove = 4.0f, kBias = 11.0f;
    static __device__ __forceinline__ f32x16 m32(V8 a, V8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
    static __device__ __forceinline__ f32x4 m16k32(V8 a, V8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
    static __device__ __forceinline__ f32x4 m16k16(V4 a, V4 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x16f16(a, b, c, 0, 0, 0); }
};
template <> struct Mma<bf16> {
    typedef bf16x8 V8; typedef bf16x4 V4;
    static constexpr unsigned short kExp = 0x7f80, kOne = 0x3f80, kSign = 0x8000;
    static constexpr float kMove = 8.0f, kBias = 0.0f;
    static __device__ __forceinline__ f32x16 m32(V8 a, V8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
    static __device__ __forceinline__ f32x4 m16k32(V8 a, V8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
    static __device__ __forceinline__ f32x4 m16k16(V4 a, V4 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(s16x4, a), __builtin_bit_cast(s16x4, b), c, 0, 0, 0);
    }
};

#define WMI_LDS __attribute__((address_space(3)))
#define WMI_GLB __attribute__((address_space(1)))

// LDS transpose loads: 16 lanes hand in the addresses of 4 rows x 16 columns (lane i: row i / 4, columns 4 (i % 4) ..), each gets one
// column's 4 rows. N of them at LDS addresses ad[] + OFF, waited for in the same block: as a builtin the compiler would also wait
// for every LDS-DMA in flight before each of them, the next tile's included.
__device__ __forceinline__ unsigned lds_addr(const char *p) { return (unsigned)(uintptr_t)(const WMI_LDS char *)p; }
template <int OFF> __device__ __forceinline__ void lds_read_tr(const unsigned (&ad)[4], s16x4 (&v)[4]) {
    asm volatile("ds_read_b64_tr_b16 %0, %4 offset:%8\n\tds_read_b64_tr_b16 %1, %5 offset:%8\n\tds_read_b64_tr_b16 %2, %6 offset:%8\n\t"
                 "ds_read_b64_tr_b16 %3, %7 offset:%8\n\ts_waitcnt lgkmcnt(0)"
                 : "=&v"(v[0]), "=&v"(v[1]), "=&v"(v[2]), "=&v"(v[3]) : "v"(ad[0]), "v"(ad[1]), "v"(ad[2]), "v"(ad[3]), "n"(OFF) : "memory");
}
template <int OFF> __device__ __forceinline__ void lds_read_tr(const unsigned (&ad)[8], s16x4 (&v)[8]) {
    asm volatile("ds_read_b64_tr_b16 %0, %8 offset:%16\n\tds_read_b64_tr_b16 %1, %9 offset:%16\n\tds_read_b64_tr_b16 %2, %10 offset:%16\n\t"
                 "ds_read_b64_tr_b16 %3, %11 offset:%16\n\tds_read_b64_tr_b16 %4, %12 offset:%16\n\tds_read_b64_tr_b16 %5, %13 offset:%16\n\t"
                 "ds_read_b64_tr_b16 %6, %14 offset:%16\n\tds_read_b64_tr_b16 %7, %15 offset:%16\n\ts_waitcnt lgkmcnt(0)"
                 : "=&v"(v[0]), "=&v"(v[1]), "=&v"(v[2]), "=&v"(v[3]), "=&v"(v[4]), "=&v"(v[5]), "=&v"(v[6]), "=&v"(v[7])
                 : "v"(ad[0]), "v"(ad[1]), "v"(ad[2]), "v"(ad[3]), "v"(ad[4]), "v"(ad[5]), "v"(ad[6]), "v"(ad[7]), "n"(OFF) : "memory");
}

// K and V tiles lie in the LDS as rows of DP elements, their 16-byte chunks permuted by row (chunk ^ swz(row)): the chunks that one
// fragment read touches (one chunk of 16 rows, or four chunks of four rows) then fall into different banks.
template <int DP> __device__ __forceinline__ int swz(int row) { return DP == 128 ? ((row & 3) << 2) | ((row >> 2) & 3) : (((row >> 1) & 1) << 2) | ((row >> 2) & 3); }

__device__ __attribute__((aligned(16))) unsigned attn_zero_chunk[4];     // what lanes without a key load

struct AttnReq { int q0, n, len; };
// lengths and offsets of a request, forced into the call's buffers whatever the arrays hold
__device__ __forceinline__ AttnReq attn_req(const PagedAttn &a, int cu0, int cu1, int kv_len) {
    AttnReq r;
    r.q0 = min(max(cu0, 0), a.n_rows);
    r.n = min(max(cu1, r.q0), a.n_rows) - r.q0;
    const long room = (long)a.cols << a.lp;
    r.len = (int)min((long)max(kv_len, 0), min(room, 0x7fffffffL));
    return r;
}
__device__ __forceinline__ AttnReq attn_req(const PagedAttn &a, int i) { return attn_req(a, a.cu[i], a.cu[i + 1], a.kv_lens[i]); }
// the first key that the row at position `pos` sees (a position in front of the keys and a window of 2^31 - 1 do not overflow)
__device__ __forceinline__ int attn_first_key(const PagedAttn &a, int pos) { return a.window > 0 && pos >= a.window ? pos - a.window + 1 : 0; }
// keys [lo, hi) that the packed rows r0 .. r1 - 1 of a request see between them
__device__ __forceinline__ void attn_keys(const PagedAttn &a, const AttnReq &q, int r0, int r1, int &lo, int &hi) {
    const int first = q.len - q.n + r0 / a.group, last = q.len - q.n + (r1 - 1) / a.group;
    hi = max(last + 1, 0);
    lo = attn_first_key(a, first);
}
// how many parts the keys of a tile of rows are cut into: at most `splits`, none shorter than `least` key tiles
__device__ __forceinline__ int attn_parts(int n_kt, int splits, int least) { return max(1, min(splits, n_kt / least)); }

constexpr int kStepRows = 16, kStepKeys = 16, kChunkKeys = 64;
constexpr int kStepLeast = 32, kChunkLeast = 4;        // shortest part, in key tiles (512 and 256 keys): below that the join costs more than it saves
constexpr int kMaxParts = 256;                         // the join gives every part a thread

// partial results of a split call: [part][row][query head][DP] accumulators, then {reference exponent, sum}
struct AttnParts { float *o; float2 *ml; int splits; };

// A row's reference while its keys go by. Where score * c is 2^20 or more, the rounded product that a reference is made of and the fma in
// the exponent part by a tenth of a power of two and more (from 2^28 on by more than the type's range: finite scores gave NaN, or zeros).
// Such a row takes its largest score off first, which leaves the largest ones exact; the products then only scale what is summed up already
// (and have to be finite themselves).
template <class T> struct AttnRef {
    float limit = -INFINITY;                               // scores above it move the reference (-infinity: none seen)
    float sub = 0.0f, base = 0.0f;                         // exponents are (score - base) c - sub; base 0: sub is the reference
    __device__ __forceinline__ float at(float c) const { return limit == -INFINITY ? limit : base != 0.0f ? base * c - Mma<T>::kBias : sub; }
    // to the largest score `top` if it passes the limit; the factor for what has been summed up
    __device__ __forceinline__ float move(float top, float c) {
        if (!(top > limit)) return 1.0f;
        const float was = at(c), mx = top * c;
        const bool big = fabsf(mx) >= 0x1p20f;
        base = big ? top : 0.0f;
        sub = (big ? 0.0f : mx) - Mma<T>::kBias;
        limit = big ? top : (sub + (Mma<T>::kBias + Mma<T>::kMove)) / c;
        return __builtin_amdgcn_exp2f(was - at(c));
    }
};

// A result in the cache's type. It is a mean of values of V, but the weights above the line are rounded and those below are not: a mean of
// f16's largest values can pass 65504 by that rounding and stays there. (Infinity and NaN, which V holds itself, go through.)
template <class T> __device__ __forceinline__ T attn_result(float x) {
    if constexpr (std::is_same<T, f16>::value) { if (fabsf(x) < INFINITY) x = __builtin_amdgcn_fmed3f(x, -65504.0f, 65504.0f); }
    return (T)x;
}

template <class T> __device__ __forceinline__ u16x4 not_finite(typename Mma<T>::V4 v) {
    const u16x4 b = __builtin_bit_cast(u16x4, v);
    return (u16x4)((b & Mma<T>::kExp) == Mma<T>::kExp);                    // all ones where infinite or NaN
}
template <class T> __device__ __forceinline__ u16x8 not_finite8(typename Mma<T>::V8 v) {
    const u16x8 b = __builtin_bit_cast(u16x8, v);
    return (u16x8)((b & Mma<T>::kExp) == Mma<T>::kExp);
}
__device__ __forceinline__ bool any_set(u16x4 v) { const uint2 w = __builtin_bit_cast(uint2, v); return (w.x | w.y) != 0; }
__device__ __forceinline__ bool any_set(u16x8 v) { const uint4 w = __builtin_bit_cast(uint4, v); return (w.x | w.y | w.z | w.w) != 0; }

// ---- single tokens (and any rows at all, 16 at a time)
// One workgroup = (request, key head, part of the keys); its 4 waves take 16-key tiles in turn, each through two LDS buffers of its
// own filled by LDS-DMA (no barrier in the loop: a wave waits for its own loads only, counted, so that the next tile is always on
// its way). A tile's page is one table entry (PAGE16: pages of 16 tokens and more); 64 tiles' entries are read at a time.
template <class T, int DP, bool PAGE16>
__global__ __launch_bounds__(256, 2) void paged_step_kernel(PagedAttn a, AttnParts ps) {
    typedef Mma<T> M;
    typedef typename M::V8 V8;
    typedef typename M::V4 V4;
    constexpr int CH = DP / 8, RPI = 64 / CH, NI = kStepKeys / RPI, TILE = kStepKeys * DP * 2, NB = DP / 16, NK = DP / 32;
    __shared__ __attribute__((aligned(16))) char smem[4 * 2 * 2 * TILE];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), n16 = lane & 15, g4 = lane >> 4;
    const int head = blockIdx.x % a.hkv, req = blockIdx.x / a.hkv, part = blockIdx.y;
    const AttnReq rq = attn_req(a, req);
    const int rows = rq.n * a.group, *tbl = a.table + req * a.table_stride;
    const float c = fmaxf(fabsf(a.scale) * 1.4426950408889634f, 1e-38f);    // a negative scale turns q round; 0 leaves equal scores
    const T *kc = (const T *)a.k + head * a.head_stride, *vc = (const T *)a.v + head * a.head_stride;
    char *mine = smem + wave * 4 * TILE;
    const int lrow = lane / CH, lslot = lane % CH;
    const long v_minus_k = (const char *)vc - (const char *)kc;
    const T *kl[NI];                                                       // a lane's address in load i of a tile, from the tile's first key on
    bool past[NI];                                                         // ... whose dims lie past the head's: zeros as K (q is 0 there, and infinity times 0 is none)
#pragma unroll
    for (int i = 0; i < NI; i++) {
        const int ch = lslot ^ swz<DP>(i * RPI + lrow);
        past[i] = ch * 8 >= a.dim;
        kl[i] = kc + (i * RPI + lrow) * a.token_stride + (past[i] ? 0 : ch * 8);                // (as V any of the key's own: what comes of them is not written)
    }

    for (int r0 = 0; r0 < rows; r0 += kStepRows) {
        const int r1 = min(rows, r0 + kStepRows);
        int lo, hi;
        attn_keys(a, rq, r0, r1, lo, hi);
        const int kt0 = lo / kStepKeys, n_kt = max((hi + kStepKeys - 1) / kStepKeys - kt0, 0), parts = attn_parts(n_kt, ps.splits, kStepLeast);
        if (part >= parts) continue;
        const int t0 = kt0 + (int)((long)n_kt * part / parts) + wave, t1 = kt0 + (int)((long)n_kt * (part + 1) / parts);
        const int row = min(r0 + n16, r1 - 1), tok = row / a.group, hq = head * a.group + row % a.group, pos = rq.len - rq.n + tok;
        const int first = rq.len - rq.n + r0 / a.group, klow = attn_first_key(a, pos);
        const bool one = r0 / a.group == (r1 - 1) / a.group;               // one token: every key in [lo, hi) is seen by every row
        V8 qf[NK];
#pragma unroll
        for (int ks = 0; ks < NK; ks++) {
            u16x8 x = {0, 0, 0, 0, 0, 0, 0, 0};
            const int e = ks * 32 + g4 * 8;
            if (e < a.dim) x = *(const u16x8 *)((const T *)a.q + (rq.q0 + tok) * a.q_row + hq * a.q_head + e);
            if (a.scale < 0.0f) x ^= M::kSign;
            qf[ks] = __builtin_bit_cast(V8, x);
        }
        f32x4 o[NB];
#pragma unroll
        for (int i = 0; i < NB; i++) o[i] = f32x4{0, 0, 0, 0};
        AttnRef<T> ref;
        bool shift = false;                                                // some row's scores are too large to do without base
        float l = 0.0f;
        int pg[PAGE16 ? 1 : NI];
        // table entries: PAGE16 -- lane x holds the entry of this wave's tile number (base + x); else one entry per load and lane
        auto entries = [&](int t) {
            if constexpr (PAGE16) {
                const long j = (long)(t + 4 * lane) * kStepKeys;
                pg[0] = j < hi ? tbl[j >> a.lp] : -1;
                __builtin_amdgcn_s_waitcnt(0xf70);                         // vmcnt(0): once in 64 tiles, so that the loop's waits stay counted
            } else {
#pragma unroll
                for (int i = 0; i < NI; i++) {                             // always loaded (clamped into the keys): the loop counts on NI loads
                    const int j = t * kStepKeys + i * RPI + lrow, e = tbl[min(max(j, lo), hi - 1) >> a.lp];
                    pg[i] = j >= lo && j < hi ? e : -1;
                }
            }
        };
        auto page_ok = [&](int p) { return (unsigned)p < (unsigned)a.n_pages; };
        auto copy = [&](const T *k, const T *v, int buf, int i) __attribute__((always_inline)) {       // (non-temporal: every byte is read once in the call)
            char *kd = mine + buf * 2 * TILE + i * 1024;
            __builtin_amdgcn_global_load_lds((const WMI_GLB void *)k, (WMI_LDS void *)kd, 16, 0, 2);
            __builtin_amdgcn_global_load_lds((const WMI_GLB void *)v, (WMI_LDS void *)(kd + TILE), 16, 0, 2);
        };
        auto stage = [&](int t, int buf, int at) {
            const int k0 = t * kStepKeys, up = PAGE16 ? __builtin_amdgcn_readlane(pg[0], at) : 0;
            if (PAGE16 && k0 >= lo && k0 + kStepKeys <= hi && page_ok(up)) {             // all keys exist, in one page: a scalar plus a constant of the lane
                const long off = up * a.page_stride + (long)(k0 & ((1 << a.lp) - 1)) * a.token_stride;
#pragma unroll
                for (int i = 0; i < NI; i++) {
                    const T *k = kl[i] + off;
                    copy(past[i] ? (const T *)attn_zero_chunk : k, (const T *)((const char *)k + v_minus_k), buf, i);
                }
                return;
            }
#pragma unroll
            for (int i = 0; i < NI; i++) {
                const int lr = i * RPI + lrow, j = k0 + lr, ch = lslot ^ swz<DP>(lr), page = PAGE16 ? up : pg[i];
                const bool on = j >= lo && j < hi && page_ok(page) && ch * 8 < a.dim;
                const long off = page * a.page_stride + (long)(j & ((1 << a.lp) - 1)) * a.token_stride + ch * 8;
                copy(on ? kc + off : (const T *)attn_zero_chunk, on ? vc + off : (const T *)attn_zero_chunk, buf, i);
            }
        };
        auto compute = [&](int t, int buf, bool page_bad, unsigned bad_keys) {
            const char *kb = mine + buf * 2 * TILE, *vb = kb + TILE;
            f32x4 s = {0, 0, 0, 0};
#pragma unroll
            for (int ks = 0; ks < NK; ks++) s = M::m16k32(*(const V8 *)(kb + n16 * DP * 2 + (((ks * 4 + g4) ^ swz<DP>(n16)) << 4)), qf[ks], s);
            const int k0 = t * kStepKeys;
            const bool cut = k0 < lo || k0 + kStepKeys > hi || page_bad, mixed = !one && (k0 + kStepKeys - 1 > first || a.window > 0);
            if (cut || mixed) {
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const int kk = g4 * 4 + r, j = k0 + kk;
                    if (j > pos || j < klow || j < lo || j >= hi || ((bad_keys >> kk) & 1)) s[r] = -INFINITY;
                }
            }
            const float mx = fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3]));
            if (__any(mx > ref.limit)) {
                const float top = fmaxf(mx, __shfl_xor(mx, 16)), al = ref.move(fmaxf(top, __shfl_xor(top, 32)), c);
                l *= al;
#pragma unroll
                for (int i = 0; i < NB; i++) o[i] *= al;
                shift = __any(ref.base != 0.0f);
            }
            if (shift) {
#pragma unroll
                for (int r = 0; r < 4; r++) s[r] -= ref.base;
            }
            V4 p;
#pragma unroll
            for (int r = 0; r < 4; r++) { const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r], c, -ref.sub)); l += e; p[r] = (T)e; }
            unsigned ad[NB];
            s16x4 raw[NB];
            V4 v[NB];
#pragma unroll
            for (int i = 0; i < NB; i++) {
                const int kr = g4 * 4 + (n16 >> 2), ch = i * 2 + ((n16 & 3) >> 1);
                ad[i] = lds_addr(vb + kr * DP * 2 + ((ch ^ swz<DP>(kr)) << 4) + (n16 & 1) * 8);
            }
            lds_read_tr<0>(ad, raw);
#pragma unroll
            for (int i = 0; i < NB; i++) v[i] = __builtin_bit_cast(V4, raw[i]);
            if (mixed) {                                                   // keys that some rows see and others do not: see seen_only below
                bool bad = false;
#pragma unroll
                for (int i = 0; i < NB; i++) bad |= any_set(not_finite<T>(v[i]));
                if (__any(bad)) {
                    u16x4 see;
#pragma unroll
                    for (int r = 0; r < 4; r++) see[r] = s[r] == -INFINITY ? 0 : M::kOne;
#pragma unroll
                    for (int i = 0; i < NB; i++) {
                        const u16x4 nf = not_finite<T>(v[i]);
                        const f32x4 cnt = M::m16k16(__builtin_bit_cast(V4, (u16x4)(nf & M::kOne)), __builtin_bit_cast(V4, see), f32x4{0, 0, 0, 0});
                        v[i] = __builtin_bit_cast(V4, (u16x4)(__builtin_bit_cast(u16x4, v[i]) & ~nf));
#pragma unroll
                        for (int r = 0; r < 4; r++) if (cnt[r] > 0.0f) o[i][r] = NAN;
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < NB; i++) o[i] = M::m16k16(v[i], p, o[i]);
        };
        if (t0 < t1) {
            // bit kk: key kk of the tile lies on a page the cache does not have
            auto bad_of = [&](int at) -> unsigned {
                if constexpr (PAGE16) return page_ok(__builtin_amdgcn_readlane(pg[0], at)) ? 0u : 0xffffu;
                else {
                    unsigned b = 0;
#pragma unroll
                    for (int i = 0; i < NI; i++) {
                        const unsigned long long v = __ballot(!page_ok(pg[i]));
#pragma unroll
                        for (int r = 0; r < RPI; r++) b |= (unsigned)((v >> (r * CH)) & 1) << (i * RPI + r);
                    }
                    return b;
                }
            };
            entries(t0);
            unsigned bad_now = bad_of(0), bad_next = 0;
            stage(t0, 0, 0);
            if constexpr (!PAGE16) entries(t0 + 4);
            int k = 1, buf = 0;                                            // k: number of the next tile within the 64 whose entries are held
            for (int t = t0; t < t1; t += 4, buf ^= 1) {
                const int tn = t + 4;
                if (tn < t1) {
                    if constexpr (PAGE16) { if (k == 64) { entries(tn); k = 0; } }
                    bad_next = bad_of(k);
                    stage(tn, buf ^ 1, k);
                    if constexpr (!PAGE16) entries(tn + 4);
                    k++;
                    if constexpr (PAGE16) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * NI) : "memory");
                    else asm volatile("s_waitcnt vmcnt(%0)" ::"n"(3 * NI) : "memory");
                } else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
                compute(t, buf, bad_now != 0, bad_now);
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");         // this buffer's reads are done before the next loads into it go out
                bad_now = bad_next;
            }
        }
        // the four waves' parts meet in the LDS
        l += __shfl_xor(l, 16); l += __shfl_xor(l, 32);
        __syncthreads();
        float *red = (float *)smem;                                        // [wave][row][DP + 2]
#pragma unroll
        for (int i = 0; i < NB; i++)
#pragma unroll
            for (int r = 0; r < 4; r++) red[(wave * kStepRows + n16) * (DP + 2) + i * 16 + g4 * 4 + r] = o[i][r];
        if (g4 == 0) { red[(wave * kStepRows + n16) * (DP + 2) + DP] = ref.at(c); red[(wave * kStepRows + n16) * (DP + 2) + DP + 1] = l; }
        __syncthreads();
        for (int x = tid; x < (r1 - r0) * (DP / 4); x += 256) {
            const int rr = x / (DP / 4), e = (x % (DP / 4)) * 4;
            if (e >= a.dim) continue;
            const float *w0 = red + rr * (DP + 2);
            constexpr int WS = kStepRows * (DP + 2);
            float mm = -INFINITY, ll = 0.0f, acc[4] = {0, 0, 0, 0};
#pragma unroll
            for (int w = 0; w < 4; w++) mm = fmaxf(mm, w0[w * WS + DP]);
#pragma unroll
            for (int w = 0; w < 4; w++) {
                const float mw = w0[w * WS + DP], f = mw == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(mw - mm);
                ll += w0[w * WS + DP + 1] * f;
#pragma unroll
                for (int r = 0; r < 4; r++) acc[r] += w0[w * WS + e + r] * f;
            }
            const int pr = r0 + rr, orow = rq.q0 + pr / a.group, oh = head * a.group + pr % a.group;
            if (parts == 1) {
                const float inv = ll == 0.0f ? 0.0f : 1.0f / ll;           // a row that sees nothing gives zeros
                V4 y;
#pragma unroll
                for (int r = 0; r < 4; r++) y[r] = attn_result<T>(acc[r] * inv);
                *(V4 *)((T *)a.out + orow * a.o_row + oh * a.o_head + e) = y;
            } else {
                const long at = ((long)part * a.n_rows + orow) * (a.hkv * a.group) + oh;
                *(f32x4 *)(ps.o + at * DP + e) = f32x4{acc[0], acc[1], acc[2], acc[3]};
                if (e == 0) ps.ml[at] = make_float2(mm, ll);
            }
        }
        __syncthreads();
    }
}

// ---- chunks of new tokens
// One workgroup = 4 or 8 waves of 32 packed rows of a request, one key head, one part of the keys. A row tile is found from the
// workgroup's number alone: request i's tiles start at number floor(cu[i] * group / rows) + i, which leaves room for all of them
// (a few numbers stay empty). Workgroups are dealt round-robin to the 8 XCDs: every XCD gets a contiguous run of (head, row
// tile), so that the row tiles that stream the same keys share an L2, the ones with the most keys first.
// Keys a row sees and others of its tile do not are masked to -infinity, p = 0; what V holds there must not be infinite or NaN in
// the product, so in tiles that need a mask such values are taken out and reach only the rows that do see them (as NaN).
template <class T, int DP, int WV>
__global__ __launch_bounds__(64 * WV, 2) void paged_chunk_kernel(PagedAttn a, AttnParts ps, int n_tiles) {
    typedef Mma<T> M;
    typedef typename M::V8 V8;
    typedef typename M::V4 V4;
    constexpr int ROWS = 32 * WV, CH = DP / 8, RPI = 64 / CH, NI = kChunkKeys / RPI / WV, TILE = kChunkKeys * DP * 2, NB = DP / 32, NK = DP / 16;
    __shared__ __attribute__((aligned(16))) char smem[2 * 2 * TILE];
    __shared__ __attribute__((aligned(16))) unsigned bad_flag[2][WV];       // per buffer: some key of this wave's share has no page ...
    __shared__ unsigned char bad_key[2][kChunkKeys];                       // ... and which
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), n32 = lane & 31, h = lane >> 5;
    const int nblk = gridDim.x, xq = nblk >> 3, xr = nblk & 7, xcd = blockIdx.x & 7, xi = blockIdx.x >> 3;
    const int logical = (xcd < xr ? xcd * (xq + 1) : xr * (xq + 1) + (xcd - xr) * xq) + xi;
    const int part = logical % ps.splits, tile = n_tiles - 1 - (logical / ps.splits) % n_tiles, head = logical / ps.splits / n_tiles;
    int req = 0, cu0, cu1, kv_len;
    for (int left = a.n_seq;;) {                                           // the last request whose first tile number is <= tile, 64 ways at a time
        const int step = (left + 63) / 64, i = min(req + lane * step, a.n_seq - 1), c0 = a.cu[i], c1 = a.cu[i + 1], kv = a.kv_lens[i];
        const bool ok = lane * step < left && (long)c0 * a.group / ROWS + i <= tile;
        const int k = __builtin_amdgcn_readfirstlane(max(__popcll(__ballot(ok)) - 1, 0));
        req += k * step; left = min(step, left - k * step);
        if (step == 1) {                                                   // its lane has what the request is (a round trip less before the first loads)
            cu0 = __builtin_amdgcn_readlane(c0, k); cu1 = __builtin_amdgcn_readlane(c1, k); kv_len = __builtin_amdgcn_readlane(kv, k);
            break;
        }
    }
    const AttnReq rq = attn_req(a, cu0, cu1, kv_len);
    const long r0l = ((long)tile - ((long)cu0 * a.group / ROWS + req)) * ROWS;
    const int rows = rq.n * a.group;
    if (r0l < 0 || r0l >= rows) return;
    const int r0 = (int)r0l, r1 = min(rows, r0 + ROWS);
    int lo, hi;
    attn_keys(a, rq, r0, r1, lo, hi);
    const int kt0 = lo / kChunkKeys, n_kt = max((hi + kChunkKeys - 1) / kChunkKeys - kt0, 0), parts = attn_parts(n_kt, ps.splits, kChunkLeast);
    if (part >= parts) return;
    const int t0 = kt0 + (int)((long)n_kt * part / parts), t1 = kt0 + (int)((long)n_kt * (part + 1) / parts);
    const int *tbl = a.table + req * a.table_stride;
    const float c = fmaxf(fabsf(a.scale) * 1.4426950408889634f, 1e-38f);
    const T *kc = (const T *)a.k + head * a.head_stride, *vc = (const T *)a.v + head * a.head_stride;

    const int w0 = r0 + wave * 32, row = min(w0 + n32, r1 - 1), tok = row / a.group, hq = head * a.group + row % a.group, pos = rq.len - rq.n + tok;
    const bool busy = w0 < r1;
    const int pmin = rq.len - rq.n + w0 / a.group, pmax = rq.len - rq.n + (min(w0 + 32, r1) - 1) / a.group;   // this wave's positions
    const int klow_min = attn_first_key(a, pmin), klow_max = attn_first_key(a, pmax);
    const int klow = attn_first_key(a, pos);
    V8 qf[NK];
#pragma unroll
    for (int ks = 0; ks < NK; ks++) {
        u16x8 x = {0, 0, 0, 0, 0, 0, 0, 0};
        const int e = ks * 16 + h * 8;
        if (e < a.dim) x = *(const u16x8 *)((const T *)a.q + (rq.q0 + tok) * a.q_row + hq * a.q_head + e);
        if (a.scale < 0.0f) x ^= M::kSign;
        qf[ks] = __builtin_bit_cast(V8, x);
    }
    // Loads: one wave instruction moves RPI keys (1 KB) of K or V; this wave's are key groups wave, wave + WV, .. of a tile. Where a
    // group lies in one page and every key of the tile exists, its address is a scalar (page, token) plus a constant of the lane;
    // the chunk a lane fetches does not depend on which of the wave's groups it is.
    const int lrow = lane / CH, lslot = lane % CH, lch = lslot ^ swz<DP>(wave * RPI + lrow);
    const bool past = lch * 8 >= a.dim;                                    // dims past the head's: zeros as K (q is 0 there, and infinity times 0 is none)
    const T *kl = kc + lrow * a.token_stride + (past ? 0 : lch * 8);       // (as V any of the key's own: what comes of them is not written)
    const long v_minus_k = (const char *)vc - (const char *)kc;
    int pages;                                                             // lane l: page of key group l of the tile that is loaded next
    auto entries = [&](int t) { const int j = t * kChunkKeys + (lane & (kChunkKeys / RPI - 1)) * RPI; return tbl[min(max(j, lo), hi - 1) >> a.lp]; };
    auto copy = [&](const T *k, const T *v, int buf, int i) __attribute__((always_inline)) {
        char *dst = smem + buf * 2 * TILE + (wave + WV * i) * 1024;
        __builtin_amdgcn_global_load_lds((const WMI_GLB void *)k, (WMI_LDS void *)dst, 16, 0, 0);
        __builtin_amdgcn_global_load_lds((const WMI_GLB void *)v, (WMI_LDS void *)(dst + TILE), 16, 0, 0);
    };
    auto stage = [&](int t, int buf) {
        const int k0 = t * kChunkKeys;
        bool inner = k0 >= lo && k0 + kChunkKeys <= hi && (1 << a.lp) >= RPI;
        if (inner) {
#pragma unroll
            for (int i = 0; i < NI; i++) inner &= (unsigned)__builtin_amdgcn_readlane(pages, wave + WV * i) < (unsigned)a.n_pages;
        }
        bool any = false;
        if (inner) {
#pragma unroll
            for (int i = 0; i < NI; i++) {
                const int page = __builtin_amdgcn_readlane(pages, wave + WV * i), token = (k0 + (wave + WV * i) * RPI) & ((1 << a.lp) - 1);
                const T *k = kl + (page * a.page_stride + token * a.token_stride);
                copy(past ? (const T *)attn_zero_chunk : k, (const T *)((const char *)k + v_minus_k), buf, i);
            }
        } else {                                                           // a tile at an end of the keys, or with a page that is not there
            bool bad = false;
            int pg[NI];
#pragma unroll
            for (int i = 0; i < NI; i++) {
                const int j = k0 + (wave + WV * i) * RPI + lrow;
                const bool in = j >= lo && j < hi;
                pg[i] = tbl[min(max(j, lo), hi - 1) >> a.lp];
                const bool has = (unsigned)pg[i] < (unsigned)a.n_pages, on = in && has && lch * 8 < a.dim;
                bad |= in && !has;
                const long off = pg[i] * a.page_stride + (long)(j & ((1 << a.lp) - 1)) * a.token_stride + lch * 8;
                copy(on ? kc + off : (const T *)attn_zero_chunk, on ? vc + off : (const T *)attn_zero_chunk, buf, i);
            }
            any = __any(bad);
            if (any && lslot == 0) {
#pragma unroll
                for (int i = 0; i < NI; i++) bad_key[buf][(wave + WV * i) * RPI + lrow] = (unsigned)pg[i] >= (unsigned)a.n_pages;
            }
        }
        if (lane == 0) bad_flag[buf][wave] = any;
    };
    f32x16 o[NB];
#pragma unroll
    for (int b = 0; b < NB; b++)
#pragma unroll
        for (int i = 0; i < 16; i++) o[b][i] = 0.0f;
    AttnRef<T> ref;
    bool shift = false;                                                    // some row's scores are too large to do without base
    float l = 0.0f;
    const int kf = n32 * DP * 2 + ((h ^ swz<DP>(n32)) << 4);               // K fragment ks of half kh: kb + kh * 32 rows + (kf ^ ks * 32)
    const int vrow = 4 * h + ((lane & 15) >> 2), vcol = ((lane >> 4) & 1) * 2 + ((lane & 3) >> 1);
    const int vf = vrow * DP * 2 + ((vcol ^ swz<DP>(vrow)) << 4) + (lane & 1) * 8;   // V^T of keys 8 x + vrow: vb + 8 x rows + (vf ^ block * 64 ^ (x & 1) * 32)
    // V^T fragments of keys 16 s + {4 h + 0..3, 8 + 4 h + 0..3} for all blocks of 32 dims
    auto read_v = [&](const unsigned (&ad)[2 * NB], auto s_tag, V8 (&v)[NB]) __attribute__((always_inline)) {
        constexpr int S = decltype(s_tag)::value;
        s16x4 raw[2 * NB];
        lds_read_tr<16 * S * DP * 2>(ad, raw);
#pragma unroll
        for (int b = 0; b < NB; b++) {
            const s16x4 x = raw[2 * b], y = raw[2 * b + 1];
            v[b] = __builtin_bit_cast(V8, __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
        }
    };

    if (t0 < t1) { pages = entries(t0); stage(t0, 0); pages = entries(t0 + 1); }
    for (int t = t0; t < t1; t++) {
        const int buf = (t - t0) & 1, k0 = t * kChunkKeys;
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");   // everybody's share of this tile has landed, the other buffer is free
        if (t + 1 < t1) { stage(t + 1, buf ^ 1); pages = entries(t + 2); }
        if (!busy || k0 > pmax || k0 + kChunkKeys <= klow_min) continue;
        const char *kb = smem + buf * 2 * TILE, *vb = kb + TILE;
        f32x16 s[2];
#pragma unroll
        for (int kh = 0; kh < 2; kh++) {
#pragma unroll
            for (int i = 0; i < 16; i++) s[kh][i] = 0.0f;
#pragma unroll
            for (int ks = 0; ks < NK; ks++) s[kh] = M::m32(*(const V8 *)(kb + kh * 32 * DP * 2 + (kf ^ (ks * 32))), qf[ks], s[kh]);
        }
        unsigned flags = 0;
#pragma unroll
        for (int w = 0; w < WV; w++) flags |= bad_flag[buf][w];
        const bool hole = __builtin_amdgcn_readfirstlane(flags) != 0;
        const bool mixed = k0 + kChunkKeys - 1 > pmin || k0 < klow_max || hole;
        if (mixed) {
#pragma unroll
            for (int kh = 0; kh < 2; kh++)
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    const int kk = kh * 32 + (i & 3) + 8 * (i >> 2) + 4 * h, j = k0 + kk;
                    if (j > pos || j < klow) s[kh][i] = -INFINITY;
                }
            if (hole) {
#pragma unroll
                for (int kh = 0; kh < 2; kh++)
#pragma unroll
                    for (int i = 0; i < 16; i++) {
                        const int kk = kh * 32 + (i & 3) + 8 * (i >> 2) + 4 * h;
                        if (bad_flag[buf][(kk / RPI) % WV] && bad_key[buf][kk]) s[kh][i] = -INFINITY;
                    }
            }
        }
        float mx = -INFINITY;
#pragma unroll
        for (int kh = 0; kh < 2; kh++)
#pragma unroll
            for (int i = 0; i < 16; i++) mx = fmaxf(mx, s[kh][i]);
        if (__any(mx > ref.limit)) {
            const float al = ref.move(fmaxf(mx, __shfl_xor(mx, 32)), c);
            l *= al;
#pragma unroll
            for (int b = 0; b < NB; b++) o[b] *= al;
            shift = __any(ref.base != 0.0f);
        }
        if (shift) {
#pragma unroll
            for (int kh = 0; kh < 2; kh++)
#pragma unroll
                for (int i = 0; i < 16; i++) s[kh][i] -= ref.base;
        }
        V8 p[4];
#pragma unroll
        for (int kh = 0; kh < 2; kh++)
#pragma unroll
            for (int i = 0; i < 16; i++) {
                const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kh][i], c, -ref.sub));
                l += e;
                p[kh * 2 + (i >> 3)][i & 7] = (T)e;
            }
        unsigned ad[2 * NB];
#pragma unroll
        for (int b = 0; b < NB; b++) { ad[2 * b] = lds_addr(vb + (vf ^ (b * 64))); ad[2 * b + 1] = lds_addr(vb + 8 * DP * 2 + (vf ^ (b * 64) ^ 32)); }
        auto pv = [&](auto x_tag) __attribute__((always_inline)) {
            constexpr int X = decltype(x_tag)::value;
            V8 v[NB];
            read_v(ad, x_tag, v);
            if (mixed) {
                u16x8 bad = not_finite8<T>(v[0]);
#pragma unroll
                for (int b = 1; b < NB; b++) bad |= not_finite8<T>(v[b]);
                if (__any(any_set(bad))) {
                    u16x8 see;
#pragma unroll
                    for (int i = 0; i < 8; i++) see[i] = s[X >> 1][(X & 1) * 8 + i] == -INFINITY ? 0 : M::kOne;
#pragma unroll
                    for (int b = 0; b < NB; b++) {
                        const u16x8 nf = not_finite8<T>(v[b]);
                        f32x16 cnt;
#pragma unroll
                        for (int i = 0; i < 16; i++) cnt[i] = 0.0f;
                        cnt = M::m32(__builtin_bit_cast(V8, (u16x8)(nf & M::kOne)), __builtin_bit_cast(V8, see), cnt);
#pragma unroll
                        for (int i = 0; i < 16; i++) if (cnt[i] > 0.0f) o[b][i] = NAN;
                        v[b] = __builtin_bit_cast(V8, (u16x8)(__builtin_bit_cast(u16x8, v[b]) & ~nf));
                    }
                }
            }
#pragma unroll
            for (int b = 0; b < NB; b++) o[b] = M::m32(v[b], p[X], o[b]);
        };
        pv(std::integral_constant<int, 0>());
        pv(std::integral_constant<int, 1>());
        pv(std::integral_constant<int, 2>());
        pv(std::integral_constant<int, 3>());
    }
    l += __shfl_xor(l, 32);
    if (w0 + n32 >= r1) return;                                            // rows past the tile's last one repeat it
    if (parts == 1) {
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        T *dst = (T *)a.out + (rq.q0 + tok) * a.o_row + hq * a.o_head;
        float big = 0.0f;
#pragma unroll
        for (int b = 0; b < NB; b++) {
            o[b] *= inv;
#pragma unroll
            for (int i = 0; i < 16; i++) big = fmaxf(big, fabsf(o[b][i]));
        }
        if (std::is_same<T, f16>::value && big > 65504.0f) {               // (attn_result for each costs short prompts 2.5 % instead of 1)
#pragma unroll
            for (int b = 0; b < NB; b++)
#pragma unroll
                for (int i = 0; i < 16; i++) o[b][i] = (float)attn_result<T>(o[b][i]);
        }
#pragma unroll
        for (int b = 0; b < NB; b++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int e = b * 32 + 8 * i + 4 * h;
                if (e < a.dim) *(V4 *)(dst + e) = V4{(T)o[b][4 * i], (T)o[b][4 * i + 1], (T)o[b][4 * i + 2], (T)o[b][4 * i + 3]};
            }
    } else {
        const long at = ((long)part * a.n_rows + rq.q0 + tok) * (a.hkv * a.group) + hq;
#pragma unroll
        for (int b = 0; b < NB; b++)
#pragma unroll
            for (int i = 0; i < 4; i++) *(f32x4 *)(ps.o + at * DP + b * 32 + 8 * i + 4 * h) = f32x4{o[b][4 * i], o[b][4 * i + 1], o[b][4 * i + 2], o[b][4 * i + 3]};
        if (h == 0) ps.ml[at] = make_float2(ref.at(c), l);
    }
}

// out = sum over a row's parts. One workgroup a (row, query head), the parts dealt to its 4 waves and added up in a fixed order; the
// number of parts follows from the lengths as in the kernel that made them (tiles of ROWS packed rows, KEYS keys).
template <class T, int DP, int ROWS, int KEYS, int LEAST>
__global__ __launch_bounds__(256) void paged_join_kernel(PagedAttn a, AttnParts ps) {
    constexpr int E = DP / 64;                                             // dims of a lane
    __shared__ float scale_of[kMaxParts], red[4][DP], sum[4];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, hqs = a.hkv * a.group, row = blockIdx.x / hqs, hq = blockIdx.x % hqs;
    int lo = 0, hi = a.n_seq;
    while (lo < hi) { const int x = (lo + hi) >> 1; if (a.cu[x + 1] <= row) lo = x + 1; else hi = x; }
    if (lo >= a.n_seq || row < a.cu[lo]) return;
    const AttnReq rq = attn_req(a, lo);
    const int pr = (row - rq.q0) * a.group + hq % a.group, r0 = pr / ROWS * ROWS, r1 = min(rq.n * a.group, r0 + ROWS);
    int k0, k1;
    attn_keys(a, rq, r0, r1, k0, k1);
    const int n_kt = max((k1 + KEYS - 1) / KEYS - k0 / KEYS, 0), parts = attn_parts(n_kt, ps.splits, LEAST);
    if (parts == 1) return;                                                // written by the kernel itself
    const long stride = (long)a.n_rows * hqs, at = (long)row * hqs + hq;
    const float2 ml = tid < parts ? ps.ml[tid * stride + at] : make_float2(-INFINITY, 0.0f);
    float m = ml.x;
    for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
    if (lane == 0) sum[wave] = m;
    __syncthreads();
    m = fmaxf(fmaxf(sum[0], sum[1]), fmaxf(sum[2], sum[3]));
    const float f = ml.x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(ml.x - m);
    float l = ml.y * f;
    for (int o = 32; o > 0; o >>= 1) l += __shfl_xor(l, o);
    scale_of[tid] = f;
    __syncthreads();
    if (lane == 0) sum[wave] = l;
    float acc[E] = {};
    const float *src = ps.o + at * DP + lane * E;
#pragma unroll 8
    for (int p = wave; p < parts; p += 4) {
#pragma unroll
        for (int e = 0; e < E; e++) acc[e] += src[p * stride * DP + e] * scale_of[p];
    }
#pragma unroll
    for (int e = 0; e < E; e++) red[wave][lane * E + e] = acc[e];
    __syncthreads();
    l = (sum[0] + sum[1]) + (sum[2] + sum[3]);
    if (tid < a.dim) ((T *)a.out)[row * a.o_row + hq * a.o_head + tid] = attn_result<T>(((red[0][tid] + red[1][tid]) + (red[2][tid] + red[3][tid])) * (l == 0.0f ? 0.0f : 1.0f / l));
}

// How a call is cut up. The step kernel takes calls whose requests bring at most 16 packed rows each, as far as the caller says;
// it is right for any, 16 rows at a time.
struct AttnShape { bool step; int waves, tiles, splits; };
static AttnShape attn_shape(const PagedAttn &a) {
    AttnShape s;
    const long new_rows = (long)(a.max_new > 0 ? a.max_new : a.n_rows) * a.group, keys = a.max_kv > 0 ? a.max_kv : 0x7fffffff;
    s.step = new_rows <= kStepRows;
    // Eight waves share a tile where the keys of one head outgrow an XCD's 4 MB of L2 (8192 keys of 128 dims) and there are rows for
    // them: half the tile traffic (chunks of 4096 at 28 000 keys 5.2 ms against 5.65). Four otherwise: less waiting for each
    // other and less idle in a request's last tile (prompts of up to 224 tokens 34 us against 54, 64 dims 3.1 ms against 3.5).
    s.waves = a.dim > 64 && keys > 8192 && new_rows >= 256 ? 8 : 4;
    s.tiles = s.step ? a.n_seq : (int)((long)a.n_rows * a.group / (32 * s.waves) + a.n_seq);
    const long work = (long)s.tiles * a.hkv, full = s.step ? 2048 : 1024, least = s.step ? kStepLeast * kStepKeys : kChunkLeast * kChunkKeys;
    long n = full / work;
    if (n > keys / least) n = keys / least;
    const bool joinable = (long)a.n_rows * a.hkv * a.group < 1L << 24;     // (the join's 256 threads a pair fit a grid)
    s.splits = n < 1 || !joinable ? 1 : n > kMaxParts ? kMaxParts : (int)n;
    return s;
}

size_t paged_attention_workspace(const PagedAttn &a) {
    if (a.n_rows == 0 || a.n_seq == 0) return 0;
    const AttnShape s = attn_shape(a);
    const size_t each = (size_t)s.splits * a.n_rows * a.hkv * a.group;
    return s.splits == 1 ? 0 : each * ((a.dim <= 64 ? 64 : 128) * sizeof(float) + sizeof(float2));
}

template <class T, int DP> static bool attn_launch(const PagedAttn &a, void *workspace, hipStream_t st) {
    const AttnShape s = attn_shape(a);
    const long pairs = (long)a.n_rows * a.hkv * a.group;
    const AttnParts ps{(float *)workspace, (float2 *)((float *)workspace + (s.splits == 1 ? 0 : s.splits * pairs * DP)), s.splits};
    const dim3 join((unsigned)pairs);
    bool ok;
    if (s.step) {
        const dim3 grid((unsigned)(a.n_seq * a.hkv), s.splits);
        ok = serve_launch(a.lp >= 4 ? paged_step_kernel<T, DP, true> : paged_step_kernel<T, DP, false>, grid, dim3(256), 0, st, a, ps);
        if (s.splits > 1) ok = ok && serve_launch(paged_join_kernel<T, DP, kStepRows, kStepKeys, kStepLeast>, join, dim3(256), 0, st, a, ps);
    } else {
        const dim3 grid((unsigned)((long)s.tiles * a.hkv * s.splits)), threads(64 * s.waves);
        ok = serve_launch(s.waves == 8 ? paged_chunk_kernel<T, DP, 8> : paged_chunk_kernel<T, DP, 4>, grid, threads, 0, st, a, ps, s.tiles);
        if (s.splits > 1) ok = ok && serve_launch(s.waves == 8 ? paged_join_kernel<T, DP, 256, kChunkKeys, kChunkLeast> : paged_join_kernel<T, DP, 128, kChunkKeys, kChunkLeast>, join, dim3(256), 0, st, a, ps);
    }
    return ok;
}

bool paged_attention(const PagedAttn &a, void *workspace, hipStream_t st) {
    if (a.dtype == WMI_F16) return a.dim <= 64 ? attn_launch<f16, 64>(a, workspace, st) : attn_launch<f16, 128>(a, workspace, st);
    return a.dim <= 64 ? attn_launch<bf16, 64>(a, workspace, st) : attn_launch<bf16, 128>(a, workspace, st);
}

namespace {

int log2_of(int x) { int l = 0; while ((1 << l) < x) l++; return l; }
bool power_of_two(int x) { return x > 0 && !(x & (x - 1)); }

// what every entry asks of a cache description, its memory apart; 0, -1 or -3
int check_cache(const wmi_paged_cache *c) {
    if (!c || c->n_pages < 1 || c->n_kv_heads < 1 || c->head_dim < 1) return -1;
    if (c->dtype != WMI_F16 && c->dtype != WMI_BF16) return -1;
    if (c->page_stride < 0 || c->token_stride < 0 || c->head_stride < 0) return -1;
    if (!power_of_two(c->page_tokens) || c->page_tokens > 1024 || (long long)c->n_pages * c->page_tokens > 0x7fffffffLL) return -3;
    return 0;
}
bool aligned16(const void *p) { return ((uintptr_t)p & 15) == 0; }

// whether two [rows][heads][dim] arrays of the same strides share an element, the second `delta` elements behind the first (self: an
// array with itself, two of its rows or heads)
bool rows_meet(long delta, long rows, long heads, long dim, long row, long head, bool self) {
    if (self && ((head >= dim && row >= head * (heads - 1) + dim) || (row >= dim && head >= row * (rows - 1) + dim))) return false;      // one axis inside the other
    for (long dh = 1 - heads; dh < heads; dh++) {
        const long x = delta - dh * head, d0 = row > 0 ? x / row : 0;
        for (long d = d0 - 1; d <= d0 + 1; d++) {                       // the nearest row steps there are
            const long dr = d < 1 - rows ? 1 - rows : d > rows - 1 ? rows - 1 : d, gap = x - dr * row;
            if (gap > -dim && gap < dim && !(self && dh == 0 && dr == 0)) return true;
        }
    }
    return false;
}
// whether what attention writes (out, the workspace) meets anything else of the call
bool attn_shares(const PagedAttn &a, const void *workspace, size_t ws_bytes) {
    struct Span { uintptr_t at, end; };
    auto span = [](const void *p, long bytes) { return Span{(uintptr_t)p, (uintptr_t)p + (uintptr_t)bytes}; };
    auto meet = [](Span x, Span y) { return x.at < y.end && y.at < x.end; };
    const long heads = (long)a.hkv * a.group, kv = 2 * ((a.n_pages - 1) * a.page_stride + ((1L << a.lp) - 1) * a.token_stride + (a.hkv - 1) * a.head_stride + a.dim);
    const Span q = span(a.q, 2 * ((a.n_rows - 1) * a.q_row + (heads - 1) * a.q_head + a.dim)), out = span(a.out, 2 * ((a.n_rows - 1) * a.o_row + (heads - 1) * a.o_head + a.dim));
    const Span ws = span(workspace, (long)ws_bytes);
    const Span other[] = {span(a.k, kv), span(a.v, kv), span(a.table, a.cols > 0 ? 4 * ((a.n_seq - 1) * a.table_stride + a.cols) : 0), span(a.cu, 4 * (a.n_seq + 1L)), span(a.kv_lens, 4L * a.n_seq)};
    for (const Span &o : other) if (meet(out, o) || (ws_bytes > 0 && meet(ws, o))) return true;
    if (ws_bytes > 0 && (meet(ws, q) || meet(ws, out))) return true;
    if (rows_meet(0, a.n_rows, heads, a.dim, a.o_row, a.o_head, true)) return true;
    // q and out may be parts of one buffer's rows: spans that meet are looked at closely if their strides are alike
    return meet(out, q) && (a.q_row != a.o_row || a.q_head != a.o_head || rows_meet(((long)out.at - (long)q.at) / 2, a.n_rows, heads, a.dim, a.o_row, a.o_head, false));
}

// the description in the kernels' terms, checked; 0, -1 or -3
int fill_attn(const wmi_paged_cache *c, const wmi_paged_attn *p, PagedAttn &a) {
    const int rc = check_cache(c);
    if (rc) return rc;
    if (!p || p->n_rows < 0 || p->n_seq < 0 || p->n_q_heads < 1 || p->n_q_heads % c->n_kv_heads || p->table_cols < 0 || p->window < 0 || p->max_new < 0 || p->max_kv < 0) return -1;
    if (!(p->scale == p->scale) || p->scale - p->scale != 0.0f) return -1;          // NaN or infinite
    if (c->head_dim % 8 || c->head_dim > 128 || p->n_q_heads / c->n_kv_heads > 128) return -3;
    if ((long long)p->n_rows * p->n_q_heads > 0x3fffffffLL || (long long)p->n_seq * c->n_kv_heads > 0x3fffffLL) return -3;      // workgroup and packed row numbers are 32-bit
    if ((long long)p->table_cols * c->page_tokens > 0x7fffff00LL) return -3;      // key numbers are 32-bit, and the kernels' run up to 255 past the last
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
    // Workgroups read all lengths while others write: what is written overlaps nothing else (the last plan's kv_lens as this one's
    // ctx_lens in the same buffer would).
    const struct { const void *p; long long n; } use[] = {{ctx_lens, n_seq}, {new_lens, n_seq}, {free_pages, n_free}, {block_table, n_seq > 0 && table_cols > 0 ? (n_seq - 1) * table_stride + table_cols : 0},
                                                          {cu_q, n_seq + 1LL}, {kv_lens, n_seq}, {slots, n_rows_cap}, {positions, n_rows_cap}, {counts, 4}};
    for (int i = 3; i < 9; i++)
        for (int j = 0; j < i; j++)
            if (use[i].n > 0 && use[j].n > 0 && (uintptr_t)use[i].p < (uintptr_t)use[j].p + 4 * use[j].n && (uintptr_t)use[j].p < (uintptr_t)use[i].p + 4 * use[i].n) return -1;
    hipStream_t st = (hipStream_t)stream;
    const ServeCall call(st);
    if (!call.ok()) return -4;
    if (!call.own(cu_q, counts) || (n_seq > 0 && !call.own(ctx_lens, new_lens, kv_lens)) || (n_seq > 0 && table_cols > 0 && !call.owns(block_table)) ||
        (n_free > 0 && !call.owns(free_pages)) || (n_rows_cap > 0 && !call.own(slots, positions))) return -1;
    PlanArgs a{ctx_lens, new_lens, free_pages, block_table, cu_q, kv_lens, slots, positions, counts, (long)table_stride, n_seq, n_free, log2_of(page_tokens), table_cols, n_rows_cap};
    const size_t lds = 2 * sizeof(int) * ((size_t)n_seq + 1);
    if (lds > 48 * 1024 && hipFuncSetAttribute((const void *)paged_plan_kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds) != hipSuccess) { (void)hipGetLastError(); return -4; }
    // rows beyond two a thread are spread over workgroups, one a CU at most, each of which repeats the prefix sum (4096 requests and 303 000
    // rows, the whole call: 11.8 us with 2048 rows a workgroup, 12.0 with 1024, 14.0 with 4096)
    const int want = n_rows_cap / 2048 + (n_rows_cap % 2048 != 0), groups = want < 1 ? 1 : want > 256 ? 256 : want;
    return serve_launch(paged_plan_kernel, dim3(groups), dim3(kPlanThreads), lds, st, a) ? 0 : -4;
}

WHISPER_API int wmi_paged_write(const wmi_paged_cache *cache, const void *k_new, long long k_row_stride, long long k_head_stride, const void *v_new,
                                long long v_row_stride, long long v_head_stride, const int *slots, int n_rows, void *stream) {
    const int rc = check_cache(cache);
    if (rc) return rc;
    if (!cache->k || !cache->v || n_rows < 0 || (n_rows > 0 && (!k_new || !v_new || !slots)) || k_row_stride < 0 || k_head_stride < 0 || v_row_stride < 0 || v_head_stride < 0) return -1;
    if (n_rows == 0) return 0;
    if (cache->k == cache->v && (k_new != v_new || k_row_stride != v_row_stride || k_head_stride != v_head_stride)) return -1;      // two values for one place
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
    return serve_launch(wide ? paged_write_kernel<f32x4> : paged_write_kernel<unsigned short>, dim3(blocks), dim3(256), 0, st, a) ? 0 : -4;
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
    if (!a.k || !a.v) return -1;
    if (a.n_rows == 0 || a.n_seq == 0) return 0;
    if (!a.q || !a.out || !a.cu || !a.kv_lens || (a.cols > 0 && !a.table) || a.table_stride < a.cols) return -1;
    const long long all = a.page_stride | a.token_stride | a.head_stride | a.q_row | a.q_head | a.o_row | a.o_head;
    if (all % 8 || a.q_row < 0 || a.q_head < 0 || a.o_row < 0 || a.o_head < 0 || !aligned16(a.k) || !aligned16(a.v) || !aligned16(a.q) || !aligned16(a.out)) return -1;
    const size_t need = paged_attention_workspace(a);
    if (need > workspace_bytes) return -2;
    if (need > 0 && (!workspace || !aligned16(workspace))) return -1;
    if (attn_shares(a, workspace, need)) return -1;
    hipStream_t st = (hipStream_t)stream;
    const ServeCall call(st);
    if (!call.ok()) return -4;
    if (!call.own(a.k, a.v, a.q, (const void *)a.out, (const void *)a.cu, (const void *)a.kv_lens) || (a.cols > 0 && !call.owns(a.table))) return -1;
    if (need > 0 && !call.owns(workspace)) return -1;
    return paged_attention(a, workspace, st) ? 0 : -4;
}

}  // extern "C"
