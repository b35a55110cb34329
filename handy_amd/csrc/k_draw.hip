// One token a row from its logits, for gfx950: temperature, top-k, top-p, min-p, and a draw from a given uniform number.
#include "kernels.h"
#include "serving_host.h"

namespace wmi {

// Weights w_i = exp((x_i - max x) / T) lie in [0, 1] and are computed in 64 bits, then held as whole numbers of 2^-45: sums of up
// to 2^18 of them fit 64 bits and are exact, so they do not depend on the order in which they are made, and every comparison of
// running masses (top-p's border, the draw) is exact. What the rounding of a weight costs is 2^-46 of the largest one.
// The filters keep a prefix of the order (x descending, index ascending): the prefix ends inside the entries of one value (the
// cut), of which the first few by index are kept.
constexpr int kDrawThreads = 1024, kDrawWaves = kDrawThreads / 64;
constexpr double kMassOne = 35184372088832.0;               // 2^45

typedef unsigned long long u64;

// unsigned order of floats: key(a) < key(b) <=> a < b; -0 counts as +0, NaN as -infinity
__device__ __forceinline__ unsigned draw_key(float x) {
    x = x + 0.0f;
    if (!(x == x)) x = -INFINITY;
    const unsigned u = __float_as_uint(x);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float draw_val(unsigned k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }
constexpr unsigned kKeyNone = 0x007fffffu;                   // key(-infinity): entries that cannot be drawn

__device__ __forceinline__ u64 mass_of(double w) { return (u64)(w * kMassOne + 0.5); }

__device__ __forceinline__ u64 wave_sum64(u64 v) { for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o); return v; }
__device__ u64 draw_block_sum(u64 v, u64 *sh) {
    v = wave_sum64(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
    __syncthreads();
    u64 s = 0;
    for (int w = 0; w < kDrawWaves; w++) s += sh[w];
    return s;
}

template <class T>
__global__ __launch_bounds__(kDrawThreads) void draw_kernel(DrawArgs a) {
    __shared__ u64 sh[kDrawWaves];
    __shared__ u64 bins[256];
    __shared__ unsigned sh_digit, sh_top, sh_idx;
    __shared__ u64 sh_above;
    __shared__ int sh_tok;
    const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, V = a.n_vocab;
    const T *x = (const T *)a.logits + row * a.row_stride;
    auto key = [&](int i) { return draw_key((float)x[i]); };
    // largest value, its lowest index
    if (tid == 0) { sh_top = 0; sh_idx = 0xffffffffu; }
    __syncthreads();
    unsigned top = 0;
    for (int i = tid; i < V; i += kDrawThreads) top = max(top, key(i));
    atomicMax(&sh_top, top);
    __syncthreads();
    top = sh_top;
    for (int i = tid; i < V; i += kDrawThreads) if (key(i) == top) { atomicMin(&sh_idx, (unsigned)i); break; }
    __syncthreads();
    const int best = (int)sh_idx;
    if (top <= kKeyNone) {                                    // nothing can be drawn
        if (tid == 0) { a.token[row] = -1; if (a.logprob) a.logprob[row] = -INFINITY; }
        return;
    }
    const float t_in = a.temperature ? a.temperature[row] : 1.0f;
    const bool drawn = t_in > 0.0f;
    const double T64 = drawn ? (double)t_in : 1.0, topv = (double)draw_val(top);
    auto weight = [&](unsigned k) { return k == top ? 1.0 : k <= kKeyNone ? 0.0 : exp(((double)draw_val(k) - topv) / T64); };
    u64 z = 0;
    for (int i = tid; i < V; i += kDrawThreads) z += mass_of(weight(key(i)));
    z = draw_block_sum(z, sh);
    int token = best;
    if (drawn) {
        // the cut: entries above cut_key are kept, and the first `ties` entries (by index) equal to it
        unsigned cut_key = kKeyNone;
        u64 ties = 0;
        // radix selection from the top: the key at which the running sum of measure(key), from the largest key down, reaches `want`
        // (> 0); above: the sum over larger keys. Entries below or at kKeyNone count nothing.
        auto select = [&](u64 want, auto measure, unsigned &k_out, u64 &above_out) {
            unsigned prefix = 0;
            u64 above = 0;
            for (int shift = 24; shift >= 0; shift -= 8) {
                __syncthreads();
                if (tid < 256) bins[tid] = 0;
                __syncthreads();
                for (int i = tid; i < V; i += kDrawThreads) {
                    const unsigned k = key(i);
                    if (shift < 24 && (k >> (shift + 8)) != (prefix >> (shift + 8))) continue;
                    const u64 m = measure(k);
                    if (m) atomicAdd(&bins[(k >> shift) & 255], m);
                }
                __syncthreads();
                if (tid == 0) {
                    u64 s = above;
                    int b = 255;
                    for (; b > 0; b--) { if (s + bins[b] >= want) break; s += bins[b]; }
                    sh_digit = (unsigned)b; sh_above = s;
                }
                __syncthreads();
                prefix |= sh_digit << shift;
                above = sh_above;
            }
            k_out = prefix; above_out = above;
        };
        auto kept_mass = [&]() {                              // mass of what the cut keeps
            u64 s = 0;
            for (int i = tid; i < V; i += kDrawThreads) { const unsigned k = key(i); if (k > cut_key) s += mass_of(weight(k)); }
            return draw_block_sum(s, sh) + ties * mass_of(weight(cut_key));
        };
        const int top_k = a.top_k ? a.top_k[row] : 0;
        if (top_k > 0 && top_k < V) {
            u64 n = 0;
            for (int i = tid; i < V; i += kDrawThreads) n += key(i) > kKeyNone;
            n = draw_block_sum(n, sh);
            if ((u64)top_k < n) {
                u64 above;
                select((u64)top_k, [&](unsigned k) { return (u64)(k > kKeyNone); }, cut_key, above);
                ties = (u64)top_k - above;
            }
        }
        const float top_p = a.top_p ? a.top_p[row] : 1.0f;
        if (top_p < 1.0f) {
            // rank j is kept while the mass before it is < top_p * mass of the first k, that is < want
            const u64 zk = ties ? kept_mass() : z;
            const double lim = (double)top_p * (double)zk;
            const u64 want = lim > 1.0 ? (u64)ceil(lim) : 1;  // the first is always kept
            unsigned k2;
            u64 above;
            const unsigned ck = cut_key;
            const u64 ct = ties, wt = mass_of(weight(ck));
            select(want, [&](unsigned k) { return k > ck ? mass_of(weight(k)) : 0; }, k2, above);
            if (k2 <= ck) { k2 = ck; above = zk - ct * wt; }  // the border lies among the entries of top-k's own cut
            const u64 w2 = mass_of(weight(k2));
            if (above < want && w2) {
                u64 t2 = (want - above + w2 - 1) / w2;
                if (k2 == ck && t2 > ct) t2 = ct;
                cut_key = k2; ties = t2;
            }
        }
        const float min_p = a.min_p ? a.min_p[row] : 0.0f;
        const bool use_m = min_p > 0.0f;
        const double m64 = (double)min_p;
        auto keeps = [&](unsigned k) { return !use_m || weight(k) >= m64; };
        // the draw, in the vocabulary's order: every wave owns a run of it
        const int per = ((V + kDrawWaves - 1) / kDrawWaves + 63) & ~63, i0 = min(V, wave * per), i1 = min(V, i0 + per);
        const u64 cut_w = keeps(cut_key) ? mass_of(weight(cut_key)) : 0;
        __shared__ u64 seg_mass[kDrawWaves], seg_ties[kDrawWaves];
        u64 s = 0, t = 0;
        for (int i = i0 + lane; i < i1; i += 64) {
            const unsigned k = key(i);
            if (k > cut_key && keeps(k)) s += mass_of(weight(k));
            t += k == cut_key;
        }
        s = wave_sum64(s); t = wave_sum64(t);
        if (lane == 0) { seg_mass[wave] = s; seg_ties[wave] = t; }
        if (tid == 0) sh_tok = best;
        __syncthreads();
        u64 total = 0, before = 0, tb = 0, tie_run = 0;
        for (int w = 0; w < kDrawWaves; w++) {
            if (w == wave) { before = total; tb = tie_run; }
            const u64 left = ties > tie_run ? ties - tie_run : 0, take = seg_ties[w] < left ? seg_ties[w] : left;
            total += seg_mass[w] + take * cut_w;
            tie_run += seg_ties[w];
        }
        double u = (double)a.uniform[row];
        if (!(u > 0.0)) u = 0.0;
        if (u == 0.0) {                                       // the first kept entry of any weight, below the masses' resolution too
            if (tid == 0) sh_idx = 0xffffffffu;
            __syncthreads();
            for (int i = tid; i < V; i += kDrawThreads) {
                const unsigned k = key(i);
                if ((k > cut_key || (k == cut_key && ties)) && keeps(k) && weight(k) > 0.0) { atomicMin(&sh_idx, (unsigned)i); break; }
            }
            __syncthreads();
            if (tid == 0) sh_tok = sh_idx == 0xffffffffu ? best : (int)sh_idx;
            total = 0;                                        // nothing left to look for
        }
        u64 target = (u64)(fmin(u, 1.0 - 0x1p-24) * (double)total);          // below total: total >= 2^45
        const u64 left = ties > tb ? ties - tb : 0, mine = s + (t < left ? t : left) * cut_w;
        if (total > 0 && before <= target && target < before + mine) {       // this wave holds the token
            u64 run = before, trun = tb;
            for (int base = i0; base < i1; base += 64) {
                const int i = base + lane;
                const unsigned k = i < i1 ? key(i) : 0;
                const bool tie = k == cut_key && i < i1;
                const u64 tmask = __ballot(tie);
                const u64 rank = trun + __popcll(tmask & ((1ull << lane) - 1));
                u64 m = 0;
                if (k > cut_key && keeps(k)) m = mass_of(weight(k));
                else if (tie && rank < ties) m = cut_w;
                u64 c = m;
                for (int o = 1; o < 64; o <<= 1) { const u64 y = __shfl_up(c, o); if (lane >= o) c += y; }
                const u64 hit = __ballot(run + c > target);
                if (hit) { if (lane == 0) sh_tok = base + __builtin_ctzll(hit); break; }
                run += __shfl(c, 63);
                trun += __popcll(tmask);
            }
        }
        __syncthreads();
        token = sh_tok;
    }
    if (tid == 0) {
        a.token[row] = token;
        if (a.logprob) {
            const unsigned k = key(token);
            a.logprob[row] = (float)((k == top ? 0.0 : ((double)draw_val(k) - topv) / T64) - log((double)z * (1.0 / kMassOne)));
        }
    }
}

bool draw_tokens(const DrawArgs &a, hipStream_t st) {
    if (a.n_rows <= 0) return true;
    if (a.dtype == WMI_F32) hipLaunchKernelGGL(draw_kernel<float>, dim3(a.n_rows), dim3(kDrawThreads), 0, st, a);
    else if (a.dtype == WMI_F16) hipLaunchKernelGGL(draw_kernel<f16>, dim3(a.n_rows), dim3(kDrawThreads), 0, st, a);
    else hipLaunchKernelGGL(draw_kernel<__bf16>, dim3(a.n_rows), dim3(kDrawThreads), 0, st, a);
    return hipGetLastError() == hipSuccess;
}

}  // namespace wmi

using namespace wmi;

extern "C" {

WHISPER_API int wmi_sample_tokens(const void *logits, int dtype, long long row_stride, int n_rows, int n_vocab, const float *uniform, const float *temperature,
                                  const int *top_k, const float *top_p, const float *min_p, int *token, float *logprob, void *stream) {
    if (n_rows < 0 || n_vocab < 1 || row_stride < 0 || (dtype != WMI_F16 && dtype != WMI_BF16 && dtype != WMI_F32)) return -1;
    if (n_vocab > kDrawMaxVocab) return -3;
    if (n_rows == 0) return 0;
    if (!logits || !uniform || !token || ((uintptr_t)logits & (dtype == WMI_F32 ? 3 : 1))) return -1;
    hipStream_t st = (hipStream_t)stream;
    const ServeCall call(st);
    if (!call.ok()) return -4;
    if (!call.own(logits, (const void *)uniform, (const void *)token) || (temperature && !call.owns(temperature)) || (top_k && !call.owns(top_k)) ||
        (top_p && !call.owns(top_p)) || (min_p && !call.owns(min_p)) || (logprob && !call.owns(logprob))) return -1;
    const DrawArgs a{logits, temperature, top_p, min_p, uniform, top_k, token, logprob, (long)row_stride, n_rows, n_vocab, dtype};
    return draw_tokens(a, st) ? 0 : -4;
}

}  // extern "C"
