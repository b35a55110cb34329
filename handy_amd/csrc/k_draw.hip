// One token a row from its logits, for gfx950: temperature, top-k, top-p, min-p, and a draw from a given uniform number.
#include "kernels.h"
#include "serving_host.h"

namespace wmi {

// Weights w_i = exp((x_i - max x) / T) lie in [0, 1]. They are computed in 64 bits and rounded to whole numbers of 2^-45: sums of up to
// 2^18 of them fit 64 bits and are exact, so they do not depend on the order in which they are made (nor on which workgroup shape
// made them), and every comparison of running masses (top-p's border, the draw) is exact. A weight's rounding costs 2^-46 of the
// largest one: a draw nearer than that to a border may fall on its other side.
// The filters keep a prefix of the order (x descending, index ascending). It is described by a value, the cut: entries above it are
// kept, and of the entries equal to it the first few by index.
//   1. the row's largest and lowest finite value
//   2. all weights: the whole mass (for the log-probability) and, with top-k or top-p, counts and masses in kDrawBins bins of equal
//      width from the largest value down
//   3. the cut lies in the first bin whose running count (mass) reaches what is asked for: its members, mostly a few dozen, are
//      collected and ranked; crowded bins are resolved by radix selection instead
//   4. the kept mass of every wave's run of the vocabulary, then of the run that holds the draw, a few entries a thread
// One workgroup a row. Every pass reads the row again: it comes from HBM once and from the caches afterwards.
constexpr double kMassOne = 35184372088832.0;               // 2^45
constexpr int kDrawBins = 2048, kDrawList = 128, kDrawSmall = 16384;

typedef unsigned long long u64;

__device__ __forceinline__ u64 wave_sum64(u64 v) { for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o); return v; }
__device__ __forceinline__ u64 wave_scan64(u64 v, int lane) { for (int o = 1; o < 64; o <<= 1) { const u64 y = __shfl_up(v, o); if (lane >= o) v += y; } return v; }

// unsigned order of floats (no NaN, no -0): key(a) < key(b) <=> a < b
__device__ __forceinline__ unsigned draw_key(float x) { const unsigned u = __float_as_uint(x); return u & 0x80000000u ? ~u : u | 0x80000000u; }
__device__ __forceinline__ float draw_val(unsigned k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }

// weights relative to a row's largest value `top`
struct DrawScale {
    double top, s;                                           // s = log2(e) / T
    // 2^((x - top) s), rounded to a multiple of 2^-45: 2^f on [-1/2, 1/2] by a polynomial (Chebyshev interpolation, 2^-51 relative),
    // the exponent by ldexp; adding 128 leaves 45 bits behind the point
    __device__ __forceinline__ double weight(float x) const {
        const double y = fmax(((double)x - top) * s, -1000.0), t = y + 6755399441055744.0, f = y - (t - 6755399441055744.0);
        double p = 0x1.e6064532b85cep-28;
        p = __builtin_fma(p, f, 0x1.b675bd731322bp-24);
        p = __builtin_fma(p, f, 0x1.62bfd472702f4p-20);
        p = __builtin_fma(p, f, 0x1.ffcb5405401d9p-17);
        p = __builtin_fma(p, f, 0x1.4309130972597p-13);
        p = __builtin_fma(p, f, 0x1.5d87fe9d7ab38p-10);
        p = __builtin_fma(p, f, 0x1.3b2ab6fba1dcfp-7);
        p = __builtin_fma(p, f, 0x1.c6b08d703ce45p-5);
        p = __builtin_fma(p, f, 0x1.ebfbdff82c598p-3);
        p = __builtin_fma(p, f, 0x1.62e42fefa3a19p-1);
        p = __builtin_fma(p, f, 1.0);
        return (__builtin_amdgcn_ldexp(p, (int)__double2loint(t)) + 128.0) - 128.0;
    }
    __device__ __forceinline__ u64 mass(float x) const { return (u64)(weight(x) * kMassOne); }
};

template <class T> struct DrawIn;                            // four consecutive logits at any alignment
template <> struct DrawIn<float> { typedef float V __attribute__((ext_vector_type(4), aligned(4))); };
template <> struct DrawIn<f16> { typedef f16 V __attribute__((ext_vector_type(4), aligned(2))); };
template <> struct DrawIn<__bf16> { typedef __bf16 V __attribute__((ext_vector_type(4), aligned(2))); };

template <int TH> struct DrawShared {
    static constexpr int W = TH / 64;
    u64 mass[kDrawBins];                                     // per bin, then running from the largest value down
    unsigned count[kDrawBins];
    u64 list_mass[kDrawList];
    float list[kDrawList];
    u64 radix[256];
    u64 seg_mass[W], wm[W];
    unsigned seg_ties[W], wc[W];
    float hi[W], lo[W];
    u64 above;
    float cut;
    unsigned n_list, kmin, kmax, digit, tok;
    int bin;
};

template <class T, int TH>
__global__ __launch_bounds__(TH) void draw_kernel(DrawArgs a) {
    typedef typename DrawIn<T>::V V4;
    constexpr int W = TH / 64, U = 4;
    __shared__ DrawShared<TH> sh;
    const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), V = a.n_vocab;
    const T *src = (const T *)a.logits + row * a.row_stride;
    const int run = ((V + W - 1) / W + 255) & ~255;          // entries of a wave
    const int base = min(V, wave * run), lim = min(V, base + run);
    auto clean = [](float v) { return fmaxf(v + 0.0f, -INFINITY); };               // -0 -> +0, NaN -> -infinity
    // one pass over the row: body(x, i) for every entry of this wave; past the end it sees -infinity (the wave stays whole)
    auto pass = [&](auto body) __attribute__((always_inline)) {
        for (int b = base; b < lim; b += 256 * U) {
            float x[4 * U];
#pragma unroll
            for (int j = 0; j < U; j++) {
                const int i = b + 256 * j + lane * 4;
                if (i + 4 <= lim) {
                    const V4 v = *(const V4 *)(src + i);
#pragma unroll
                    for (int c = 0; c < 4; c++) x[4 * j + c] = (float)v[c];
                } else {
#pragma unroll
                    for (int c = 0; c < 4; c++) x[4 * j + c] = i + c < lim ? (float)src[i + c] : -INFINITY;
                }
            }
#pragma unroll
            for (int j = 0; j < U; j++) {
                if (b + 256 * j >= lim) break;               // uniform
#pragma unroll
                for (int c = 0; c < 4; c++) body(clean(x[4 * j + c]), b + 256 * j + lane * 4 + c);
            }
        }
    };

    // 1. largest and lowest finite value
    float top = -INFINITY, low = INFINITY;
    pass([&](float x, int) { top = fmaxf(top, x); low = fminf(low, x == -INFINITY ? INFINITY : x); });
    for (int o = 32; o > 0; o >>= 1) { top = fmaxf(top, __shfl_xor(top, o)); low = fminf(low, __shfl_xor(low, o)); }
    if (lane == 0) { sh.hi[wave] = top; sh.lo[wave] = low; }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < W; w++) { top = fmaxf(top, sh.hi[w]); low = fminf(low, sh.lo[w]); }
    if (top == -INFINITY) {                                  // nothing can be drawn
        if (tid == 0) { a.token[row] = -1; if (a.logprob) a.logprob[row] = -INFINITY; }
        return;
    }
    const float t_in = a.temperature ? a.temperature[row] : 1.0f;
    const bool drawn = t_in > 0.0f;
    const double T64 = drawn ? (double)t_in : 1.0;
    const DrawScale sc{(double)top, 1.4426950408889634 / T64};
    const int top_k = drawn && a.top_k ? a.top_k[row] : 0;
    const float top_p = drawn && a.top_p ? a.top_p[row] : 1.0f, min_p = drawn && a.min_p ? a.min_p[row] : 0.0f;
    const bool use_k = top_k > 0 && top_k < V, use_p = top_p < 1.0f, use_m = min_p > 0.0f;

    const u64 top_m = (u64)kMassOne;
    auto mass_of = [&](float x) { return x == top ? top_m : sc.mass(x); };           // (an infinite largest value has no difference to itself)
    float cut = -INFINITY;
    unsigned ties = 0;
    u64 z;

    // 2. masses, and the histogram. Bins of equal width from the largest value down, in halves so that no difference overflows; with
    // top-p alone they need not reach below the values whose mass is 0.
    float floor_v = low;
    if (use_p && !use_k) floor_v = fmaxf(low, (float)((double)top - 32.0 * T64));
    const float half_top = 0.5f * top, width = half_top - 0.5f * floor_v, per_bin = width > 0.0f ? (float)kDrawBins / width : 0.0f;
    auto bin_of = [&](float v) { return (int)fminf((half_top - 0.5f * v) * per_bin, (float)(kDrawBins - 1)); };
    auto block_sum = [&](u64 s) -> u64 {
        s = wave_sum64(s);
        __syncthreads();
        if (lane == 0) sh.wm[wave] = s;
        __syncthreads();
        u64 t = 0;
#pragma unroll
        for (int w = 0; w < W; w++) t += sh.wm[w];
        return t;
    };
    // the value at which the running count (by_mass: mass) from the largest value down reaches want > 0, and the sum over larger values
    auto select = [&](u64 want, bool by_mass, float &v_out, u64 &above_out) __attribute__((always_inline)) {
        auto running = [&](int b) -> u64 { return b < 0 ? 0 : by_mass ? sh.mass[b] : (u64)sh.count[b]; };
        if (tid == 0) { sh.n_list = 0; sh.kmin = 0xffffffffu; sh.kmax = 0; }
        for (int i = tid; i < kDrawBins; i += TH) if (running(i) >= want && running(i - 1) < want) sh.bin = i;
        __syncthreads();
        const int bin = sh.bin;
        const u64 above = running(bin - 1);
        pass([&](float x, int) {
            if (x != -INFINITY && bin_of(x) == bin) {
                const unsigned at = atomicAdd(&sh.n_list, 1u), key = draw_key(x);
                atomicMin(&sh.kmin, key); atomicMax(&sh.kmax, key);
                if (at < (unsigned)kDrawList) { sh.list[at] = x; sh.list_mass[at] = by_mass ? mass_of(x) : 1; }
            }
        });
        __syncthreads();
        const int n = (int)sh.n_list;
        if (sh.kmin == sh.kmax) { v_out = draw_val(sh.kmin); above_out = above; }
        else if (n <= kDrawList) {                           // every member looks at every other
            if (tid < n) {
                const float v = sh.list[tid];
                u64 gt = above, eq = 0;
                for (int j = 0; j < n; j++) { const float o = sh.list[j]; const u64 m = sh.list_mass[j]; if (o > v) gt += m; else if (o == v) eq += m; }
                if (gt < want && gt + eq >= want) { sh.cut = v; sh.above = gt; }          // the members of one value agree
            }
            __syncthreads();
            v_out = sh.cut; above_out = sh.above;
        } else {                                             // radix selection among the members, 8 bits of the key at a time
            unsigned prefix = 0;
            u64 sum = above;
            for (int shift = 24; shift >= 0; shift -= 8) {
                for (int i = tid; i < 256; i += TH) sh.radix[i] = 0;
                __syncthreads();
                pass([&](float x, int) {
                    const unsigned key = draw_key(x);
                    if (x != -INFINITY && bin_of(x) == bin && (shift == 24 || (key >> (shift + 8)) == (prefix >> (shift + 8)))) {
                        const u64 m = by_mass ? mass_of(x) : 1;
                        if (m) atomicAdd(&sh.radix[(key >> shift) & 255], m);
                    }
                });
                __syncthreads();
                if (wave == 0) {                             // lane l: digits 255 - 4 l and the three below
                    u64 d[4], t = 0;
#pragma unroll
                    for (int i = 0; i < 4; i++) { d[i] = sh.radix[255 - 4 * lane - i]; t += d[i]; }
                    u64 r = sum + wave_scan64(t, lane) - t;
#pragma unroll
                    for (int i = 0; i < 4; i++) { if (r < want && r + d[i] >= want) { sh.digit = 255 - 4 * lane - i; sh.above = r; } r += d[i]; }
                }
                __syncthreads();
                prefix |= sh.digit << shift;
                sum = sh.above;
            }
            v_out = draw_val(prefix); above_out = sum;
        }
        __syncthreads();
    };

    if (top == INFINITY) {                                   // infinite entries share everything: the cut is among them
        u64 n = 0;
        pass([&](float x, int) { n += x == INFINITY; });
        n = block_sum(n);
        z = n * top_m;
        cut = top;
        ties = drawn ? (unsigned)n : 1;
        if (use_k && ties > (unsigned)top_k) ties = (unsigned)top_k;
        if (use_p) { const double l = ceil((double)top_p * (double)ties); ties = l > 1.0 ? (unsigned)l : 1; }
        if (use_m && min_p > 1.0f) ties = 1;
    } else {
        const bool hist = use_k || use_p;
        if (hist) {
            for (int i = tid; i < kDrawBins; i += TH) { sh.count[i] = 0; sh.mass[i] = 0; }
            __syncthreads();
        }
        double acc = 0.0;                                    // at most 256 multiples of 2^-45 up to 1: exact
        pass([&](float x, int) {
            const double w = sc.weight(x);
            acc += w;
            if (hist && x != -INFINITY) {
                const int b = bin_of(x);
                if (use_k) atomicAdd(&sh.count[b], 1u);
                if (use_p && w > 0.0) atomicAdd(&sh.mass[b], (u64)(w * kMassOne));
            }
        });
        const u64 own = wave_sum64((u64)(acc * kMassOne));
        if (lane == 0) { sh.seg_mass[wave] = own; sh.seg_ties[wave] = 0; }
        __syncthreads();
        z = 0;
#pragma unroll
        for (int w = 0; w < W; w++) z += sh.seg_mass[w];

        // 3. the cut
        if (hist) {                                          // running sums over the bins, in place
            constexpr int B = kDrawBins / TH;
            u64 m = 0;
            unsigned c = 0;
#pragma unroll
            for (int i = 0; i < B; i++) { m += sh.mass[tid * B + i]; c += sh.count[tid * B + i]; }
            u64 xm = wave_scan64(m, lane);
            unsigned xc = c;
            for (int o = 1; o < 64; o <<= 1) { const unsigned y = __shfl_up(xc, o); if (lane >= o) xc += y; }
            if (lane == 63) { sh.wm[wave] = xm; sh.wc[wave] = xc; }
            __syncthreads();
            xm -= m; xc -= c;
            for (int w = 0; w < wave; w++) { xm += sh.wm[w]; xc += sh.wc[w]; }
#pragma unroll
            for (int i = 0; i < B; i++) { xm += sh.mass[tid * B + i]; sh.mass[tid * B + i] = xm; xc += sh.count[tid * B + i]; sh.count[tid * B + i] = xc; }
            __syncthreads();
        }
        if (!drawn) { cut = top; ties = 1; }
#pragma clang loop unroll(disable)
        for (int by_mass = 0; by_mass < 2; by_mass++) {      // top-k by counts, then top-p by masses
            u64 want;
            if (!by_mass) {
                if (!use_k || (unsigned)top_k >= sh.count[kDrawBins - 1]) continue;
                want = (u64)top_k;
            } else {
                // rank j is kept while the mass before it is < top_p * mass of the first k, that is < want; the first always is
                if (!use_p) break;
                u64 zk = z;
                if (ties) {
                    u64 s = 0;
                    pass([&](float x, int) { if (__any(x > cut)) s += x > cut ? mass_of(x) : 0; });
                    zk = block_sum(s) + ties * mass_of(cut);
                }
                const double limit = ceil((double)top_p * (double)zk);
                want = limit > 1.0 ? (u64)limit : 1;
            }
            float v;
            u64 above;
            select(want, by_mass != 0, v, above);
            if (!by_mass) { cut = v; ties = (unsigned)(want - above); }
            else if (ties == 0 || v >= cut) {
                const u64 w = mass_of(v), t = (want - above + w - 1) / w;
                ties = v == cut && t > ties ? ties : (unsigned)t;
                cut = v;
            }
        }
        if (use_m) {
            // the lowest value whose weight is at least min_p, by a 64-way search over the keys up to the largest value's
            unsigned lo = draw_key(-INFINITY) + 1, n = draw_key(top) - lo + 1;            // the first of [lo, lo + n] that is (lo + n: above the largest)
            const double m64 = (double)min_p;
            while (n > 0) {
                const unsigned step = n / 64 + 1, at = lane * step;
                const bool light = at < n && !(exp(((double)draw_val(lo + at) - (double)top) / T64) >= m64);       // the answer lies behind
                const unsigned k = __popcll(__ballot(light));
                if (k == 0) break;
                lo += (k - 1) * step + 1;
                n = min(step - 1, n - ((k - 1) * step + 1));
            }
            const float v = draw_val(lo);                    // kept: x >= v
            if (v > top) { cut = top; ties = 1; }            // (the first always is)
            else if (v > cut) { cut = draw_val(lo - 1); ties = 0; }
        }
    }

    // 4. the draw, in the vocabulary's order
    const u64 cut_m = ties ? mass_of(cut) : 0;
    const double u = fmin(a.uniform[row] > 0.0f ? (double)a.uniform[row] : 0.0, 1.0 - 0x1p-24);
    if (u == 0.0) {                                          // the first kept entry of any weight, below the masses' resolution too
        if (tid == 0) sh.tok = 0xffffffffu;
        __syncthreads();
        unsigned first = 0xffffffffu;
        pass([&](float x, int i) {
            if ((x > cut || (ties && x == cut)) && (x == top || ((double)x - (double)top) / T64 > -745.13)) first = min(first, (unsigned)i);
        });
        if (first != 0xffffffffu) atomicMin(&sh.tok, first);
    } else {
        if (cut > -INFINITY) {                               // masses above the cut and entries equal to it, by wave
            u64 s = 0;
            unsigned t = 0;
            pass([&](float x, int) {
                if (__any(x > cut)) s += x > cut ? mass_of(x) : 0;
                t += x == cut;
            });
            s = wave_sum64(s);
            for (int o = 32; o > 0; o >>= 1) t += __shfl_xor(t, o);
            __syncthreads();
            if (lane == 0) { sh.seg_mass[wave] = s; sh.seg_ties[wave] = t; }
        }
        __syncthreads();
        // lane s: the run of wave s
        const unsigned st = lane < W ? sh.seg_ties[lane] : 0;
        unsigned tx = st;
        for (int o = 1; o < 64; o <<= 1) { const unsigned y = __shfl_up(tx, o); if (lane >= o) tx += y; }
        tx -= st;
        const unsigned left = ties > tx ? ties - tx : 0;
        const u64 sm = lane < W ? sh.seg_mass[lane] + (u64)min(st, left) * cut_m : 0, sums = wave_scan64(sm, lane), total = __shfl(sums, 63);
        const u64 target = (u64)(u * (double)total);         // < total: total >= 2^45
        const int pick = __builtin_ctzll(__ballot(sums > target));
        const u64 before = __shfl(sums - sm, pick);
        const unsigned tie_before = __shfl(tx, pick);
        const int b = min(V, pick * run), e = min(V, b + run);
        // that run of the vocabulary, each thread E entries in a row
        const int E = ((e - b) + TH - 1) / TH, i0 = min(e, b + tid * E), i1 = min(e, i0 + E);
        unsigned t = 0;
        if (ties) for (int i = i0; i < i1; i++) t += clean((float)src[i]) == cut;
        unsigned ts = t;
        for (int o = 1; o < 64; o <<= 1) { const unsigned y = __shfl_up(ts, o); if (lane >= o) ts += y; }
        if (lane == 63) sh.wc[wave] = ts;
        __syncthreads();
        ts += tie_before - t;
        for (int w = 0; w < wave; w++) ts += sh.wc[w];
        auto mass_at = [&](int i, unsigned &rank) -> u64 {
            const float v = clean((float)src[i]);
            if (v > cut) return mass_of(v);
            return v == cut && rank++ < ties ? cut_m : 0;
        };
        u64 m = 0;
        unsigned rank = ts;
        for (int i = i0; i < i1; i++) m += mass_at(i, rank);
        u64 ms = wave_scan64(m, lane);
        if (lane == 63) sh.wm[wave] = ms;
        __syncthreads();
        ms += before - m;
        for (int w = 0; w < wave; w++) ms += sh.wm[w];
        if (ms <= target && target < ms + m) {               // one thread
            rank = ts;
            u64 c = ms;
            int i = i0;
            for (; i < i1 - 1; i++) { c += mass_at(i, rank); if (c > target) break; }
            sh.tok = (unsigned)i;
        }
    }
    __syncthreads();
    if (tid == 0) {
        const int token = (int)sh.tok;
        a.token[row] = token;
        if (a.logprob) {
            const float v = clean((float)src[token]);
            a.logprob[row] = (float)((v == top ? 0.0 : ((double)v - (double)top) / T64) - log((double)z * (1.0 / kMassOne)));
        }
    }
}

template <class T> static void draw_launch(const DrawArgs &a, hipStream_t st) {
    // short rows: four waves a row, so that several rows share a compute unit
    if (a.n_vocab <= kDrawSmall) hipLaunchKernelGGL((draw_kernel<T, 256>), dim3(a.n_rows), dim3(256), 0, st, a);
    else hipLaunchKernelGGL((draw_kernel<T, 1024>), dim3(a.n_rows), dim3(1024), 0, st, a);
}

bool draw_tokens(const DrawArgs &a, hipStream_t st) {
    if (a.n_rows <= 0) return true;
    if (a.dtype == WMI_F32) draw_launch<float>(a, st);
    else if (a.dtype == WMI_F16) draw_launch<f16>(a, st);
    else draw_launch<__bf16>(a, st);
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
