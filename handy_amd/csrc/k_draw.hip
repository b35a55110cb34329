// One token a row from its logits, for gfx950: temperature, top-k, top-p, min-p, and a draw from a given uniform number.
#include "kernels.h"
#include "serving_host.h"
#include <type_traits>

namespace wmi {

// Weights w_i = exp((x_i - max x) / T) lie in [0, 1]. They are computed in 64 bits and rounded to whole numbers of 2^-45: sums of up to
// 2^18 of them fit 64 bits and are exact, so they do not depend on the order in which they are made (nor on which workgroup shape
// made them), and neither do the comparisons of running masses (top-p's border, the draw). Rounded are a weight, by 2^-46 of the largest
// one, and the two products that masses are compared with, top_p and the uniform number times a mass, by 2^-52 of themselves: a draw nearer
// than that to a border may fall on its other side.
// The filters keep a prefix of the order (x descending, index ascending). It is described by a value, the cut: entries above it are
// kept, and of the entries equal to it the first few by index.
// One workgroup a row; the row comes from HBM once and out of the caches in later passes:
//   1. the largest value
//   2. the whole mass (for the log-probability; without a filter also what the draw needs, by wave)
//   3. the cut. A short top-k or a min_p: the k-th largest of the threads' own maxima (at least k entries reach it) or the border
//      weight bounds it from below; the entries that reach the bound are listed in the LDS, and the rest of the work runs over the list. Other
//      filters (and lists that overflow): pass 2 also adds counts and masses up in kDrawBins bins of equal width from the largest
//      value down, masses by wave; the cut lies in the first bin whose running sum reaches what is asked for. Either way that bin's
//      members are ranked, or narrowed down by radix first if there are many.
//   4. the draw, in the vocabulary's order: the wave's run that holds it, the thread's few entries, the entry.
// Bound by 64-bit arithmetic (pass 2: 19 such instructions a weight, about 7 of its 11 us for 51866 entries on one compute unit) and by
// the waits of the short steps, which a second row on the same compute unit covers. Five rows of 51866 32-bit logits at a temperature:
// 25 us; 1024 rows with every filter in use: 150 us (1.4 TB/s of logits); 48 rows of 131071 bf16: 95 us.
constexpr double kMassOne = 35184372088832.0;               // 2^45
constexpr float kListMinP = 1.0f / 1024;                    // a min_p from here on is taken to leave few entries
constexpr int kDrawBins = 768, kDrawRank = 1024, kDrawClose = 128, kDrawCap = 1024;

typedef unsigned long long u64;

__device__ __forceinline__ u64 wave_sum64(u64 v) { for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o); return v; }
__device__ __forceinline__ u64 wave_scan64(u64 v, int lane) { for (int o = 1; o < 64; o <<= 1) { const u64 y = __shfl_up(v, o); if (lane >= o) v += y; } return v; }
__device__ __forceinline__ unsigned wave_scan32(unsigned v, int lane) { for (int o = 1; o < 64; o <<= 1) { const unsigned y = __shfl_up(v, o); if (lane >= o) v += y; } return v; }

// unsigned order of floats (no NaN, no -0): key(a) < key(b) <=> a < b
__device__ __forceinline__ unsigned draw_key(float x) { const unsigned u = __float_as_uint(x); return u & 0x80000000u ? ~u : u | 0x80000000u; }
__device__ __forceinline__ float draw_val(unsigned k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }

// weights relative to a row's largest value `top`
struct DrawScale {
    double top, s;                                           // s = log2(e) / T
    // 2^((x - top) s): 2^f on [-1/2, 1/2] by a polynomial (Chebyshev interpolation, 2^-51 relative), its exponent moved by the whole
    // part (never below 2^-1001)
    __device__ __forceinline__ double exact(float x) const {
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
        return __hiloint2double(__double2hiint(p) + (__double2loint(t) << 20), __double2loint(p));
    }
    // rounded to a multiple of 2^-45: 128 plus the weight keeps 45 bits behind the point, and is that whole number but for its exponent
    __device__ __forceinline__ u64 mass(float x) const { return (u64)__double_as_longlong(exact(x) + 128.0) - 0x4060000000000000ull; }
};

template <class T> struct DrawIn;                            // four consecutive logits at any alignment
template <> struct DrawIn<float> { typedef float V __attribute__((ext_vector_type(4), aligned(4))); };
template <> struct DrawIn<f16> { typedef f16 V __attribute__((ext_vector_type(4), aligned(2))); };
template <> struct DrawIn<__bf16> { typedef __bf16 V __attribute__((ext_vector_type(4), aligned(2))); };

template <int TH> struct DrawShared {
    static constexpr int W = TH / 64;
    union {
        u64 hist[W][kDrawBins];                              // masses by wave and bin
        struct {
            float list[W][kDrawCap];                         // entries that can be kept, by wave and in order ...
            unsigned short list_at[W][kDrawCap];             // ... and where in the wave's run (at most 16384 entries) they stand
        };
    };
    u64 mass[kDrawBins];                                     // running from the largest value down
    unsigned count[kDrawBins];
    u64 rank_mass[kDrawRank], radix[256], seg_mass[W], wm[W], above;
    float rank[kDrawRank], hi[W], lo[W], cut;
    unsigned seg_ties[W], wc[W], n_listed[W], n_member[W];
    unsigned n_rank, kmin, kmax, digit, tok, walk_rank;
    unsigned n_close;
    int bin, walk_at;
    unsigned short close[kDrawClose];
    unsigned char rank_wave[kDrawRank];
};

template <class T, int TH>
__global__ __launch_bounds__(TH, 4) void draw_kernel(DrawArgs a) {
    typedef typename DrawIn<T>::V V4;
    constexpr int W = TH / 64, U = 4, LOW = sizeof(T) == 4 ? 0 : std::is_same<T, f16>::value ? 13 : 16;      // low bits that a float made from T does not use
    __shared__ DrawShared<TH> sh;
    const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), V = a.n_vocab;
    const T *src = (const T *)a.logits + (a.row_of ? a.row_of[row] : row) * a.row_stride;
    const float t_in = a.temperature ? a.temperature[row] : 1.0f, p_in = a.top_p ? a.top_p[row] : 1.0f, m_in = a.min_p ? a.min_p[row] : 0.0f, u_in = a.uniform[row];
    const int k_in = a.top_k ? a.top_k[row] : 0;
    const int run = ((V + W - 1) / W + 255) & ~255;          // entries of a wave
    const int base = min(V, wave * run), lim = min(V, base + run);
    auto clean = [](float v) { return fmaxf(v + 0.0f, -INFINITY); };               // -0 -> +0, NaN -> -infinity
    // one pass over the row, four entries a lane at a time: body(x[4], i) for entries i .. i + 3 (-infinity past the wave's end; the
    // wave stays whole)
    auto stream4 = [&](auto body) __attribute__((always_inline)) {
        for (int b = base; b < lim; b += 256 * U) {
            float y[4 * U];
#pragma unroll
            for (int j = 0; j < U; j++) {
                const int i = b + 256 * j + lane * 4;
                if (i + 4 <= lim) {
                    const V4 v = *(const V4 *)(src + i);
#pragma unroll
                    for (int c = 0; c < 4; c++) y[4 * j + c] = (float)v[c];
                } else {
#pragma unroll
                    for (int c = 0; c < 4; c++) y[4 * j + c] = i + c < lim ? (float)src[i + c] : -INFINITY;
                }
            }
#pragma unroll
            for (int j = 0; j < U; j++) {
                if (b + 256 * j >= lim) break;               // uniform
#pragma unroll
                for (int c = 0; c < 4; c++) y[4 * j + c] = clean(y[4 * j + c]);
                body(y + 4 * j, b + 256 * j + lane * 4);
            }
        }
    };
    bool listed = false;
    // one pass over what can be kept: body(x, i) for every entry i of this wave's part of the list, or of the row
    auto pass = [&](auto body) __attribute__((always_inline)) {
        if (listed) {
            const int n = (int)sh.n_listed[wave];
            for (int j0 = 0; j0 < n; j0 += 64) {
                const bool on = j0 + lane < n;
                body(on ? sh.list[wave][j0 + lane] : -INFINITY, on ? base + (int)sh.list_at[wave][j0 + lane] : 0);
            }
        } else stream4([&](const float *v, int i) {
#pragma unroll
            for (int c = 0; c < 4; c++) body(v[c], i + c);
        });
    };
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

    // 1. largest and lowest finite value
    float top = -INFINITY, low = INFINITY;
    stream4([&](const float *v, int) {
#pragma unroll
        for (int c = 0; c < 4; c++) { top = fmaxf(top, v[c]); low = fminf(low, v[c] == -INFINITY ? INFINITY : v[c]); }
    });
    const float own_top = top;
    for (int o = 32; o > 0; o >>= 1) { top = fmaxf(top, __shfl_xor(top, o)); low = fminf(low, __shfl_xor(low, o)); }
    if (lane == 0) { sh.hi[wave] = top; sh.lo[wave] = low; }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < W; w++) { top = fmaxf(top, sh.hi[w]); low = fminf(low, sh.lo[w]); }
    if (top == -INFINITY) {                                  // nothing can be drawn
        if (tid == 0) { a.token[row] = -1; if (a.logprob) a.logprob[row] = -INFINITY; }
        return;
    }
    const bool drawn = t_in > 0.0f;
    const double T64 = drawn ? (double)t_in : 1.0;
    const DrawScale sc{(double)top, 1.4426950408889634 / T64};
    const int top_k = drawn ? k_in : 0;
    const float top_p = drawn ? p_in : 1.0f, min_p = drawn ? m_in : 0.0f;
    const bool use_k = top_k > 0 && top_k < V, use_p = top_p < 1.0f, use_m = min_p > 0.0f;
    const u64 top_m = (u64)kMassOne;
    auto mass_of = [&](float v) { return v == top ? top_m : sc.mass(v); };           // (an infinite largest value has no difference to itself)
    float cut = -INFINITY;
    unsigned ties = 0;
    u64 z = 0;

    // bins of equal width from the largest value down to floor_v, in halves so that no difference overflows
    const float half_top = 0.5f * top;
    float per_bin = 0.0f;
    auto set_bins = [&](float floor_v) { const float width = half_top - 0.5f * floor_v; per_bin = width > 0.0f ? (float)kDrawBins / width : 0.0f; };
    auto bin_of = [&](float v) { return (int)fminf((half_top - 0.5f * v) * per_bin, (float)(kDrawBins - 1)); };
    // running sums over the bins, in place
    auto run_bins = [&]() __attribute__((always_inline)) {
        constexpr int B = (kDrawBins + TH - 1) / TH;
        const int b0 = min(kDrawBins, tid * B), b1 = min(kDrawBins, b0 + B);
        u64 m = 0;
        unsigned c = 0;
        for (int i = b0; i < b1; i++) { m += sh.mass[i]; c += sh.count[i]; }
        u64 xm = wave_scan64(m, lane);
        unsigned xc = wave_scan32(c, lane);
        __syncthreads();
        if (lane == 63) { sh.wm[wave] = xm; sh.wc[wave] = xc; }
        __syncthreads();
        xm -= m; xc -= c;
        for (int w = 0; w < wave; w++) { xm += sh.wm[w]; xc += sh.wc[w]; }
        for (int i = b0; i < b1; i++) { xm += sh.mass[i]; sh.mass[i] = xm; xc += sh.count[i]; sh.count[i] = xc; }
        __syncthreads();
    };
    auto clear_bins = [&]() { for (int i = tid; i < kDrawBins; i += TH) { sh.count[i] = 0; sh.mass[i] = 0; } };
    // the digit (of 256, from the highest down) in which `sum` and the digits' measures reach want, by wave 0
    auto pick_digit = [&](u64 want, u64 sum) {
        if (wave == 0) {                                     // lane l: digits 255 - 4 l and the three below
            u64 d[4], t = 0;
#pragma unroll
            for (int i = 0; i < 4; i++) { d[i] = sh.radix[255 - 4 * lane - i]; t += d[i]; }
            u64 r = sum + wave_scan64(t, lane) - t;
#pragma unroll
            for (int i = 0; i < 4; i++) { if (r < want && r + d[i] >= want) { sh.digit = 255 - 4 * lane - i; sh.above = r; } r += d[i]; }
        }
        __syncthreads();
    };
    // the same as select among n collected members: 256 bins of equal width between the lowest and the highest, then the members of
    // one of them, each against each. False: too many fall into that bin
    auto narrow = [&](u64 want, bool by_mass, int n, u64 above) -> bool {
        const float lo = draw_val(sh.kmin), per = 255.99f / (0.5f * draw_val(sh.kmax) - 0.5f * lo);
        auto digit_of = [&](float v) { return (unsigned)fminf((0.5f * v - 0.5f * lo) * per, 255.0f); };
        for (int i = tid; i < 256; i += TH) sh.radix[i] = 0;
        if (tid == 0) sh.n_close = 0;
        __syncthreads();
        for (int i = tid; i < n; i += TH) { const u64 m = by_mass ? sh.rank_mass[i] : 1; if (m) atomicAdd(&sh.radix[digit_of(sh.rank[i])], m); }
        __syncthreads();
        pick_digit(want, above);
        const unsigned digit = sh.digit;
        const u64 base_sum = sh.above;
        for (int i = tid; i < n; i += TH)
            if (digit_of(sh.rank[i]) == digit) { const unsigned at = atomicAdd(&sh.n_close, 1u); if (at < (unsigned)kDrawClose) sh.close[at] = (unsigned short)i; }
        __syncthreads();
        const int k = (int)sh.n_close;
        if (k > kDrawClose) return false;
        if (tid < k) {
            const float v = sh.rank[sh.close[tid]];
            u64 gt = base_sum, eq = 0;
            for (int j = 0; j < k; j++) { const int at = sh.close[j]; const float o = sh.rank[at]; const u64 m = by_mass ? sh.rank_mass[at] : 1; if (o > v) gt += m; else if (o == v) eq += m; }
            if (gt < want && gt + eq >= want) { sh.cut = v; sh.above = gt; }              // the members of one value agree
        }
        __syncthreads();
        return true;
    };
    // the value at which the running count (by_mass: mass) from the largest value down reaches want > 0, and the sum over larger
    // values. Leaves what it collected of that bin: sh.bin, sh.n_rank, sh.kmin, sh.kmax, sh.n_member, sh.rank*
    auto select = [&](u64 want, bool by_mass, float &v_out, u64 &above_out) __attribute__((always_inline)) {
        auto running = [&](int b) -> u64 { return b < 0 ? 0 : by_mass ? sh.mass[b] : (u64)sh.count[b]; };
        for (int i = tid; i < kDrawBins; i += TH) if (running(i) >= want && running(i - 1) < want) sh.bin = i;
        __syncthreads();
        const int bin = sh.bin;
        u64 above = running(bin - 1);
        unsigned lo = 0, hi = 0xffffffffu;                   // the keys (without their unused bits) the cut's lies among; the bin's own are an interval
        bool whole = true;                                   // that is the bin
        for (;;) {
            if (tid == 0) { sh.n_rank = 0; sh.kmin = 0xffffffffu; sh.kmax = 0; }
            __syncthreads();
            unsigned members = 0, kmin = 0xffffffffu, kmax = 0;
            pass([&](float x, int) {
                const unsigned key = draw_key(x);
                if (x != -INFINITY && (whole ? bin_of(x) == bin : (key >> LOW) - lo <= hi - lo)) {
                    const unsigned at = atomicAdd(&sh.n_rank, 1u);
                    kmin = min(kmin, key); kmax = max(kmax, key);
                    members++;
                    if (at < (unsigned)kDrawRank) { sh.rank[at] = x; sh.rank_wave[at] = (unsigned char)wave; }
                }
            });
            for (int o = 32; o > 0; o >>= 1) { members += __shfl_xor(members, o); kmin = min(kmin, (unsigned)__shfl_xor(kmin, o)); kmax = max(kmax, (unsigned)__shfl_xor(kmax, o)); }
            if (lane == 0 && members) { atomicMin(&sh.kmin, kmin); atomicMax(&sh.kmax, kmax); }
            if (lane == 0) sh.n_member[wave] = members;
            __syncthreads();
            const int n = (int)sh.n_rank;
            if (n <= kDrawRank) {                            // (their masses here, not in the pass, where one member costs its whole wave the arithmetic)
                for (int i = tid; i < n; i += TH) sh.rank_mass[i] = mass_of(sh.rank[i]);
                __syncthreads();
            }
            if (sh.kmin == sh.kmax) { v_out = draw_val(sh.kmin); above_out = above; break; }
            if (n <= kDrawRank && narrow(want, by_mass, n, above)) { v_out = sh.cut; above_out = sh.above; break; }
            // too many: 256 intervals of equal width of their keys; the one the cut is in
            lo = sh.kmin >> LOW; hi = sh.kmax >> LOW;
            const int bits = 32 - __builtin_clz(hi - lo), shift = bits > 8 ? bits - 8 : 0;
            for (int i = tid; i < 256; i += TH) sh.radix[i] = 0;
            __syncthreads();
            pass([&](float x, int) {
                const unsigned d = (draw_key(x) >> LOW) - lo;
                if (x != -INFINITY && d <= hi - lo) {
                    const u64 m = by_mass && shift > 0 ? mass_of(x) : 1;
                    if (m) atomicAdd(&sh.radix[d >> shift], m);
                }
            });
            __syncthreads();
            auto value_of = [&](unsigned key) { return draw_val(key << LOW | (key >> (31 - LOW) ? 0 : (1u << LOW) - 1)); };
            if (by_mass && shift == 0) {                     // every interval is one value: counted
                for (int i = tid; i <= (int)(hi - lo); i += TH) sh.radix[i] *= mass_of(value_of(lo + i));
                __syncthreads();
            }
            pick_digit(want, above);
            above = sh.above;
            lo += sh.digit << shift; hi = min(hi, lo + ((1u << shift) - 1));
            whole = false;
            if (lo == hi) { v_out = value_of(lo); above_out = above; break; }
            __syncthreads();
        }
        __syncthreads();
        if (!whole) { if (tid == 0) sh.bin = -1; __syncthreads(); }      // (what is collected is not the bin's)
    };

    if (top == INFINITY) {                                   // infinite entries share everything: the cut is among them
        unsigned n = 0;
        stream4([&](const float *v, int) {
#pragma unroll
            for (int c = 0; c < 4; c++) n += v[c] == INFINITY;
        });
        const unsigned all = (unsigned)block_sum(n);         // (a wave's sum of lanes, then of waves)
        for (int o = 32; o > 0; o >>= 1) n += __shfl_xor(n, o);
        if (lane == 0) { sh.seg_mass[wave] = 0; sh.seg_ties[wave] = n; }
        z = all * top_m;
        cut = top;
        ties = drawn ? all : 1;
        if (use_k && ties > (unsigned)top_k) ties = (unsigned)top_k;
        if (use_p) { const double l = ceil((double)top_p * (double)ties); ties = l > 1.0 ? (unsigned)l : 1; }
        if (use_m && min_p > 1.0f) ties = 1;
    } else {
        const bool filtered = !drawn || use_k || use_p || use_m;
        // min_p bounds the list unless top-p's masses are those of the first top_k, which may reach behind it
        const bool by_m = use_m && min_p >= kListMinP && !(use_k && use_p);
        bool binned = drawn && !by_m && (use_k ? top_k > TH / 2 : use_p);
#pragma clang loop unroll(disable)
        for (;;) {
            if (binned) {
                // without top-k the bins need not reach below the values whose mass is 0
                set_bins(use_k ? low : fmaxf(low, (float)((double)top - 32.0 * T64)));
                clear_bins();
                for (int i = tid; i < W * kDrawBins; i += TH) (&sh.hist[0][0])[i] = 0;
                __syncthreads();
            }
            // 2. the whole mass
            u64 own = 0;
            if (!binned) stream4([&](const float *v, int) {
#pragma unroll
                for (int c = 0; c < 4; c++) own += sc.mass(v[c]);
            });
            else stream4([&](const float *v, int) {
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    const u64 m = sc.mass(v[c]);
                    const int b = bin_of(v[c]);
                    own += m;
                    if (use_k && v[c] != -INFINITY) atomicAdd(&sh.count[b], 1u);
                    if (m) atomicAdd(&sh.hist[wave][b], m);
                }
            });
            own = wave_sum64(own);
            if (lane == 0) { sh.seg_mass[wave] = own; sh.seg_ties[wave] = 0; }
            __syncthreads();
            z = 0;
#pragma unroll
            for (int w = 0; w < W; w++) z += sh.seg_mass[w];
            if (!filtered || binned) break;

            // 3. the list: entries from the bin on that holds the k-th largest of the threads' maxima -- from the lowest maximum in it
            float least = top;
            if (drawn && (by_m || !use_k)) least = fminf(top, (float)((double)top + T64 * (log(fmin((double)min_p, 1.0)) - 1e-6)));       // (a slack far beyond every rounding here)
            else if (drawn) {
                const unsigned kk = (unsigned)top_k;
                clear_bins();
                set_bins(low);
                const int mine = own_top == -INFINITY ? kDrawBins : bin_of(own_top);
                if (tid == 0) { sh.bin = kDrawBins; sh.kmin = 0xffffffffu; }
                __syncthreads();
                if (mine < kDrawBins) atomicAdd(&sh.count[mine], 1u);
                __syncthreads();
                run_bins();
                for (int i = tid; i < kDrawBins; i += TH) if (sh.count[i] >= kk && (i == 0 || sh.count[i - 1] < kk)) sh.bin = i;
                __syncthreads();
                const int upto = sh.bin;                     // (kDrawBins: fewer than k threads hold anything -- everything is listed)
                if (mine <= upto && mine < kDrawBins) atomicMin(&sh.kmin, draw_key(own_top));
                __syncthreads();
                least = upto < kDrawBins ? draw_val(sh.kmin) : low;
            }
            unsigned n = 0;
            stream4([&](const float *v, int i) {
                u64 has[4];
#pragma unroll
                for (int j = 0; j < 4; j++) has[j] = __ballot(v[j] >= least);
                if ((has[0] | has[1] | has[2] | has[3]) != 0) {          // a lane's four entries come one after the other
                    unsigned at = n;
#pragma unroll
                    for (int j = 0; j < 4; j++) { at += __builtin_amdgcn_mbcnt_hi((unsigned)(has[j] >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)has[j], 0)); n += __popcll(has[j]); }
#pragma unroll
                    for (int j = 0; j < 4; j++)
                        if (v[j] >= least) {
                            if (at < (unsigned)kDrawCap) { sh.list[wave][at] = v[j]; sh.list_at[wave][at] = (unsigned short)(i + j - base); }
                            at++;
                        }
                }
            });
            if (lane == 0) sh.n_listed[wave] = n;
            __syncthreads();
            listed = true;
#pragma unroll
            for (int w = 0; w < W; w++) listed &= sh.n_listed[w] <= (unsigned)kDrawCap;
            if (listed) {
                if (use_k || use_p) {
                    set_bins(least);
                    clear_bins();
                    __syncthreads();
                    pass([&](float v, int) {
                        if (v != -INFINITY) {
                            const int b = bin_of(v);
                            atomicAdd(&sh.count[b], 1u);
                            if (use_p) { const u64 m = sc.mass(v); if (m) atomicAdd(&sh.mass[b], m); }
                        }
                    });
                }
                break;
            }
            binned = true;
            __syncthreads();
        }

        // 3. the cut
        if (!drawn) { cut = top; ties = 1; }
        else if (use_k || use_p) {
            if (binned) {
                for (int i = tid; i < kDrawBins; i += TH) {
                    u64 m = 0;
#pragma unroll
                    for (int w = 0; w < W; w++) m += sh.hist[w][i];
                    sh.mass[i] = m;
                }
            }
            __syncthreads();
            run_bins();
        }
        bool ranked = false;                                 // select has run: its bin's members are known
#pragma clang loop unroll(disable)
        for (int by_mass = 0; by_mass < 2; by_mass++) {      // top-k by counts, then top-p by masses
            u64 want;
            if (!by_mass) {
                if (!use_k || (unsigned)top_k > sh.count[kDrawBins - 1]) continue;
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
                if (listed && want > sh.mass[kDrawBins - 1]) break;      // the list ends before: min_p's border decides
            }
            float v;
            u64 above;
            select(want, by_mass != 0, v, above);
            ranked = true;
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
                const bool light = at < n && !(sc.exact(draw_val(lo + at)) >= m64);       // the answer lies behind
                const unsigned k = __popcll(__ballot(light));
                if (k == 0) break;
                lo += (k - 1) * step + 1;
                n = min(step - 1, n - ((k - 1) * step + 1));
            }
            const float v = draw_val(lo);                    // kept: x >= v
            if (v > top) { cut = top; ties = 1; }            // (the first always is)
            else if (v > cut) { cut = draw_val(lo - 1); ties = 0; }
        }
        // masses above the cut and entries equal to it, by wave (without a cut: pass 2's)
        if (cut > -INFINITY) {
            u64 s = 0;
            unsigned t = 0;
            const int bin = binned ? bin_of(cut) : -1;
            if (binned && ranked && bin == sh.bin && (sh.n_rank <= (unsigned)kDrawRank || sh.kmin == sh.kmax)) {
                for (int i = lane; i < bin; i += 64) s += sh.hist[wave][i];
                if (sh.kmin == sh.kmax) t = lane == 0 && draw_val(sh.kmin) == cut ? sh.n_member[wave] : 0;
                if (sh.kmin != sh.kmax || draw_val(sh.kmin) > cut)
                    for (int j = lane; j < (int)min(sh.n_rank, (unsigned)kDrawRank); j += 64)
                        if (sh.rank_wave[j] == wave) { if (sh.rank[j] > cut) s += sh.rank_mass[j]; else t += sh.rank[j] == cut; }
            } else {
                if (binned) for (int i = lane; i < bin; i += 64) s += sh.hist[wave][i];
                pass([&](float x, int) {
                    const bool here = !binned || bin_of(x) == bin;       // (the bins before hold only entries above the cut)
                    if (__any(here && x > cut)) s += here && x > cut ? mass_of(x) : 0;
                    t += x == cut;
                });
            }
            s = wave_sum64(s);
            for (int o = 32; o > 0; o >>= 1) t += __shfl_xor(t, o);
            __syncthreads();
            if (lane == 0) { sh.seg_mass[wave] = s; sh.seg_ties[wave] = t; }
        }
    }

    // 4. the draw, in the vocabulary's order
    const u64 cut_m = ties ? mass_of(cut) : 0;
    const double u = fmin(u_in > 0.0f ? (double)u_in : 0.0, 1.0 - 0x1p-24);
    __syncthreads();
    if (u == 0.0) {                                          // the first kept entry of any weight, below the masses' resolution too
        if (tid == 0) sh.tok = 0xffffffffu;
        __syncthreads();
        unsigned first = 0xffffffffu;
        pass([&](float x, int i) {
            if ((x > cut || (ties && x == cut)) && (x == top || ((double)x - (double)top) / T64 > -745.13)) first = min(first, (unsigned)i);
        });
        if (first != 0xffffffffu) atomicMin(&sh.tok, first);
    } else {
        // lane s: the run of wave s
        const unsigned st = lane < W ? sh.seg_ties[lane] : 0, tx = wave_scan32(st, lane) - st, left = ties > tx ? ties - tx : 0;
        const u64 sm = lane < W ? sh.seg_mass[lane] + (u64)min(st, left) * cut_m : 0, sums = wave_scan64(sm, lane), total = __shfl(sums, 63);
        const u64 target = (u64)(u * (double)total);         // < total: total >= 2^45
        const int pick = __builtin_ctzll(__ballot(sums > target));
        const u64 before = __shfl(sums - sm, pick);
        const unsigned tie_before = __shfl(tx, pick);
        // that run of the vocabulary or that part of the list, each thread E entries in a row, loaded 8 at a time
        const int b = min(V, pick * run), n = listed ? (int)sh.n_listed[pick] : min(V, b + run) - b;
        const int E = (n + TH - 1) / TH, i0 = min(n, tid * E), i1 = min(n, i0 + E);
        auto value = [&](int i) { return listed ? sh.list[pick][i] : clean((float)src[b + i]); };
        auto walk = [&](auto body) __attribute__((always_inline)) {
            for (int g = i0; g < i1; g += 8) {
                float y[8];
#pragma unroll
                for (int j = 0; j < 8; j++) y[j] = value(min(g + j, i1 - 1));
#pragma unroll
                for (int j = 0; j < 8; j++) if (g + j < i1) body(y[j]);
            }
        };
        unsigned t = 0;
        if (ties) walk([&](float v) { t += v == cut; });
        unsigned ts = wave_scan32(t, lane);
        if (lane == 63) sh.wc[wave] = ts;
        __syncthreads();
        ts += tie_before - t;
        for (int w = 0; w < wave; w++) ts += sh.wc[w];
        unsigned rank = ts;
        u64 m = 0;
        walk([&](float v) { m += v > cut ? mass_of(v) : v == cut && rank++ < ties ? cut_m : 0; });
        u64 ms = wave_scan64(m, lane);
        if (lane == 63) sh.wm[wave] = ms;
        __syncthreads();
        ms += before - m;
        for (int w = 0; w < wave; w++) ms += sh.wm[w];
        if (ms <= target && target < ms + m) { sh.walk_at = i0; sh.walk_rank = ts; sh.above = ms; }      // one thread; its entries, one a lane
        __syncthreads();
        if (wave == 0) {
            const int i = sh.walk_at + lane;
            const bool on = lane < E && i < n;
            const float v = on ? value(i) : -INFINITY;
            const u64 eq = __ballot(on && v == cut);
            const u64 w = !on ? 0 : v > cut ? mass_of(v) : v == cut && sh.walk_rank + __popcll(eq & ((1ull << lane) - 1)) < ties ? cut_m : 0;
            const u64 hit = __ballot(sh.above + wave_scan64(w, lane) > target);
            if (lane == 0) {
                const int at = sh.walk_at + __builtin_ctzll(hit);
                sh.tok = (unsigned)(b + (listed ? (int)sh.list_at[pick][at] : at));
            }
        }
    }
    __syncthreads();
    if (tid == 0) {
        const int token = (int)sh.tok;
        a.token[row] = token;
        if (a.logprob) {
            const float v = clean((float)src[token]);
            if (a.whole) a.logprob[row] = (float)((double)v / T64 - (double)a.whole[a.row_of ? a.row_of[row] : row].lse);
            else a.logprob[row] = (float)((v == top ? 0.0 : ((double)v - (double)top) / T64) - log((double)z * (1.0 / kMassOne)));
        }
    }
}

// Threads of a row. Short rows: four waves, so that more rows share a compute unit. Else sixteen if every row has a compute unit of its
// own (256), or eight, two rows a compute unit, whose waits then fall under the other's arithmetic (1024 rows of 51866 entries: 99 us
// against 125). Longer rows take sixteen again: a thread's share is long enough (600 rows of 262144: 317 us against 360).
static int draw_threads(int n_rows, int n_vocab) { return n_vocab <= 16384 ? 256 : n_rows > 256 && n_vocab <= 131072 ? 512 : 1024; }
template <class T> static bool draw_launch(const DrawArgs &a, hipStream_t st) {
    const int th = draw_threads(a.n_rows, a.n_vocab);
    return serve_launch(th == 256 ? draw_kernel<T, 256> : th == 512 ? draw_kernel<T, 512> : draw_kernel<T, 1024>, dim3(a.n_rows), dim3(th), 0, st, a);
}

bool draw_tokens(const DrawArgs &a, hipStream_t st) {
    if (a.n_rows <= 0) return true;
    if (a.dtype == WMI_F32) return draw_launch<float>(a, st);
    return a.dtype == WMI_F16 ? draw_launch<f16>(a, st) : draw_launch<__bf16>(a, st);
}

}  // namespace wmi

using namespace wmi;

extern "C" {

WHISPER_API int wmi_sample_tokens(const void *logits, int dtype, long long row_stride, int n_rows, int n_vocab, const float *uniform, const float *temperature,
                                  const int *top_k, const float *top_p, const float *min_p, int *token, float *logprob, void *stream) {
    if (n_rows < 0 || n_vocab < 1 || row_stride < 0 || (dtype != WMI_F16 && dtype != WMI_BF16 && dtype != WMI_F32)) return -1;
    if (n_vocab > kDrawMaxVocab) return -3;
    if (n_rows == 0) return 0;
    if ((long long)n_rows * draw_threads(n_rows, n_vocab) > 0xffffffffLL) return -3;      // threads of a grid
    if (!logits || !uniform || !token || ((uintptr_t)logits & (dtype == WMI_F32 ? 3 : 1))) return -1;
    // Rows are drawn by workgroups of their own, each of which reads its entry of every array before it writes its outputs: those may lie in
    // place of a parameter's, and nowhere else among what is read.
    auto meet = [](const void *a, long long a_bytes, const void *b, long long b_bytes) { return (uintptr_t)a < (uintptr_t)b + b_bytes && (uintptr_t)b < (uintptr_t)a + a_bytes; };
    const long long each = 4LL * n_rows, all = ((n_rows - 1) * row_stride + n_vocab) * (dtype == WMI_F32 ? 4 : 2);
    if (logprob && meet(token, each, logprob, each)) return -1;
    for (const void *out : {(const void *)token, (const void *)logprob}) {
        if (!out) continue;
        if (meet(out, each, logits, all)) return -1;
        for (const void *in : {(const void *)uniform, (const void *)temperature, (const void *)top_k, (const void *)top_p, (const void *)min_p})
            if (in && in != out && meet(out, each, in, each)) return -1;
    }
    hipStream_t st = (hipStream_t)stream;
    const ServeCall call(st);
    if (!call.ok()) return -4;
    if (!call.own(logits, (const void *)uniform, (const void *)token) || (temperature && !call.owns(temperature)) || (top_k && !call.owns(top_k)) ||
        (top_p && !call.owns(top_p)) || (min_p && !call.owns(min_p)) || (logprob && !call.owns(logprob))) return -1;
    const DrawArgs a{logits, temperature, top_p, min_p, uniform, top_k, nullptr, token, logprob, (long)row_stride, n_rows, n_vocab, dtype, nullptr};
    return draw_tokens(a, st) ? 0 : -4;
}

}  // extern "C"
