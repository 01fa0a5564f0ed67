// sample_uniform.hip — a token for each row of logits from the row's own uniform number: temperature, then top-k, top-p and min-p, then the first token
// (in the order of the vocabulary) whose summed weight exceeds uniform * (sum of what is left).
//
// With m the row's largest logit, token i has the weight w_i = exp((x_i - m) / T).  All three filters keep a prefix of the tokens in descending order (ties: ascending index), so a row's
// answer is decided by two numbers: where the prefix ends, and the sum of its weights.  Nothing is sorted.  The first launch reads the logits once, a chunk of a row a workgroup, and leaves the chunk's
// maximum, its weights (and, for top-k, tokens) in bins of 1/24 of x / T, and a list of its largest tokens.  The second, a workgroup a row, adds the chunks' bins up and finds the bin that the prefix
// ends in.  If the lists have all tokens down to that bin, the chunks' bins are not read: of few tokens (kDirect) each counts what is in front of
// it; up to kList of them stay in LDS, are settled inside the bin, and the drawn one is found by sums over the upper and the lower bits of the index.  Else the order inside the bin is settled by a
// radix select over (logit, index), and the chunk that the drawn number falls into is walked.
// A token's index is an answer that has to be right to the last bit, so weights are 64-bit numbers and are summed as integers, so that the order of the atomics changes nothing: with
// t = 24 x / T in 64 bits, a token lies in the cell of the whole number next to t and adds exp((t - cell) / 24), 0.98 to 1.02, in steps of 2^-40 to it (a polynomial of degree 5, 1e-13 off); a cell
// counts exp(cell / 24).
// Tokens more than 42 T below the largest (e^-42 = 4e-19 of its weight) are left out.
// Rows of 151936 logits (their read alone: 24 us for 256 of them, 4 for one), both launches: one row 15 us with top-k 20, 35 with 1000, 60 with top-p 0.95 that keeps some ten thousand tokens; 256 rows 45, 82
// and 137 (77 + 60), 112 with settings mixed (54 + 58).  The first is bound by 64-bit arithmetic and, for top-p, by the LDS atomics on the bins (two copies of them where a chunk is large: 95 -> 77); the
// second, a workgroup a row, by a chain of scans and LDS round trips, and by walks over a row where the lists end too early.
// What a chunk cannot contribute is left out by one comparison a token: with top-k, whatever lies below the k-th of the chunk's maxima of 4 neighbours (there are k tokens above it), with min-p
// alone, whatever lies below min_p of the chunk's maximum.
#include <algorithm>
#include <cfloat>
#include <type_traits>
#include "serving.h"
#include "device_utils.h"
#include "../common.h"
#include "elem.h"
#include "scan.h"

namespace nvr { namespace kx {

namespace {
// (a token's place in its cell is meant with the product 24 x / T rounded, wherever it is formed)
#pragma clang fp contract(off)
constexpr int kBins = 1024, kPick = 1024, kList = 2048, kRadix = 2048, kNear = 1536;
constexpr double kPerUnit = 24.;                                          // bins to a unit of x / T
constexpr int kOne = 40;                                                  // weights inside a cell are integers of 2^-40
// A token's weight is formed alike in a goal and in the sums that are held against it (by the cell's weight, or by weight()), so that what is off in it (5e-13 by the steps, 2e-13 by the series) is off in both.
// Left are the roundings of sums of doubles: a goal that a sum ought to equal (half of two equal logits) may still lie on either side of it, so top-p's goals are taken a little lower (a sum as large as the goal
// has reached it), the drawn number's a little higher (it has to be passed)
constexpr double kReached = 1. - 2e-14, kPassed = 1. + 2e-14;

// arg: first index of the maximum (greedy rows); cut: the list has every token of bins up to it (-1: there is no list); near: its length; binned: how many bins are in memory, the others are empty (0: the list
// has all that counts); total: the weights of the bins, the chunk's maximum 1
struct ChunkNote { float max; int32_t arg, cut, near, binned, pad; double total; };
struct SampleParams {
    SampleArgs a;
    int32_t V, P, chunk;                                                  // chunks of a row, their tokens
    ChunkNote *notes; unsigned long long *mass; unsigned int *cnt;        // [B][P], [B][P][kBins] twice
    uint2 *near;                                                          // [B][P][kNear]: (key, index)
    bool whole;                                                           // rows in 16-byte pieces
};
// What a row asks for.  T of 0 (or less, or not a number): the largest logit
struct RowAsk { float T; double inv, c; bool greedy; long long k; float p, min_p; };
__device__ __forceinline__ RowAsk row_ask(const SampleArgs &a, int row, int V) {
    RowAsk r;
    r.T = a.temperature ? a.temperature[row] : 1.f;
    r.greedy = !(r.T > 0.f);
    r.inv = kPerUnit / (double)r.T;
    r.c = 1.4426950408889634 / (double)r.T;
    r.k = a.top_k ? a.top_k[row] : 0;
    if (r.k <= 0 || r.k >= V) r.k = 0;
    r.p = a.top_p ? a.top_p[row] : 1.f;
    if (!(r.p >= 0.f && r.p < 1.f)) r.p = 1.f;
    r.min_p = a.min_p ? a.min_p[row] : 0.f;
    r.min_p = r.min_p > 0.f ? fminf(r.min_p, 1.f) : 0.f;
    return r;
}
__device__ __forceinline__ float seen(float x) { return x == x ? x + 0.f : -INFINITY; }  // (not a number: never chosen; -0 is 0)
// t to the nearest whole number: its low bits behind 2^52 + 2^51 (|t| < 2^50; additions are four times as fast here as 64-bit rounding, conversion and scaling)
constexpr double kWhole = 6755399441055744.0;
__device__ __forceinline__ int low_of(double whole) { return (int)(uint32_t)__double_as_longlong(whole); }
// 2^t for t <= 0: the series of exp(r ln 2), |r| <= 1/2
__device__ __forceinline__ double exp2_64(double t) {
    t = fmax(t, -1000.);
    const double whole = t + kWhole, r = t - (whole - kWhole);
    double s = 7.054911620801121e-9;                                      // ln(2)^k / k!
    s = fma(s, r, 1.0178086009239696e-7); s = fma(s, r, 1.3215486790144305e-6); s = fma(s, r, 1.5252733804059838e-5); s = fma(s, r, 1.5403530393381606e-4);
    s = fma(s, r, 1.3333558146428441e-3); s = fma(s, r, 9.618129107628477e-3); s = fma(s, r, 5.5504108664821576e-2); s = fma(s, r, 2.402265069591007e-1);
    s = fma(s, r, 6.931471805599453e-1); s = fma(s, r, 1.0);
    return __longlong_as_double(__double_as_longlong(s) + ((long long)low_of(whole) << 52));
}
__device__ __forceinline__ double weight(float x, float m, double c) { return x == m ? 1.0 : exp2_64(((double)x - (double)m) * c); }
// exp(f / 24) in steps of 2^-40, |f| <= 1/2: the series, every term 2^40 times as large, on top of 2^52: the integer is then the number's low bits
__device__ __forceinline__ double above_2_52(double f) {
    constexpr double one = 1099511627776.0;
    double s = one / (120. * 24 * 24 * 24 * 24 * 24);
    s = fma(s, f, one / (24. * 24 * 24 * 24 * 24)); s = fma(s, f, one / (6. * 24 * 24 * 24)); s = fma(s, f, one / (2. * 24 * 24)); s = fma(s, f, one / 24.);
    return fma(s, f, one + 4503599627370496.0);
}
__device__ __forceinline__ unsigned long long in_cell(double f) { return (unsigned long long)__double_as_longlong(above_2_52(f)) & 0xfffffffffffffull; }
// A maximum that nothing but its equals is near: infinite, or so large that the next number is 2^26 cells away
__device__ __forceinline__ bool lonely(float m, double inv) { return !(fabs((double)m * inv) < 1125899906842624.); }
// bin of x below the maximum m (kBins - 1 and beyond: left out): cells are whole numbers, so bins under a chunk's maximum are a shift away from those under the row's
__device__ __forceinline__ int bin_of(float x, float m, double inv) {
    if (x == m) return 0;
    if (lonely(m, inv)) return kBins - 1;
    const double top = (double)m * inv, d = (top + kWhole) - (fmax((double)x * inv, top - 2. * kBins) + kWhole);
    return d < (double)(kBins - 1) ? (int)d : kBins - 1;
}
__device__ __forceinline__ unsigned int key_of(float f) { const unsigned int u = __float_as_uint(f); return (u & 0x80000000u) ? ~u : (u | 0x80000000u); }
__device__ __forceinline__ float of_key(unsigned int k) { return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k); }
// the last bin that tokens of weight min_p may lie in, and the last in which all have it: (m - x) 24 / T is less than 1 away from x's bin
__device__ __forceinline__ void min_p_bins(float min_p, int &sure, int &last) {
    const double e = -kPerUnit * log((double)min_p);
    sure = (int)fmin(fmax(floor(e) - 2., -1.), (double)(kBins - 2)); last = (int)fmin(ceil(e) + 2., (double)(kBins - 2));
}

// v[j] of registers, a bit of j at a time.  By masks: as conditions the compiler compares anew for each of the selections
template <int N>
__device__ __forceinline__ float pick_of(const float (&v)[N], int j) {
    unsigned int t[N];
#pragma unroll
    for (int i = 0; i < N; ++i) t[i] = __float_as_uint(v[i]);
#pragma unroll
    for (int s = N / 2; s; s /= 2) {
        unsigned int mask = (unsigned int)((int)((unsigned int)j * (0x80000000u / s)) >> 31);
        asm("" : "+v"(mask));
#pragma unroll
        for (int i = 0; i < s; ++i) t[i] = (t[i + s] & mask) | (t[i] & ~mask);
    }
    return __uint_as_float(t[0]);
}
// tokens of a chunk from i on: 4 of them (those behind `end`: -inf)
__device__ __forceinline__ float4_t four(const float *x, int i, int end, bool whole) {
    float4_t v;
    if (whole && i + 4 <= end) v = *reinterpret_cast<const float4_t *>(x + i);
    else
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = i + e < end ? x[i + e] : -INFINITY;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = seen(v[e]);
    return v;
}
__device__ __forceinline__ unsigned int wave_largest(unsigned int v) {
    v = max(v, moved<0x111, 0xf>(v)); v = max(v, moved<0x112, 0xf>(v)); v = max(v, moved<0x114, 0xf>(v)); v = max(v, moved<0x118, 0xf>(v));
    v = max(v, moved<0x142, 0xa>(v)); v = max(v, moved<0x143, 0xc>(v));
    return from_lane(v, 63);
}
template <class T>
__device__ __forceinline__ T wave_total(T v) { return from_lane(wave_scan(v), 63); }
}  // namespace

// A chunk of EPT tokens a thread, held in registers: its maximum, its largest tokens, its bins
template <int EPT, int THREADS>
__global__ __launch_bounds__(THREADS, 8) void sample_scan_kernel(SampleParams p) {
    constexpr int COPIES = EPT == 16 ? 2 : 1;
    __shared__ unsigned long long mass[kBins][COPIES];
    __shared__ unsigned int cnt[kBins];
    __shared__ uint2 near[kNear];
    __shared__ double sums[THREADS / 64];
    __shared__ float wmax[THREADS / 64];
    __shared__ unsigned int wsum[THREADS / 64], listed;
    __shared__ int cut, list_cut, first_at;
    __shared__ unsigned int bins_used;
    constexpr int NG = EPT / 4, BT = kBins / THREADS;                     // maxima of 4 tokens; bins of a thread
    const int c = blockIdx.x, row = blockIdx.y, tid = threadIdx.x, wave = tid >> 6;
    const float *x = p.a.logits + (int64_t)row * p.a.ld;
    const int base = c * p.chunk, end = min(p.V, base + p.chunk);
    auto index = [&](int j) { return base + ((j / 4) * THREADS + tid) * 4 + (j & 3); };
    float v[EPT];
#pragma unroll
    for (int j = 0; j < EPT / 4; ++j) {
        const float4_t f = four(x, index(4 * j), end, p.whole);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[4 * j + e] = f[e];
    }
    const RowAsk ask = row_ask(p.a, row, p.V);
    for (int b = tid; b < kBins; b += THREADS) { for (int e = 0; e < COPIES; ++e) mass[b][e] = 0; cnt[b] = 0; }
    if (tid == 0) { cut = list_cut = kBins - 2; listed = 0; first_at = 0x7fffffff; bins_used = 0; }
    float high[NG];
#pragma unroll
    for (int g = 0; g < NG; ++g) high[g] = fmaxf(fmaxf(v[4 * g], v[4 * g + 1]), fmaxf(v[4 * g + 2], v[4 * g + 3]));
    float m = high[0];
#pragma unroll
    for (int g = 1; g < NG; ++g) m = fmaxf(m, high[g]);
    m = wave_max(m);
    if ((tid & 63) == 0) wmax[wave] = m;
    __syncthreads();
    m = wmax[0];
#pragma unroll
    for (int w = 1; w < THREADS / 64; ++w) m = fmaxf(m, wmax[w]);
    ChunkNote *note = p.notes + (int64_t)row * p.P + c;
    if (ask.greedy) {
        int at = 0x7fffffff;
#pragma unroll
        for (int j = EPT - 1; j >= 0; --j) if (v[j] == m) at = index(j);
        if (at < 0x7fffffff) atomicMin(&first_at, at);
        __syncthreads();
        if (tid == 0) *note = ChunkNote{m, first_at, -1, 0, 0, 0, 0.};
        return;
    }
    if (m == -INFINITY) {                                                 // (nothing to choose here: the bins are not looked at)
        if (tid == 0) *note = ChunkNote{m, 0, kBins, 0, 0, 0, 0.};
        return;
    }
    const bool counted = ask.k > 0, lone = lonely(m, ask.inv), filtered = counted || ask.p < 1.f || ask.min_p > 0.f;
    double total = 0.;                                                    // weights, the chunk's maximum 1 (of rows that top-p or nothing ends)
    auto listing = [&](float x, int j) {
        const unsigned int at = atomicAdd(&listed, 1u);
        if (at < kNear) near[at] = make_uint2(key_of(x), (unsigned int)index(j));
    };
    // f(x, j) for the tokens not below `least`, one a lane at a time: a wave comes to f as often as its busiest lane
    auto each_from = [&](float least, auto f) {
        unsigned int some = 0;
#pragma unroll
        for (int j = 0; j < EPT; ++j) some |= (v[j] >= least ? 1u : 0u) << j;
        while (some) {
            const int j = __ffs((int)some) - 1;
            some &= some - 1;
            f(pick_of(v, j), j);
        }
    };
    int list_end = kBins, bins_end = kBins;                               // tokens of bins up to these go into the list, into the bins
    int binned = 0;
    if (lone) {                                                           // (only the equals of the maximum count)
#pragma unroll
        for (int j = 0; j < EPT; ++j) if (v[j] == m) { listing(m, j); total += 1.; }
        __syncthreads();
        if (listed > kNear) {
            const int64_t at = ((int64_t)row * p.P + c) * kBins;
            if (tid == 0) { p.mass[at] = (unsigned long long)listed << kOne; if (counted) p.cnt[at] = listed; }
            binned = 1; list_end = -1;
        }
    } else if (!filtered) {
        list_end = -1;
#pragma unroll
        for (int j = 0; j < EPT; ++j) total += exp2_64(((double)v[j] - (double)m) * ask.c);
    } else {
        const double t_m = (double)m * ask.inv, whole_m = t_m + kWhole, lowest = t_m - 1.5 * kBins;
        auto cell_of = [&](float x, double &f) {                          // bins below the maximum; f: the place inside the cell
            const double t = fmax((double)x * ask.inv, lowest), whole = t + kWhole;
            f = t - (whole - kWhole);
            return low_of(whole_m) - low_of(whole);
        };
        // the bins of the k-th maximum, and of the one at the list's end: the k-th too, or, of many, three times a chunk's share of k; without top-k one of 11 maxima (96 of a chunk of 4096 tokens)
        const unsigned int want = counted ? (unsigned int)min(ask.k, 0x7fffffffll) : NG * THREADS * 3 / 32, want_list = want <= 96 || !counted ? want : max(96u, (unsigned int)min(3ll * ask.k / p.P, (long long)kNear));
#pragma unroll
        for (int g = 0; g < NG; ++g) { double f; const int b = cell_of(high[g], f); if (b < kBins - 1) atomicAdd(&cnt[b], 1u); }
        __syncthreads();
        unsigned int own[BT], n = 0;
#pragma unroll
        for (int i = 0; i < BT; ++i) { own[i] = cnt[BT * tid + i]; n += own[i]; }
        n = scan<unsigned int>(n, wsum) - n;
#pragma unroll
        for (int i = 0; i < BT; ++i) {
            if (n < want && n + own[i] >= want) cut = BT * tid + i;       // (one thread)
            if (n < want_list && n + own[i] >= want_list) list_cut = BT * tid + i;
            n += own[i];
            cnt[BT * tid + i] = 0;
        }
        __syncthreads();
        bins_end = counted ? cut : kBins - 2;
        if (ask.min_p > 0.f && ask.k == 0 && ask.p == 1.f) {
            int sure, last;
            min_p_bins(ask.min_p, sure, last);
            bins_end = min(bins_end, last);
        }
        list_end = min(list_cut, bins_end);                               // (fewer maxima than wanted: all that is near, if it fits)
        // the lower end of a bin's cell, as a logit; a little less, for the roundings
        auto least_of = [&](int bins) { const float f = (float)(((whole_m - kWhole) - bins - 0.5) / ask.inv); return f - fabsf(f) * 1e-6f; };
        auto into = [&](int b, double f) { atomicAdd(&mass[b][tid & (COPIES - 1)], in_cell(f)); if (counted) atomicAdd(&cnt[b], 1u); };
        bool bins = list_end < bins_end;                                  // (else the list has all that counts, if it fits)
        const bool sparse = bins_end < kBins - 2, both = bins && sparse;
        each_from(least_of(both ? bins_end : list_end), [&](float x, int j) {
            double f;
            const int b = cell_of(x, f);
            if (b <= list_end) listing(x, j);
            if (both && b <= bins_end) into(b, f);
        });
        __syncthreads();
        if (listed > kNear) { bins = true; list_end = -1; }
        if (bins || (!counted && ask.p < 1.f)) {
            if (!sparse) {                                                // all tokens: those too far below go into the last bin, which nobody reads
#pragma unroll
                for (int j = 0; j < EPT; ++j) {
                    double f;
                    const int b = min(cell_of(v[j], f), kBins - 1);
                    into(b, f);
                }
            } else if (!both) {
                each_from(least_of(bins_end), [&](float x, int) {
                    double f;
                    const int b = cell_of(x, f);
                    if (b <= bins_end) into(b, f);
                });
            }
            __syncthreads();
            const int64_t at = ((int64_t)row * p.P + c) * kBins;
            const double off = t_m - (whole_m - kWhole);
            unsigned int used = 0;
            for (int b = tid; b < kBins - 1; b += THREADS) {
                unsigned long long q = mass[b][0];
#pragma unroll
                for (int e = 1; e < COPIES; ++e) q += mass[b][e];
                if (q) used = b + 1;
                if (!counted && q) total += (double)q * exp2_64(-((double)b + off) * (1.4426950408889634 / kPerUnit));
                if (bins) { p.mass[at + b] = q; if (counted) p.cnt[at + b] = cnt[b]; }
            }
            used = wave_largest(used);
            if (bins && (tid & 63) == 0) atomicMax(&bins_used, used);
            total *= 0x1p-40;
        }
    }
    if (!counted) {
        total = wave_total(total);
        if ((tid & 63) == 0) sums[wave] = total;
    }
    __syncthreads();
    const unsigned int n = listed;
    if (list_end >= 0 && n <= kNear)
        for (unsigned int i = tid; i < n; i += THREADS) p.near[((int64_t)row * p.P + c) * kNear + i] = near[i];
    if (tid == 0) {
        total = 0.;
        if (!counted) for (int w = 0; w < THREADS / 64; ++w) total += sums[w];
        *note = ChunkNote{m, 0, list_end, list_end >= 0 ? (int)n : 0, binned ? binned : (int)bins_used, 0, total};
    }
}

namespace {
constexpr int kDirect = 256, kCount = 256, kChunks = 1024;
static_assert(kDirect <= 4 * 64, "waves that hold tokens");
struct PickShared {
    double cum[kBins];                                                    // weight of the bins up to and with this one
    unsigned int cum_n[kBins];
    unsigned long long rmass[kRadix];                                     // (also the tokens that are sorted, and the chunks' sums)
    unsigned int rcnt[kRadix];
    unsigned int key[kList], idx[kList];
    uint16_t near[kChunks], binned[kChunks];                              // tokens of a chunk's list, its bins in memory
    int16_t shift[kChunks];                                               // bins that a chunk's maximum lies under the row's (kBins: nothing of it is near)
    double wsum[16];
    unsigned long long wsum64[16];
    unsigned int wcnt[16];
    unsigned int n, nsel, sel_cnt;
    unsigned int low, high;
    int sel, found;
    unsigned long long sel_mass;
    double part;
};

struct Row {
    const SampleParams &p;
    PickShared &sh;
    const float *x;
    int row, listed, from, to;                                            // from, to: the bins that gather() went over last; listed: the chunks' lists have every token of the row's bins up to it
    RowAsk ask;
    float m;
    double off;                                                           // the maximum's place inside its cell: a cell's weight is exp(-(bins below + off) / 24)
    __device__ __forceinline__ const ChunkNote &note(int c) const { return p.notes[(int64_t)row * p.P + c]; }
    __device__ __forceinline__ double cell(int b) const { return exp2_64(-((double)b + off) * (1.4426950408889634 / kPerUnit)) * 0x1p-40; }      // weight of one unit of bin b
    __device__ __forceinline__ unsigned long long inside(float v) const { if (lonely(m, ask.inv)) return 1ull << kOne; const double t = (double)v * ask.inv; return in_cell(t - ((t + kWhole) - kWhole)); }
    // f(key, index, x, bin) for the tokens of bins lo .. hi in the chunks' lists, a wave a chunk
    template <class F>
    __device__ __forceinline__ void each_listed(int lo, int hi, F f) const {
        const int lane = threadIdx.x & 63;
        for (int c0 = threadIdx.x >> 6; c0 < p.P; c0 += kPick / 16) {     // (64 tokens of 4 chunks together)
            int n[4], most = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int c = c0 + e * (kPick / 64);
                n[e] = c < p.P && sh.shift[c] <= hi ? same((int)sh.near[c]) : 0;
                most = max(most, n[e]);
            }
            for (int i = lane; i - lane < most; i += 64) {
                uint2 q[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) if (i < n[e]) q[e] = p.near[((int64_t)row * p.P + c0 + e * (kPick / 64)) * kNear + i];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if (i >= n[e]) continue;
                    const uint2 k = q[e];
                    const float v = of_key(k.x);
                    const int b = bin_of(v, m, ask.inv);
                    if (b >= lo && b <= hi) f(k.x, k.y, v, b);
                }
            }
        }
    }
    // logits of bins lo .. hi are not below `least` nor above `most`
    __device__ __forceinline__ void ends_of(int lo, int hi, float &least, float &most) const {
        const double top = ((double)m * ask.inv + kWhole) - kWhole;       // (the cells' ends are halves)
        const float a = (float)((top - hi - 0.5) / ask.inv), z = (float)((top - lo + 0.5) / ask.inv);
        const bool lone = lonely(m, ask.inv);
        least = fminf(lone ? m : a - fabsf(a) * 1e-6f, FLT_MAX); most = lone || lo == 0 ? INFINITY : z + fabsf(z) * 1e-6f;
        if (!(least == least && most == most)) { least = -INFINITY; most = INFINITY; }      // (1 / inv beyond float)
    }
    // ... in the row itself.  Most tokens are outside: the signs of x less the bins' lower end and the upper end less x (a little beyond, for their roundings) tell, four instructions a token.
    // Numbers that are none may pass here
    template <class F>
    __device__ __forceinline__ void each_of_row(int lo, int hi, F f) const {
        float least, most;
        ends_of(lo, hi, least, most);
        for (int i0 = threadIdx.x * 4; i0 < p.V; i0 += kPick * 16) {
            float v[16];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int i = i0 + u * kPick * 4;
                float4_t w;
                if (p.whole && i + 4 <= p.V) w = *reinterpret_cast<const float4_t *>(x + i);
                else
#pragma unroll
                    for (int e = 0; e < 4; ++e) w[e] = i + e < p.V ? x[i + e] : -INFINITY;
#pragma unroll
                for (int e = 0; e < 4; ++e) v[4 * u + e] = w[e];
            }
            unsigned int outside = 0;
#pragma unroll
            for (int e = 15; e >= 0; --e) outside = __builtin_amdgcn_alignbit(outside, __float_as_uint(fminf(v[e] - least, most - v[e])), 31);
            unsigned int near = ~outside & 0xffffu;                       // one a lane at a time: a wave comes to f as often as its busiest lane
            while (near) {
                const int j = __ffs((int)near) - 1;
                near &= near - 1;
                const float w = seen(pick_of(v, j));
                const int b = bin_of(w, m, ask.inv);
                if (b >= lo && b <= hi && b < kBins - 1) f(key_of(w), (unsigned int)(i0 + (j >> 2) * kPick * 4 + (j & 3)), w, b);
            }
        }
    }
    template <class F>
    __device__ __forceinline__ void each(int lo, int hi, F f) const { if (hi <= listed) each_listed(lo, hi, f); else each_of_row(lo, hi, f); }
    // the tokens of bins lo .. hi (and maybe more) into LDS; false: they are more than it holds
    __device__ __forceinline__ bool gather(int lo, int hi) {
        if (from <= lo && hi <= to && same(sh.n) <= kList) return true;   // (they are there)
        if (lo == from && hi == to) return false;
        from = lo; to = hi;
        if (threadIdx.x == 0) sh.n = 0;
        __syncthreads();
        each(lo, hi, [&](unsigned int k, unsigned int i, float, int) {
            const unsigned int at = atomicAdd(&sh.n, 1u);
            if (at < kList) { sh.key[at] = k; sh.idx[at] = i; }
        });
        __syncthreads();
        return same(sh.n) <= kList;
    }
    template <class F>
    __device__ __forceinline__ void each_gathered(bool all_here, int lo, int hi, F f) const {
        if (!all_here) { each(lo, hi, f); return; }
        for (unsigned int i = threadIdx.x; i < sh.n; i += kPick) {
            const unsigned int k = sh.key[i];
            const float v = of_key(k);
            const int b = bin_of(v, m, ask.inv);
            if (b >= lo && b <= hi) f(k, sh.idx[i], v, b);
        }
    }
    // Among the tokens of bin b in descending order (ties: ascending index): the last one that is kept, when `need` of them are (need > 0) or as many as it takes until `before` plus their weights
    // reaches `goal`.  part: the weight of the kept ones.  Of few tokens, a thread a token, each counts those in front of it; else a radix select over 11 bits of the logit at a time, then over 11
    // and 11 of the index
    // mass: the bin's.  Its tokens weigh 0.98 to 1.02 units each, so it tells whether LDS can have them, and a walk over the row for nothing is spared
    __device__ __forceinline__ void settle(int b, double mass, unsigned int need, double before, double goal, unsigned int &key, unsigned int &index, double &part) {
        const bool here = (b <= listed || mass <= cell(b) * (1.05 * kList * 0x1p40)) && gather(b, b);
        const int tid = threadIdx.x;
        const double unit = cell(b);
        if (here) {
            unsigned long long *v = sh.rmass, *w = v + kCount;
            if (tid == 0) { sh.sel_cnt = 0; sh.found = 0x7fffffff; }
            __syncthreads();
            each_gathered(true, b, b, [&](unsigned int k, unsigned int i, float f, int) {
                const unsigned int at = atomicAdd(&sh.sel_cnt, 1u);
                if (at < kCount) { v[at] = ((unsigned long long)~k << 32) | i; w[at] = inside(f); }
            });
            __syncthreads();
            const int n = same((int)sh.sel_cnt);
            if (n == 0) { key = 0; index = 0xffffffffu; part = 0.; __syncthreads(); return; }      // (no token: everything is kept)
            if (n <= kCount) {
                int rank = 0;
                unsigned long long upto = 0;
                if (tid < n) {
                    const unsigned long long a = v[tid];
#pragma unroll 4
                    for (int j = 0; j < n; ++j) { const bool in = v[j] <= a; rank += in; upto += in ? w[j] : 0; }      // (no two are alike)
                    if (need ? rank >= (int)need : before + (double)upto * unit >= goal) atomicMin(&sh.found, rank);
                }
                __syncthreads();
                if (tid < n && rank == min(sh.found, n)) { sh.low = ~(unsigned int)(v[tid] >> 32); sh.high = (unsigned int)v[tid]; sh.part = (double)upto * unit; }      // (where rounding leaves the goal unreached, the last)
                __syncthreads();
                key = same(sh.low); index = same(sh.high); part = same(sh.part);
                __syncthreads();
                return;
            }
        }
        unsigned int left = need, equal = 0;
        unsigned long long done = 0;                                      // weight above the prefix
        // the tokens of a bin are alike in their upper bits: those are the first prefix
        float least, most;
        ends_of(b, b, least, most);
        const unsigned int low = key_of(least), high = key_of(fminf(most, m));
        const int bits = low == high ? 0 : 32 - __clz((int)(low ^ high)); // that differ
        unsigned int mask = bits >= 32 ? 0 : 0xffffffffu << bits, prefix = high & mask;
        for (int at = bits;;) {
            const int wide = 1 << min(at, 11);
            at = max(at - 11, 0);
            for (int i = tid; i < kRadix; i += kPick) { sh.rcnt[i] = 0; sh.rmass[i] = 0; }
            if (tid == 0) { sh.found = 0x7fffffff; sh.sel = -1; }
            __syncthreads();
            each_gathered(here, b, b, [&](unsigned int k, unsigned int, float v, int) {
                if ((k & mask) != prefix) return;
                const int d = wide - 1 - (int)((k >> at) & (wide - 1));   // descending
                atomicAdd(&sh.rcnt[d], 1u);
                atomicAdd(&sh.rmass[d], inside(v));
            });
            __syncthreads();
            const unsigned int c0 = sh.rcnt[2 * tid], c1 = sh.rcnt[2 * tid + 1];
            const unsigned long long m0 = sh.rmass[2 * tid], m1 = sh.rmass[2 * tid + 1];
            const unsigned int u1 = scan<unsigned int>(c0 + c1, sh.wcnt), u0 = u1 - c1;
            const unsigned long long s1 = scan<unsigned long long>(m0 + m1, sh.wsum64), s0 = s1 - m1;
            // the first digit that the end falls into (or, where rounding leaves the goal unreached, the last that has tokens)
            auto ends = [&](unsigned int n, unsigned long long s) { return need ? n >= left : before + (double)(done + s) * unit >= goal; };
            if (c0 && ends(u0, s0)) atomicMin(&sh.found, 2 * tid);
            else if (c1 && ends(u1, s1)) atomicMin(&sh.found, 2 * tid + 1);
            {
                const unsigned long long some = __ballot((c0 | c1) != 0);
                if (some && (tid & 63) == 63 - __clzll((long long)some)) atomicMax(&sh.sel, c1 ? 2 * tid + 1 : 2 * tid);
            }
            __syncthreads();
            const int d = same(sh.found != 0x7fffffff ? sh.found : sh.sel);
            if (tid == d / 2) {
                const bool odd = d & 1;
                sh.sel_cnt = odd ? u0 : u0 - c0; sh.sel_mass = odd ? s0 : s0 - m0;
                sh.nsel = odd ? c1 : c0;
            }
            __syncthreads();
            if (need) left -= min(left, same(sh.sel_cnt));
            done += same(sh.sel_mass);
            equal = same(sh.nsel);
            prefix |= (unsigned int)(wide - 1 - d) << at; mask |= (unsigned int)(wide - 1) << at;
            __syncthreads();
            if (at == 0) break;
        }
        key = prefix;
        const double w = (double)inside(of_key(prefix)) * unit, start = before + (double)done * unit;
        unsigned int n = left;
        if (!need) {
            const double q = ceil((goal - start) / w);
            n = q >= (double)equal ? equal : q < 1. ? 1u : (unsigned int)q;
            if (n > 1 && start + (n - 1) * w >= goal) --n;
            else if (n < equal && start + n * w < goal) ++n;
        }
        n = min(max(n, 1u), equal);
        part = (double)done * unit + n * w;
        index = 0xffffffffu;
        if (n == equal) return;
        unsigned int at_prefix = 0, at_mask = 0, want = n;                // which of the equal ones: the n-th smallest index
        for (int at = 11; at >= 0; at -= 11) {
            for (int i = tid; i < kRadix; i += kPick) sh.rcnt[i] = 0;
            if (tid == 0) sh.found = 0x7fffffff;
            __syncthreads();
            each_gathered(here, b, b, [&](unsigned int k, unsigned int i, float, int) { if (k == key && (i & at_mask) == at_prefix) atomicAdd(&sh.rcnt[(i >> at) & (kRadix - 1)], 1u); });
            __syncthreads();
            const unsigned int c0 = sh.rcnt[2 * tid], c1 = sh.rcnt[2 * tid + 1], nc = scan<unsigned int>(c0 + c1, sh.wcnt);
            if (c0 && nc - c1 >= want) atomicMin(&sh.found, 2 * tid);
            else if (c1 && nc >= want) atomicMin(&sh.found, 2 * tid + 1);
            __syncthreads();
            const int d = same(sh.found);
            if (tid == d / 2) sh.sel_cnt = (d & 1) ? nc - c1 : nc - c1 - c0;
            __syncthreads();
            want -= same(sh.sel_cnt);
            at_prefix |= (unsigned int)d << at; at_mask |= (unsigned int)(kRadix - 1) << at;
            __syncthreads();
        }
        index = at_prefix;
    }
};
}  // namespace

__global__ __launch_bounds__(kPick) void sample_pick_kernel(SampleParams p) {
    __shared__ PickShared sh;
    const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const ChunkNote *notes = p.notes + (int64_t)row * p.P;
    Row r{p, sh, p.a.logits + (int64_t)row * p.a.ld, row, kBins - 2, -1, -1, row_ask(p.a, row, p.V), -INFINITY, 0.};
    const RowAsk &ask = r.ask;
    const double u = (double)p.a.uniform[row];
    const ChunkNote mine = tid < p.P ? notes[tid] : ChunkNote{-INFINITY, 0, kBins, 0, 0, 0, 0.};      // (up to kChunks of them)
    {
        float *waves = reinterpret_cast<float *>(sh.wsum);
        const float v = wave_max(mine.max);
        if (lane == 0) waves[wave] = v;
        if (tid == 0) sh.found = 0x7fffffff;
        __syncthreads();
        r.m = same(wave_max(waves[lane & 15]));
        __syncthreads();
    }
    if (r.m == -INFINITY || ask.greedy) {
        if (mine.max == r.m && r.m != -INFINITY) atomicMin(&sh.found, mine.arg);
        __syncthreads();
        if (tid == 0) {
            const int64_t id = r.m != -INFINITY ? sh.found : -1;
            p.a.ids[row] = id;
            if (p.a.logprobs) p.a.logprobs[row] = id < 0 ? -INFINITY : 0.f;
        }
        return;
    }
    if (!lonely(r.m, ask.inv)) { const double t = (double)r.m * ask.inv; r.off = t - ((t + kWhole) - kWhole); }
    // the first thread for which something holds (kBins: none)
    auto first_of = [&](bool holds) {
        if (tid == 0) sh.found = kBins;
        __syncthreads();
        const unsigned long long b = __ballot(holds);
        if (lane == 0 && b) atomicMin(&sh.found, wave * 64 + __ffsll((long long)b) - 1);
        __syncthreads();
        const int f = same(sh.found);
        __syncthreads();
        return f;
    };
    // ---- the chunks: where their bins lie, how far their lists reach, the row's weight
    double everything;
    {
        int s = kBins, reach = kBins - 2;
        double t = 0.;
        if (tid < p.P && mine.max > -INFINITY) {
            s = bin_of(mine.max, r.m, ask.inv);
            if (s >= kBins - 1) s = kBins;
            else { reach = mine.cut < 0 ? -1 : min(s + mine.cut, kBins - 2); t = mine.total * weight(mine.max, r.m, ask.c); }
        }
        if (tid < p.P) { sh.shift[tid] = (int16_t)s; sh.near[tid] = (uint16_t)mine.near; sh.binned[tid] = (uint16_t)mine.binned; }
        if (tid == 0) sh.sel = kBins - 2;
        t = scan<double>(t, sh.wsum);
        if (reach < kBins - 2) atomicMin(&sh.sel, reach);
        if (tid == kPick - 1) sh.part = t;
        __syncthreads();
        everything = same(sh.part); r.listed = same(sh.sel);
    }
    const bool filtered = ask.k || ask.p < 1.f || ask.min_p > 0.f;
    const unsigned int k = (unsigned int)ask.k;                           // (below V)
    int p_sure = kBins - 2, p_last = kBins - 2;                           // min-p: bins that have it throughout, and in part
    if (ask.min_p > 0.f) min_p_bins(ask.min_p, p_sure, p_last);
    // ---- the lists have all that may be kept, down to the bin that the first filter ends in?
    bool from_lists = false, in_lds = false;                              // ... and LDS too
    if (filtered && r.listed >= 0) {
        unsigned long long *bin = sh.rmass;
        unsigned int *cnt = sh.rcnt;
        bin[tid] = 0; cnt[tid] = 0;
        if (tid == 0) sh.n = 0;
        __syncthreads();
        r.each_listed(0, r.listed, [&](unsigned int key, unsigned int i, float v, int b) {
            atomicAdd(&bin[b], r.inside(v)); atomicAdd(&cnt[b], 1u);
            const unsigned int at = atomicAdd(&sh.n, 1u);
            if (at < kList) { sh.key[at] = key; sh.idx[at] = i; }
        });
        __syncthreads();
        const bool here = same(sh.n) <= kList;
        const double cum = scan<double>((double)bin[tid] * r.cell(tid), sh.wsum);
        const unsigned int cum_n = scan<unsigned int>(cnt[tid], sh.wcnt);
        int reach = kBins;
        if (ask.k) reach = first_of(cum_n >= k);
        else if (ask.p < 1.f) reach = first_of(cum >= (double)ask.p * everything * kReached && cum_n > 0);
        if (ask.min_p > 0.f && (!ask.k || ask.p == 1.f)) reach = min(reach, p_last);      // (what top-k keeps in all is wanted for top-p)
        if (reach > r.listed && ask.k && r.listed == kBins - 2) reach = r.listed;         // (fewer tokens than top-k would keep)
        if (tid == min(reach, kBins - 1)) sh.nsel = cum_n;
        sh.cum[tid] = cum; sh.cum_n[tid] = cum_n;
        __syncthreads();
        const int few = same((int)sh.nsel);
        from_lists = reach <= r.listed && few > 0;
        if (here) { r.from = 0; r.to = r.listed; }
        if (from_lists && few > kDirect && few <= kList) in_lds = r.gather(0, reach);
        if (from_lists && few <= kDirect) {
            // ---- few: a thread a token, each counts what is in front of it and its weight (whole numbers of 2^-52, 1 at least), by the logits and then by the indices
            ulonglong2 *t = reinterpret_cast<ulonglong2 *>(sh.rmass);     // (what sorts by descending logits and ascending indices, weight)
            if (tid == 0) { sh.sel = 0; sh.low = 0xffffffffu; sh.high = 0; }
            __syncthreads();
            auto take = [&](unsigned int key, unsigned int i, float, int b) { if (b <= reach) t[atomicAdd(&sh.sel, 1)].x = ((unsigned long long)~key << 32) | i; };
            if (here) r.each_gathered(true, 0, reach, take);
            else r.each_listed(0, reach, take);
            __syncthreads();
            const int n = same(sh.sel);
            const unsigned long long mine_v = tid < n ? t[tid].x : 0;
            const unsigned int id = (unsigned int)mine_v;
            const double x = tid < n ? weight(of_key(~(unsigned int)(mine_v >> 32)), r.m, ask.c) : 0.;
            auto whole = [&](double w) { return tid < n ? max(1ull, (unsigned long long)(w * 0x1p52 + 0.5)) : 0; };
            unsigned long long q = whole(x), upto = 0, all = 0;
            const unsigned long long drawn = q;
            if (ask.p < 1.f && !ask.k) {                                  // (held against the sum of the bins: as they have it)
                const float v = of_key(~(unsigned int)(mine_v >> 32));
                q = whole((double)r.inside(v) * r.cell(bin_of(v, r.m, ask.inv)));
            }
            if (tid < n) t[tid].y = q;
            __syncthreads();
            int rank = 0;
            if (tid < n)
#pragma unroll 4
                for (int j = 0; j < n; ++j) { const ulonglong2 o = t[j]; const bool in = o.x <= mine_v; rank += in; upto += in ? o.y : 0; }
            bool keep = tid < n && (!ask.k || rank <= (int)k);
            if (ask.p < 1.f) {
                double total = everything * 0x1p52;
                if (ask.k) {
                    const unsigned long long of_wave = wave_total(keep ? q : 0);
                    if (lane == 0) sh.wsum64[wave] = of_wave;
                    __syncthreads();
                    total = (double)(sh.wsum64[0] + sh.wsum64[1] + sh.wsum64[2] + sh.wsum64[3]);
                }
                keep = keep && (rank == 1 || (double)(upto - q) < (double)ask.p * total * kReached);
            }
            keep = keep && !(ask.min_p > 0.f && x < (double)ask.min_p);
            q = keep ? drawn : 0;
            __syncthreads();
            if (tid < n) t[tid].y = q;
            __syncthreads();
            upto = 0;
            if (tid < n) {
#pragma unroll 4
                for (int j = 0; j < n; ++j) { const ulonglong2 o = t[j]; all += o.y; upto += (unsigned int)o.x <= id ? o.y : 0; }
                if (q) { if ((double)upto > u * (double)all) atomicMin(&sh.low, id); atomicMax(&sh.high, id); }
            }
            __syncthreads();
            if (q && id == (sh.low != 0xffffffffu ? sh.low : sh.high)) {  // (no goal below the sum: the last one)
                p.a.ids[row] = id;
                if (p.a.logprobs) p.a.logprobs[row] = (float)log(x * 0x1p52 / (double)all);
            }
            return;
        }
        __syncthreads();
    }
    // ---- many: the row's bins, thread b bin b: those of the lists, or from the chunks', or, of the chunks that left none, from their lists
    int stop = kBins;                                                     // bins in front of it are kept whole; of this one, tokens down to (key, index)
    unsigned int key = 0, index = 0xffffffffu;
    const double unit_of_bin = r.cell(tid);
    if (filtered && !from_lists) {
        sh.rmass[tid] = 0; sh.rcnt[tid] = 0;
        __syncthreads();
        for (int c = wave; c < p.P; c += kPick / 64) {
            const int s = sh.shift[c];
            if (s >= kBins || sh.binned[c]) continue;
            const uint2 *q = p.near + ((int64_t)row * p.P + c) * kNear;
            for (int i = lane; i < sh.near[c]; i += 64) {
                const float v = of_key(q[i].x);
                const int b = bin_of(v, r.m, ask.inv);
                if (b < kBins - 1) { atomicAdd(&sh.rmass[b], r.inside(v)); atomicAdd(&sh.rcnt[b], 1u); }
            }
        }
        __syncthreads();
        unsigned long long in_bin = sh.rmass[tid];
        unsigned int cnt = sh.rcnt[tid];
        for (int c0 = 0; c0 < p.P; c0 += 16) {                            // (16 chunks' requests together)
            auto of_chunks = [&](const auto *table, auto &sum) {
                auto q = std::remove_reference_t<decltype(sum)>(0);
                std::remove_reference_t<decltype(sum)> v[16];
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const int c = min(c0 + e, p.P - 1), b = tid - sh.shift[c];
                    v[e] = c0 + e < p.P && b >= 0 && b < sh.binned[c] && tid < kBins - 1 ? table[((int64_t)row * p.P + c) * kBins + b] : 0;
                }
#pragma unroll
                for (int e = 0; e < 16; ++e) q += v[e];
                sum += q;
            };
            of_chunks(p.mass, in_bin);
            if (ask.k) of_chunks(p.cnt, cnt);
        }
        sh.cum[tid] = scan<double>((double)in_bin * unit_of_bin, sh.wsum);
        sh.cum_n[tid] = scan<unsigned int>(cnt, sh.wcnt);
        __syncthreads();
    }
    if (filtered) {
        double total = ask.k ? same(sh.cum[kBins - 1]) : everything;
        for (int filter = 0; filter < 2; ++filter) {                      // top-k, top-p
            if (filter == 0 ? !ask.k : ask.p == 1.f) continue;
            const double goal = filter ? (double)ask.p * total * kReached : 0.;
            const int b = first_of(filter ? sh.cum[tid] >= goal && sh.cum[tid] > 0. && tid < stop : sh.cum_n[tid] >= k);
            const int bin = filter && b == kBins ? stop : b;              // (the bin that top-k ended in, or none)
            if (bin == kBins || (filter && b == kBins && key == 0 && index == 0xffffffffu)) continue;
            if (bin > p_last && (filter || ask.p == 1.f)) { stop = bin; key = 0; index = 0xffffffffu; continue; }      // (min-p leaves less)
            const double before = bin ? same(sh.cum[bin - 1]) : 0.;
            if (!filter && same(sh.cum_n[bin]) == k) { stop = bin + 1; total = same(sh.cum[bin]); continue; }
            unsigned int k2, i2;
            double part;
            r.settle(bin, same(sh.cum[bin]) - before, filter ? 0 : k - (bin ? same(sh.cum_n[bin - 1]) : 0), before, goal, k2, i2, part);
            if (bin < stop || k2 > key || (k2 == key && i2 < index)) { key = k2; index = i2; }      // (in the bin where top-k ended, its own end may come first)
            stop = bin;
            if (!filter) total = before + part;
        }
    }
    // whole bins in front of `sure`; single tokens of bins sure .. last
    const bool by_key = stop < kBins && !(key == 0 && index == 0xffffffffu);
    const int key_bin = stop, sure = min(stop, p_sure + 1), last = min(min(by_key ? stop : stop - 1, p_last), kBins - 2);
    const bool cut = filtered && last >= sure;                            // (without filters all bins are whole)
    // enough(): whether weight() of the token is min_p and more
    auto kept = [&](int b, unsigned int kk, unsigned int i, auto enough) {
        if (b < sure) return true;
        if (b > last) return false;
        if (by_key && b == key_bin && (kk < key || (kk == key && i > index))) return false;
        return !(ask.min_p > 0.f) || enough();
    };
    if (in_lds) {
        // ---- the token among up to kList in LDS (thread t has t and t + kPick): weights are whole numbers of 2^-52 (and 1 at least), summed by the upper 11 bits of the index and then by the others
        unsigned long long q[2] = {0, 0};
        unsigned int i[2] = {0, 0}, id = 0;
        double w[2] = {0., 0.};
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const unsigned int at = tid + e * kPick;
            if (at >= sh.n) continue;
            const unsigned int kk = sh.key[at];
            const float v = of_key(kk);
            i[e] = sh.idx[at]; w[e] = weight(v, r.m, ask.c);
            if (kept(bin_of(v, r.m, ask.inv), kk, i[e], [&] { return w[e] >= (double)ask.min_p; })) q[e] = max(1ull, (unsigned long long)(w[e] * 0x1p52 + 0.5));
        }
        unsigned long long done = 0;
        double sum = 0., goal = 0.;
        const int lower = max(32 - __clz(p.V - 1) - 11, 0);               // 11 at most
        for (int level = 0; level < (lower ? 2 : 1); ++level) {
            sh.rmass[2 * tid] = 0; sh.rmass[2 * tid + 1] = 0;
            if (tid == 0) { sh.found = 0x7fffffff; sh.sel = 0; }
            __syncthreads();
#pragma unroll
            for (int e = 0; e < 2; ++e)
                if (q[e] && (level == 0 || i[e] >> lower == id)) atomicAdd(&sh.rmass[level ? i[e] & ((1u << lower) - 1) : i[e] >> lower], q[e]);
            __syncthreads();
            const unsigned long long m0 = sh.rmass[2 * tid], m1 = sh.rmass[2 * tid + 1], s1 = scan<unsigned long long>(m0 + m1, sh.wsum64), s0 = s1 - m1;
            if (level == 0) {
                if (tid == kPick - 1) sh.sel_mass = s1;
                __syncthreads();
                sum = (double)same(sh.sel_mass); goal = u * sum;
                __syncthreads();
            }
            if (m0 && (double)(done + s0) > goal) atomicMin(&sh.found, 2 * tid);
            else if (m1 && (double)(done + s1) > goal) atomicMin(&sh.found, 2 * tid + 1);
            if (m0 | m1) atomicMax(&sh.sel, m1 ? 2 * tid + 1 : 2 * tid);
            __syncthreads();
            const int d = same(sh.found != 0x7fffffff ? sh.found : sh.sel);      // (no goal below the sum: the last one)
            if (tid == d / 2) sh.sel_mass = (d & 1) ? s0 : s0 - m0;
            __syncthreads();
            done += same(sh.sel_mass);
            __syncthreads();
            id = level ? id << lower | (unsigned int)d : (unsigned int)d;
        }
#pragma unroll
        for (int e = 0; e < 2; ++e)
            if (q[e] && i[e] == id) {
                p.a.ids[row] = i[e];
                if (p.a.logprobs) p.a.logprobs[row] = (float)log(w[e] * 0x1p52 / sum);
            }
        return;
    }
    // ---- what each chunk keeps: its whole bins, and its single tokens in steps of 2^-48 of the heaviest there may be (16384 of 1.02 at most)
    __syncthreads();
    double *units = sh.cum, *sums = reinterpret_cast<double *>(sh.rmass + kChunks);      // weight of a unit of each bin (the sums of bins have been looked at); of up to kChunks
    unsigned long long *single = reinterpret_cast<unsigned long long *>(sh.rmass);
    static_assert(kRadix >= 2 * kChunks, "");
    const double unit = cut ? r.cell(sure) * 0x1p-8 : 0., steps = cut ? 1. / unit : 0.;
    single[tid] = 0;
    units[tid] = unit_of_bin;
    const bool here = cut && r.gather(sure, last);
    __syncthreads();
    // A token's weight is the cell's times the place's inside (half the work of an exponential).  It and weight() are within 1e-7 of each other (5e-13 of the steps inside a cell, and 2^-53 of 24 x / T, which is
    // below 2^34 where tokens of different logits are near).  Where min_p is as close, weight() decides: it is exactly 1 for the largest logit, and the product may be below
    auto close = [&](double w) { return fabs(w - (double)ask.min_p) <= 1e-6 * w; };
    if (cut)
        r.each_gathered(here, sure, last, [&](unsigned int kk, unsigned int i, float v, int b) {
            const double w = (double)r.inside(v) * units[b];
            if (kept(b, kk, i, [&] { return (close(w) ? weight(v, r.m, ask.c) : w) >= (double)ask.min_p; })) atomicAdd(&single[i / p.chunk], (unsigned long long)(w * steps + 0.5));
        });
    __syncthreads();
    for (int c = wave; c < p.P; c += kPick / 64) {
        const int s = sh.shift[c];
        double v = 0.;
        if (s < kBins) {
            if (!filtered) v = lane == 0 ? notes[c].total * weight(notes[c].max, r.m, ask.c) : 0.;
            else if (sh.binned[c]) {
                const unsigned long long *q = p.mass + ((int64_t)row * p.P + c) * kBins;
                for (int b = lane; b < min(sure - s, (int)sh.binned[c]); b += 64) v += (double)q[b] * units[b + s];
            } else {
                const uint2 *q = p.near + ((int64_t)row * p.P + c) * kNear;
                unsigned long long n = 0;                                 // (a list's order is that of its arrival: whole numbers of 2^-52, 1 at least)
                for (int i = lane; i < sh.near[c]; i += 64) {
                    const float f = of_key(q[i].x);
                    const int b = bin_of(f, r.m, ask.inv);
                    if (b < sure && b < kBins - 1) n += max(1ull, (unsigned long long)((double)r.inside(f) * units[b] * 0x1p52 + 0.5));
                }
                const unsigned long long all = wave_total(n);
                v = lane == 0 ? (double)all * 0x1p-52 : 0.;
            }
            v = wave_total(v) + (double)single[c] * unit;
        }
        if (lane == 0) sums[c] = v;
    }
    __syncthreads();
    // the chunk that the goal falls into (thread c chunk c)
    const double own = tid < p.P ? sums[tid] : 0., upto_c = scan<double>(own, sh.wsum);
    if (tid == kPick - 1) sh.part = upto_c;
    if (tid == 0) sh.sel = 0;
    __syncthreads();
    const double sum = same(sh.part), goal = u * sum * kPassed;
    int c = first_of(own > 0. && upto_c > goal);
    if (c == kBins) {
        if (own > 0.) atomicMax(&sh.sel, tid);
        __syncthreads();
        c = same(sh.sel);
        __syncthreads();
    }
    if (tid == c) sh.part = upto_c - own;
    if (tid == 0) sh.sel = -1;
    __syncthreads();
    // ---- the token of that chunk: a thread's tokens are neighbours
    const int per = p.chunk / kPick, base = c * p.chunk + tid * per, end = min(p.V, c * p.chunk + p.chunk);      // 4 or 16
    const bool lone = lonely(r.m, ask.inv);
    const double t_m = (double)r.m * ask.inv, whole_m = t_m + kWhole;
    // the weight, as the chunk's sum has it
    auto of = [&](float v, int i, auto enough) {
        if (v == -INFINITY || (lone && v != r.m)) return 0.;
        const double at = fmax((double)v * ask.inv, t_m - 2. * kBins), whole = at + kWhole;
        const int b = lone ? 0 : low_of(whole_m) - low_of(whole);
        if (b >= kBins - 1 || (b >= sure && b > last)) return 0.;
        const double w = lone ? 1. : (above_2_52(at - (whole - kWhole)) - 4503599627370496.0) * units[b];
        return kept(b, key_of(v), (unsigned int)i, [&] { return enough(w, v); }) ? w : 0.;
    };
    auto unfiltered = [&](float v) { return bin_of(v, r.m, ask.inv) >= kBins - 1 ? 0. : weight(v, r.m, ask.c); };      // (what is left out goes by the bins, as where a chunk is)
    // (near min_p alone, and once, behind the loop: weight() for every token in it took 189 us for 256 rows of 151936 with min-p 0.001, this 186)
    auto exactly = [&](double w, float v) { return (close(w) ? weight(v, r.m, ask.c) : w) >= (double)ask.min_p; };
    float4_t f[4];
    double here_sum = 0.;
    unsigned int doubt = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) f[j] = four(r.x, base + 4 * j, 4 * j < per ? end : 0, p.whole);
#pragma unroll 1
    for (int j = 0; 4 * j < per; ++j) {                                   // (not unrolled: code that runs once costs its way from memory)
        const float4_t g = j & 2 ? j & 1 ? f[3] : f[2] : j & 1 ? f[1] : f[0];
        if (!filtered) {
#pragma unroll
            for (int e = 0; e < 4; ++e) here_sum += unfiltered(g[e]);
            continue;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e)
            here_sum += of(g[e], base + 4 * j + e, [&](double w, float) {
                doubt |= (close(w) ? 1u : 0u) << (4 * j + e);
                return !close(w) && w >= (double)ask.min_p;
            });
    }
    while (doubt) {
        const int i = base + __ffs((int)doubt) - 1;
        doubt &= doubt - 1;
        here_sum += of(seen(r.x[i]), i, exactly);
    }
    const double upto = scan<double>(here_sum, sh.wsum);
    int t = first_of(here_sum > 0. && sh.part + upto > goal);
    if (t == kBins) {
        if (here_sum > 0.) atomicMax(&sh.sel, tid);
        __syncthreads();
        t = same(sh.sel);
    }
    float *values = reinterpret_cast<float *>(sh.idx);                    // of thread t: the first wave looks at them, a lane a token
    if (tid == t) {
        sums[0] = sh.part + (upto - here_sum);
#pragma unroll
        for (int j = 0; j < 4; ++j) *reinterpret_cast<float4_t *>(values + 4 * j) = f[j];
    }
    __syncthreads();
    if (wave == 0 && t >= 0) {
        const double w = lane >= per ? 0. : filtered ? of(values[lane & 15], c * p.chunk + t * per + lane, exactly) : unfiltered(values[lane & 15]), run = sums[0] + wave_scan(w);
        const unsigned long long any = __ballot(w > 0.), hit = __ballot(w > 0. && run > goal);
        const int l = hit ? __ffsll((long long)hit) - 1 : 63 - __clzll((long long)any);      // (sums in another order may end a rounding below the goal: the last one)
        if (lane == 0) sh.found = c * p.chunk + t * per + l;
    }
    __syncthreads();
    if (tid == 0) {
        const int id = t < 0 ? -1 : sh.found;
        p.a.ids[row] = id;
        if (p.a.logprobs) p.a.logprobs[row] = id < 0 ? -INFINITY : (float)log(weight(seen(r.x[id]), r.m, ask.c) / sum);
    }
}

// Tokens of a chunk.  Each has its bins and lists, which the second launch reads: large ones where there would be many, and for many rows that are one.  us with 4096 and 16384, settings mixed: 256 rows of
// 151936 137 114, 40 74 66, 256 of 131072 114 101, 32 45 44, 8 38 41; 256 of 65536 73 73, 128 57 62, 256 of 32768 61 64, 198 of 20570 59 78; 135 of 9398 52 42, 256 of 5000 48 42.  One row of 151936 with
// top-k 20 15.9 15.1, top-k 1000 42 36, top-p 0.8 37 40, unfiltered 16 21 (the walk over the drawn chunk: the rule goes by the vocabulary there, and such rows pay for it); of 32000: 14 15, 36 42, 15 20,
// 14 21
// (the limits stand in sample_uniform_workspace_bytes too)
static int sample_chunk(int64_t B, int64_t V) { return V > 98304 || (V <= 16384 && B >= 128) ? 16384 : 4096; }
// Enough for fewer rows and smaller vocabularies too, whose chunks may be smaller and more: the most there are on either side of the rule's limits
size_t sample_uniform_workspace_bytes(int64_t B, int64_t V) {
    if (B <= 0 || V <= 0) return 0;
    int64_t most = 0;
    for (int64_t b : {B, std::min<int64_t>(B, 127)})
        for (int64_t v : {V, std::min<int64_t>(V, 98304), std::min<int64_t>(V, 16384)}) most = std::max(most, b * ((v + sample_chunk(b, v) - 1) / sample_chunk(b, v)));
    return (size_t)most * (kBins * 12 + kNear * 8 + sizeof(ChunkNote));
}
int sample_uniform(const SampleArgs &a, hipStream_t s) {
    if (a.B < 0 || a.V <= 0 || a.ld < a.V) return nvr::fail(NVR_ERR_INVALID_ARG, "nvr_sample_uniform: B=%ld V=%ld, rows %ld apart", (long)a.B, (long)a.V, (long)a.ld);
    if (a.V > (1 << 22) || a.B > 65535) return nvr::fail(NVR_ERR_UNSUPPORTED, "nvr_sample_uniform: up to 65535 rows of up to 2^22 logits (B=%ld V=%ld)", (long)a.B, (long)a.V);
    if (a.B == 0) return 0;
    if (!a.logits || !a.uniform || !a.ids || !a.workspace) return nvr::fail(NVR_ERR_INVALID_ARG, "nvr_sample_uniform: null argument");
    if (((uintptr_t)a.workspace & 15) != 0) return nvr::fail(NVR_ERR_INVALID_ARG, "nvr_sample_uniform: the workspace is not aligned to 16 bytes");
    SampleParams p{};
    p.a = a; p.V = (int32_t)a.V; p.chunk = sample_chunk(a.B, a.V); p.P = (int32_t)((a.V + p.chunk - 1) / p.chunk);
    const int64_t n = a.B * p.P;
    p.mass = (unsigned long long *)a.workspace; p.near = (uint2 *)(p.mass + n * kBins); p.cnt = (unsigned int *)(p.near + n * kNear); p.notes = (ChunkNote *)(p.cnt + n * kBins);
    p.whole = ((uintptr_t)a.logits & 15) == 0 && a.ld % 4 == 0;
    const dim3 grid((unsigned)p.P, (unsigned)a.B);
    if (p.chunk == 4096) sample_scan_kernel<8, 512><<<grid, 512, 0, s>>>(p);
    else sample_scan_kernel<16, 1024><<<grid, 1024, 0, s>>>(p);
    sample_pick_kernel<<<dim3((unsigned)a.B), kPick, 0, s>>>(p);
    NVR_KX_LAUNCHED("sample_uniform");
    return 0;
}

}}  // namespace nvr::kx
