// sample_uniform.hip — a token for each row of logits from the row's own uniform number: temperature, then top-k, top-p and min-p, then the first token
// (in the order of the vocabulary) whose summed weight exceeds uniform * (sum of what is left).
//
// With m the row's largest logit, token i has the weight w_i = exp((x_i - m) / T).  All three filters keep a prefix of the tokens in descending order (ties: ascending index), so a row's
// answer is decided by two numbers: where the prefix ends, and the sum of its weights.  Nothing is sorted: the first launch reads the logits once and leaves, for each chunk of a row, its
// maximum and the weights (and, for top-k, tokens) in bins of 1/24 of (x - m) / T; the second, a workgroup a row, adds the chunks' bins up, finds the bin that each filter ends in, reads the
// chunks that have tokens there, settles the order inside the bin by a radix select over (logit, index), finds the chunk that the drawn number falls into, and walks that one.
// A token's index is an answer that has to be right to the last bit, so weights are 64-bit numbers (exp by a polynomial of degree 10, 2e-13 off) and are summed as integers of
// 2^-44 and less of the largest: their order, hence the atomics', changes nothing.  Tokens more than 42 T below the largest (e^-42 = 4e-19 of its weight) are left out.
#include <algorithm>
#include "serving.h"
#include "device_utils.h"
#include "../common.h"
#include "elem.h"

namespace nvr { namespace kx {

namespace {
constexpr int kBins = 1024, kScan = 512, kPick = 1024, kList = 3072, kRadix = 2048;
constexpr float kPerUnit = 24.f;                                          // bins to a unit of (x - m) / T

struct ChunkNote { float max; int32_t arg; };                             // arg: first index of the maximum (greedy rows)
struct SampleParams {
    SampleArgs a;
    int32_t V, P, chunk, bits;                                            // chunks of a row, their tokens; weights are integers of 2^-bits
    ChunkNote *notes; unsigned long long *mass; unsigned int *cnt;        // [B][P], [B][P][kBins] twice
    bool whole;                                                           // rows in 16-byte pieces
};
// What a row asks for.  T of 0 (or less, or not a number, or too small to divide by): the largest logit
struct RowAsk { float T, inv; double c; bool greedy; long long k; float p, min_p; };
__device__ __forceinline__ RowAsk row_ask(const SampleArgs &a, int row, int V) {
    RowAsk r;
    r.T = a.temperature ? a.temperature[row] : 1.f;
    r.inv = kPerUnit / r.T;
    r.greedy = !(r.T > 0.f) || r.inv > 1e30f;
    r.c = 1.4426950408889634 / (double)r.T;
    r.k = a.top_k ? a.top_k[row] : 0;
    if (r.k <= 0 || r.k >= V) r.k = 0;
    r.p = a.top_p ? a.top_p[row] : 1.f;
    if (!(r.p >= 0.f && r.p < 1.f)) r.p = 1.f;
    r.min_p = a.min_p ? a.min_p[row] : 0.f;
    r.min_p = r.min_p > 0.f ? fminf(r.min_p, 1.f) : 0.f;
    return r;
}
__device__ __forceinline__ float seen(float x) { return x == x ? x : -INFINITY; }        // (not a number: never chosen)
// 2^t for t <= 0: the series of exp(r ln 2), |r| <= 1/2
__device__ __forceinline__ double exp2_64(double t) {
    if (!(t > -1000.)) return 0.;
    const double n = rint(t), r = t - n;
    double s = 7.0549116208011233e-9;                                     // ln(2)^k / k!
    s = fma(s, r, 1.0178086009239699e-7); s = fma(s, r, 1.3215486790144309e-6); s = fma(s, r, 1.5252733804059840e-5); s = fma(s, r, 1.5403530393381610e-4);
    s = fma(s, r, 1.3333558146428443e-3); s = fma(s, r, 9.6181291076284771e-3); s = fma(s, r, 5.5504108664821580e-2); s = fma(s, r, 2.4022650695910071e-1);
    s = fma(s, r, 6.9314718055994531e-1); s = fma(s, r, 1.0);
    return ldexp(s, (int)n);
}
__device__ __forceinline__ double weight(float x, float m, double c) { return x == m ? 1.0 : exp2_64(((double)x - (double)m) * c); }
// bin of x below the maximum m: monotone in x; kBins - 1 and beyond: left out.  Whole numbers throughout, so bins under a chunk's maximum are a shift away from those under the row's
__device__ __forceinline__ float cell(float x, float inv) { return floorf(x * inv); }
__device__ __forceinline__ int bin_of(float x, float m, float inv) {
    if (x == m) return 0;
    const float d = cell(m, inv) - cell(x, inv);
    return d < (float)(kBins - 1) ? (int)d : kBins - 1;
}
__device__ __forceinline__ unsigned int key_of(float f) { const unsigned int u = __float_as_uint(f); return (u & 0x80000000u) ? ~u : (u | 0x80000000u); }
__device__ __forceinline__ float of_key(unsigned int k) { return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k); }

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
}  // namespace

// A chunk of EPT tokens a thread, held in registers: its maximum, then its bins
template <int EPT>
__global__ __launch_bounds__(kScan) void sample_scan_kernel(SampleParams p) {
    __shared__ unsigned long long mass[kBins];
    __shared__ unsigned int cnt[kBins];
    __shared__ float wmax[kScan / 64];
    __shared__ int warg[kScan / 64];
    const int c = blockIdx.x, row = blockIdx.y, tid = threadIdx.x, wave = tid >> 6;
    const float *x = p.a.logits + (int64_t)row * p.a.ld;
    const int base = c * p.chunk, end = min(p.V, base + p.chunk);
    float v[EPT];
#pragma unroll
    for (int j = 0; j < EPT / 4; ++j) {
        const float4_t f = four(x, base + (j * kScan + tid) * 4, end, p.whole);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[4 * j + e] = f[e];
    }
    const RowAsk ask = row_ask(p.a, row, p.V);
    for (int b = tid; b < kBins; b += kScan) { mass[b] = 0; cnt[b] = 0; }
    float m = v[0];
#pragma unroll
    for (int j = 1; j < EPT; ++j) m = fmaxf(m, v[j]);
    m = wave_max(m);
    if ((tid & 63) == 0) wmax[wave] = m;
    __syncthreads();
    m = wmax[0];
#pragma unroll
    for (int w = 1; w < kScan / 64; ++w) m = fmaxf(m, wmax[w]);
    ChunkNote *note = p.notes + (int64_t)row * p.P + c;
    if (ask.greedy) {
        int at = 0x7fffffff;
#pragma unroll
        for (int j = EPT - 1; j >= 0; --j) if (v[j] == m) at = base + ((j / 4) * kScan + tid) * 4 + (j & 3);
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) at = min(at, __shfl_xor(at, o));
        if ((tid & 63) == 0) warg[wave] = at;
        __syncthreads();
        if (tid == 0) {
#pragma unroll
            for (int w = 1; w < kScan / 64; ++w) at = min(at, warg[w]);
            *note = ChunkNote{m, at};
        }
        return;
    }
    if (tid == 0) *note = ChunkNote{m, 0};
    if (m == -INFINITY) return;                                           // (nothing to choose here: the bins are not looked at)
    const double one = ldexp(1.0, p.bits);
    const bool counted = ask.k > 0;
#pragma unroll
    for (int j = 0; j < EPT; ++j) {
        if (v[j] == -INFINITY) continue;
        const int b = bin_of(v[j], m, ask.inv);
        if (b >= kBins - 1) continue;
        atomicAdd(&mass[b], (unsigned long long)(weight(v[j], m, ask.c) * one + 0.5));
        if (counted) atomicAdd(&cnt[b], 1u);
    }
    __syncthreads();
    const int64_t at = ((int64_t)row * p.P + c) * kBins;
    for (int b = tid; b < kBins; b += kScan) { p.mass[at + b] = mass[b]; if (counted) p.cnt[at + b] = cnt[b]; }
}

namespace {
struct PickShared {
    double cum[kBins];                                                    // weight of the bins up to and with this one
    unsigned int cum_n[kBins];
    unsigned long long rmass[kRadix];
    unsigned int rcnt[kRadix];
    unsigned int key[kList], idx[kList];
    double wsum[16];
    unsigned long long wsum64[16];
    unsigned int wcnt[16];
    unsigned int n, nsel;
    int sel, found;
    unsigned int sel_cnt;
    unsigned long long sel_mass;
    double part;
};
template <class T>
__device__ __forceinline__ T up(T v, int d) { return __shfl_up(v, d); }
// sum over the threads up to and with this one; `waves`: 16 of LDS
template <class T>
__device__ __forceinline__ T scan(T v, T *waves) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) { const T o = up(v, d); if (lane >= d) v += o; }
    __syncthreads();
    if (lane == 63) waves[wave] = v;
    __syncthreads();
    T before = 0;
    for (int w = 0; w < wave; ++w) before += waves[w];
    return before + v;
}

struct Row {
    const SampleParams &p;
    PickShared &sh;
    const float *x;
    int row;
    RowAsk ask;
    float m;
    double one;
    __device__ int shift(int c) const {                                   // bins of chunk c lie this far under the row's (kBins: nothing of it is near)
        const float mc = p.notes[(int64_t)row * p.P + c].max;
        if (mc == -INFINITY) return kBins;
        return bin_of(mc, m, ask.inv) >= kBins - 1 ? kBins : bin_of(mc, m, ask.inv);
    }
    __device__ double factor(int c) const { return weight(p.notes[(int64_t)row * p.P + c].max, m, ask.c) / one; }
    __device__ const unsigned long long *mass(int c) const { return p.mass + ((int64_t)row * p.P + c) * kBins; }
    // f(key, index, x) for the tokens of bins lo .. hi: all threads take part
    template <class F>
    __device__ void each_of_row(int lo, int hi, F f) const {
        for (int c = 0; c < p.P; ++c) {
            const int s = shift(c);
            if (s > hi) continue;
            each_of_chunk(c, lo, hi, f);
        }
    }
    template <class F>
    __device__ void each_of_chunk(int c, int lo, int hi, F f) const {
        const int base = c * p.chunk, end = min(p.V, base + p.chunk);
        for (int i = base + (int)threadIdx.x * 4; i < base + p.chunk; i += kPick * 4) {
            const float4_t v = four(x, i, end, p.whole);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (v[e] == -INFINITY) continue;
                const int b = bin_of(v[e], m, ask.inv);
                if (b >= lo && b <= hi && b < kBins - 1) f(key_of(v[e]), (unsigned int)(i + e), v[e]);
            }
        }
    }
    // the tokens of bins lo .. hi into the list; false: they are more than it holds
    __device__ bool gather(int lo, int hi) {
        if (threadIdx.x == 0) sh.n = 0;
        __syncthreads();
        for (int c = 0; c < p.P; ++c) {
            const int s = shift(c);
            if (s > hi) continue;
            const unsigned long long *q = mass(c);
            bool some = false;                                            // (the same for every thread)
            for (int b = max(lo - s, 0); b <= hi - s && !some; ++b) some = q[b] != 0;
            if (!some) continue;
            each_of_chunk(c, lo, hi, [&](unsigned int k, unsigned int i, float) {
                const unsigned int at = atomicAdd(&sh.n, 1u);
                if (at < kList) { sh.key[at] = k; sh.idx[at] = i; }
            });
        }
        __syncthreads();
        return sh.n <= kList;
    }
    template <class F>
    __device__ void each(bool listed, int lo, int hi, F f) {
        if (listed) { for (unsigned int i = threadIdx.x; i < sh.n; i += kPick) f(sh.key[i], sh.idx[i], of_key(sh.key[i])); }
        else each_of_row(lo, hi, f);
    }
    // Among the tokens of bin b in descending order (ties: ascending index): the last one that is kept, when `need` of them are (need > 0) or as many as it takes until `before` plus their weights
    // reaches `goal`.  part: the weight of the kept ones
    __device__ void settle(int b, unsigned int need, double before, double goal, unsigned int &key, unsigned int &index, double &part) {
        const bool listed = gather(b, b);
        const int tid = threadIdx.x;
        unsigned int prefix = 0, mask = 0, left = need;
        unsigned long long done = 0;                                      // weight above the prefix
        unsigned int equal = 0;
        for (int pass = 0; pass < 3; ++pass) {
            const int at = pass == 0 ? 21 : pass == 1 ? 10 : 0, wide = pass == 2 ? 1024 : 2048;
            for (int i = tid; i < kRadix; i += kPick) { sh.rcnt[i] = 0; sh.rmass[i] = 0; }
            if (tid == 0) sh.found = 0x7fffffff;
            __syncthreads();
            each(listed, b, b, [&](unsigned int k, unsigned int, float v) {
                if ((k & mask) != prefix) return;
                const int d = wide - 1 - (int)((k >> at) & (wide - 1));   // descending
                atomicAdd(&sh.rcnt[d], 1u);
                atomicAdd(&sh.rmass[d], (unsigned long long)(weight(v, m, ask.c) * one + 0.5));
            });
            __syncthreads();
            const unsigned int c0 = sh.rcnt[2 * tid], c1 = sh.rcnt[2 * tid + 1];
            const unsigned long long m0 = sh.rmass[2 * tid], m1 = sh.rmass[2 * tid + 1];
            const unsigned int nc = scan<unsigned int>(c0 + c1, sh.wcnt);
            const unsigned long long nm = scan<unsigned long long>(m0 + m1, sh.wsum64);
            // the first digit that the end falls into (or, where rounding leaves the goal unreached, the last that has tokens)
            const unsigned int u1 = nc, u0 = nc - c1;
            const unsigned long long s1 = nm, s0 = nm - m1;
            auto ends = [&](unsigned int n, unsigned long long s) { return need ? n >= left : before + (double)(done + s) / one >= goal; };
            if (c0 && ends(u0, s0)) atomicMin(&sh.found, 2 * tid);
            else if (c1 && ends(u1, s1)) atomicMin(&sh.found, 2 * tid + 1);
            if (tid == 0) sh.sel = -1;
            __syncthreads();
            if (sh.found == 0x7fffffff) { if (c1) atomicMax(&sh.sel, 2 * tid + 1); else if (c0) atomicMax(&sh.sel, 2 * tid); }
            __syncthreads();
            const int d = sh.found != 0x7fffffff ? sh.found : sh.sel;
            if (d < 0) { key = 0; index = 0xffffffffu; part = 0.; __syncthreads(); return; }        // (no token: everything is kept)
            if (tid == d / 2) {
                const bool odd = d & 1;
                sh.sel_cnt = odd ? u0 : u0 - c0; sh.sel_mass = odd ? s0 : s0 - m0;
                sh.nsel = odd ? c1 : c0;
            }
            __syncthreads();
            if (need) left -= min(left, sh.sel_cnt);
            done += sh.sel_mass;
            equal = sh.nsel;
            prefix |= (unsigned int)(wide - 1 - d) << at; mask |= (unsigned int)(wide - 1) << at;
            __syncthreads();
        }
        key = prefix;
        const double w = weight(of_key(prefix), m, ask.c);
        unsigned int n = left;
        const double start = before + (double)done / one;
        if (!need) {
            const double q = w > 0. ? ceil((goal - start) / w) : 1.;
            n = q >= (double)equal ? equal : q < 1. ? 1u : (unsigned int)q;
            if (n > 1 && start + (n - 1) * w >= goal) --n;
            else if (n < equal && start + n * w < goal) ++n;
        }
        if (n < 1) n = 1;
        if (n > equal) n = equal;
        part = (double)done / one + n * w;
        index = 0xffffffffu;
        if (n == equal) return;
        // which of the equal ones: the n-th smallest index
        unsigned int at_prefix = 0, at_mask = 0, want = n;
        for (int at = 22; at >= 0; at -= 11) {
            for (int i = tid; i < kRadix; i += kPick) sh.rcnt[i] = 0;
            if (tid == 0) sh.found = 0x7fffffff;
            __syncthreads();
            each(listed, b, b, [&](unsigned int k, unsigned int i, float) { if (k == key && (i & at_mask) == at_prefix) atomicAdd(&sh.rcnt[(i >> at) & (kRadix - 1)], 1u); });
            __syncthreads();
            const unsigned int c0 = sh.rcnt[2 * tid], c1 = sh.rcnt[2 * tid + 1], nc = scan<unsigned int>(c0 + c1, sh.wcnt);
            if (c0 && nc - c1 >= want) atomicMin(&sh.found, 2 * tid);
            else if (c1 && nc >= want) atomicMin(&sh.found, 2 * tid + 1);
            __syncthreads();
            const int d = sh.found;
            if (tid == d / 2) sh.sel_cnt = (d & 1) ? nc - c1 : nc - c1 - c0;
            __syncthreads();
            want -= sh.sel_cnt;
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
    Row r{p, sh, p.a.logits + (int64_t)row * p.a.ld, row, row_ask(p.a, row, p.V), -INFINITY, ldexp(1.0, p.bits)};
    for (int c = 0; c < p.P; ++c) r.m = fmaxf(r.m, notes[c].max);
    if (r.m == -INFINITY || r.ask.greedy) {
        if (tid == 0) {
            int64_t id = -1;
            for (int c = p.P - 1; c >= 0 && r.m != -INFINITY; --c) if (notes[c].max == r.m) id = notes[c].arg;
            p.a.ids[row] = id;
            if (p.a.logprobs) p.a.logprobs[row] = id < 0 ? -INFINITY : 0.f;
        }
        return;
    }
    const RowAsk &ask = r.ask;
    // ---- the row's bins, thread b bin b
    double mass = 0.;
    unsigned int cnt = 0;
    for (int c = 0; c < p.P; ++c) {
        const int s = r.shift(c);
        if (tid >= s && tid - s < kBins - 1 && tid < kBins - 1) {
            mass += (double)r.mass(c)[tid - s] * r.factor(c);
            if (ask.k) cnt += p.cnt[((int64_t)row * p.P + c) * kBins + tid - s];
        }
    }
    sh.cum[tid] = scan<double>(mass, sh.wsum);
    sh.cum_n[tid] = ask.k ? scan<unsigned int>(cnt, sh.wcnt) : 0;
    __syncthreads();
    // the first bin whose sum reaches a goal (kBins: none)
    auto first_bin = [&](bool reached) {
        if (tid == 0) sh.found = kBins;
        __syncthreads();
        if (reached) atomicMin(&sh.found, tid);
        __syncthreads();
        const int b = sh.found;
        __syncthreads();
        return b;
    };
    int stop = kBins;                                                     // bins in front of it are kept whole; of this one, tokens down to (key, index)
    unsigned int key = 0, index = 0xffffffffu;
    double total = sh.cum[kBins - 1];
    if (ask.k) {
        const int b = first_bin(sh.cum_n[tid] >= (unsigned int)ask.k);
        if (b < kBins) {
            const unsigned int before = b ? sh.cum_n[b - 1] : 0;
            const double mass_before = b ? sh.cum[b - 1] : 0.;
            if (sh.cum_n[b] == (unsigned int)ask.k) { stop = b + 1; total = sh.cum[b]; }
            else {
                double part;
                r.settle(b, (unsigned int)ask.k - before, 0., 0., key, index, part);
                stop = b; total = mass_before + part;
            }
        }
    }
    if (ask.p < 1.f) {
        const double goal = (double)ask.p * total;
        const int b = first_bin(sh.cum[tid] >= goal && sh.cum[tid] > 0. && (tid < stop || (tid == stop && stop < kBins)));
        const bool ends_there = b < kBins && !(b == stop && total < goal);
        if (ends_there && b <= stop) {
            unsigned int k2, i2;
            double part;
            const double before = b ? sh.cum[b - 1] : 0.;
            r.settle(b, 0, before, goal, k2, i2, part);
            // (in the bin where top-k ended, its own end may come first)
            if (b < stop || k2 > key || (k2 == key && i2 < index)) { key = k2; index = i2; }
            stop = b;
        }
    }
    // ---- min-p: tokens of weight min_p and more, by bins but for those around the border
    int sure = stop, last = stop < kBins ? stop : -1;                     // whole bins in front of `sure`; single tokens of bins sure .. last
    bool by_key = stop < kBins && !(key == 0 && index == 0xffffffffu);
    if (stop < kBins && !by_key) last = stop - 1;                         // (top-k ended with a whole bin: `stop` is the first one left out)
    const int key_bin = stop;
    if (ask.min_p > 0.f) {
        const float edge = (float)((double)r.m + (double)ask.T * log((double)ask.min_p)), off = 1e-6f * fmaxf(fabsf(r.m), fabsf(edge));      // off: what rounding may move it by
        const bool far = r.m == INFINITY;
        const int lo = far ? 0 : max(bin_of(fminf(edge + off, r.m), r.m, ask.inv) - 1, 0), hi = far ? 0 : min(bin_of(edge - off, r.m, ask.inv) + 1, kBins - 2);
        if (lo < sure) { last = by_key && key_bin <= hi ? key_bin : min(hi, sure - 1); sure = lo; }
    }
    auto kept = [&](int b, unsigned int k, unsigned int i, double w) {
        if (b < sure) return true;
        if (b > last) return false;
        if (by_key && b == key_bin && (k < key || (k == key && i > index))) return false;
        return !(ask.min_p > 0.f) || w >= (double)ask.min_p;
    };
    // ---- what each chunk keeps: its whole bins, a wave a chunk, and its single tokens
    double sum = 0.;                                                      // of the chunks so far
    const double u = p.a.uniform ? (double)p.a.uniform[row] : 0.;
    auto chunk_sum = [&](int c) {                                         // (a wave)
        const int s = r.shift(c);
        double v = 0.;
        if (s < kBins) {
            const unsigned long long *q = r.mass(c);
            for (int b = lane; b < sure - s && b < kBins - 1; b += 64) v += (double)q[b];
            v *= r.factor(c);
            if (last >= sure && s <= last) {
                bool some = false;
                for (int b = max(sure - s, 0); b <= last - s && !some; ++b) some = q[b] != 0;
                if (some) {
                    const int base = c * p.chunk, end = min(p.V, base + p.chunk);
                    for (int i = base + lane * 4; i < base + p.chunk; i += 256) {
                        const float4_t f = four(r.x, i, end, p.whole);
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            if (f[e] == -INFINITY) continue;
                            const int b = bin_of(f[e], r.m, ask.inv);
                            if (b < sure || b > last) continue;
                            const double w = weight(f[e], r.m, ask.c);
                            if (kept(b, key_of(f[e]), (unsigned int)(i + e), w)) v += w;
                        }
                    }
                }
            }
        }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
        return v;
    };
    // two walks over the chunks' sums, 16 at a time: the row's sum, then the chunk that the goal falls into.  The sums of up to kList chunks stay in LDS (a row has more only beyond 12 million tokens)
    double *sums = reinterpret_cast<double *>(sh.rmass);                  // (free by now: kRadix of them)
    __syncthreads();
    for (int c0 = 0; c0 < p.P; c0 += 16) {
        const int c = c0 + wave;
        if (c < p.P) { const double v = chunk_sum(c); if (lane == 0) sums[c] = v; }
    }
    __syncthreads();
    for (int c = 0; c < p.P; ++c) sum += sums[c];
    const double goal = u * sum;
    double before = 0.;
    int at = -1;
    {
        double run = 0.;
        int lastc = -1;
        double lastb = 0.;
        for (int c = 0; c < p.P; ++c) {
            if (sums[c] > 0.) { lastc = c; lastb = run; }
            if (at < 0 && run + sums[c] > goal) { at = c; before = run; }
            run += sums[c];
        }
        if (at < 0) { at = lastc; before = lastb; }
    }
    // ---- the token of that chunk: a thread's tokens are neighbours
    const int per = p.chunk / kPick, base = at * p.chunk, end = min(p.V, base + p.chunk);      // 4 or 16
    double w[16];
    double mine = 0.;
    for (int j = 0; j < 16; j += 4) {
        if (j >= per) break;
        const int i = base + tid * per + j;
        const float4_t f = four(r.x, i, end, p.whole);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            double v = 0.;
            if (f[e] != -INFINITY) {
                const int b = bin_of(f[e], r.m, ask.inv);
                if (b < kBins - 1 && (b < sure || b <= last)) { v = weight(f[e], r.m, ask.c); if (!kept(b, key_of(f[e]), (unsigned int)(i + e), v)) v = 0.; }
            }
            w[j + e] = v; mine += v;
        }
    }
    const double upto = scan<double>(mine, sh.wsum);
    if (tid == 0) { sh.found = 0x7fffffff; sh.sel = -1; }
    __syncthreads();
    {
        double run = before + upto - mine;
        int hit = -1, any = -1;
        for (int j = 0; j < 16; ++j) {
            if (j >= per) break;
            run += w[j];
            if (w[j] > 0.) { any = j; if (hit < 0 && run > goal) hit = j; }
        }
        if (hit >= 0) atomicMin(&sh.found, base + tid * per + hit);
        if (any >= 0) atomicMax(&sh.sel, base + tid * per + any);
    }
    __syncthreads();
    if (tid == 0) {
        const int id = sh.found != 0x7fffffff ? sh.found : sh.sel;         // (the sums of the chunk in another order may end a rounding below the goal: its last token)
        p.a.ids[row] = id;
        if (p.a.logprobs) p.a.logprobs[row] = id < 0 ? -INFINITY : (float)log(weight(seen(r.x[id]), r.m, ask.c) / sum);
    }
}

static int sample_chunk(int64_t B, int64_t V) { return B * ((V + 16383) / 16384) >= 256 ? 16384 : 4096; }   // tokens of a chunk: 12 KB of bins each, so larger ones once they fill the chip
size_t sample_uniform_workspace_bytes(int64_t B, int64_t V) {
    if (B <= 0 || V <= 0) return 0;
    const int64_t P = (V + sample_chunk(B, V) - 1) / sample_chunk(B, V);
    return (size_t)(B * P) * (kBins * 12 + sizeof(ChunkNote));
}
int sample_uniform(const SampleArgs &a, hipStream_t s) {
    if (a.B < 0 || a.V <= 0 || a.ld < a.V) return nvr::fail(NVR_ERR_INVALID_ARG, "nvr_sample_uniform: B=%ld V=%ld, rows %ld apart", (long)a.B, (long)a.V, (long)a.ld);
    if (a.V > (1 << 22) || a.B > 65535) return nvr::fail(NVR_ERR_UNSUPPORTED, "nvr_sample_uniform: up to 65535 rows of up to 2^22 logits (B=%ld V=%ld)", (long)a.B, (long)a.V);
    if (a.B == 0) return 0;
    if (!a.logits || !a.uniform || !a.ids || !a.workspace) return nvr::fail(NVR_ERR_INVALID_ARG, "nvr_sample_uniform: null argument");
    if (((uintptr_t)a.workspace & 15) != 0) return nvr::fail(NVR_ERR_INVALID_ARG, "nvr_sample_uniform: the workspace is not aligned to 16 bytes");
    SampleParams p{};
    p.a = a; p.V = (int32_t)a.V; p.chunk = sample_chunk(a.B, a.V); p.P = (int32_t)((a.V + p.chunk - 1) / p.chunk);
    int log2v = 0;
    while ((1ll << log2v) < a.V) ++log2v;
    p.bits = 62 - log2v;
    const int64_t n = a.B * p.P;
    p.mass = (unsigned long long *)a.workspace; p.cnt = (unsigned int *)(p.mass + n * kBins); p.notes = (ChunkNote *)(p.cnt + n * kBins);
    p.whole = ((uintptr_t)a.logits & 15) == 0 && a.ld % 4 == 0;
    const dim3 grid((unsigned)p.P, (unsigned)a.B);
    if (p.chunk == 4096) sample_scan_kernel<8><<<grid, kScan, 0, s>>>(p);
    else sample_scan_kernel<32><<<grid, kScan, 0, s>>>(p);
    sample_pick_kernel<<<dim3((unsigned)a.B), kPick, 0, s>>>(p);
    NVR_KX_LAUNCHED("sample_uniform");
    return 0;
}

}}  // namespace nvr::kx
