// lora.hip — low-rank adapters of many requests beside a shared projection: y[t] = base[t] + scale_a (x[t] A_a^T) B_a^T, a = the adapter of row t's request.
//
// Two products of inner sizes K and R, on the matrix cores, over TILES: up to 16 or 64 rows that share an adapter, wherever they stand in the step (up to 64 rows every wave finds its tile
// itself, up to 1024 every workgroup; more are grouped by a launch of their own).  An adapter is so read once per tile and its rows cost no more than they are.
//   down: v = scale x A^T, the waves of a workgroup (and `splits` workgroups of few rows) share K; partial sums stay in 32 bits in the workspace, [split][row][rank]
//   up:   y = base + v B^T; v in two 16-bit numbers (its rounding and the rounded rest), so that the product sees it in 16 (bfloat16) or 22 bits; the sum with base is rounded once
// Few rows of few ranks take one launch, in which every workgroup finds its tile and forms v anew for its columns.
// Bound by memory for prompts (x, base and y once; 2 R flops a byte), by launches and a chain of round trips for decode steps.  bfloat16, 8192 rows 4096 -> 12288 of rank 32: 122 us (grouping 8, down
// 24, up 91: 402 MB of base and y at 4.4 TB/s); float16, 251 rows 4096 -> 4096 of rank 64 over 7 adapters: 15 us; 32 rows 1024 -> 2048 of rank 16 over 32: 5.3 us in one launch.  float32: 253, 19 and 9 us.
#include <algorithm>
#include <type_traits>
#include "serving.h"
#include "elem.h"
#include "scan.h"
#include "../common.h"

namespace nvr { namespace kx {

namespace {
constexpr int kSmall = 64;                                                // rows up to which a workgroup finds its tile itself (64 x 1024 -> 2048 of rank 64: 11.1 us, grouped by a launch 12.9)
constexpr int kMany = 1024;                                               // ... counts the adapters' rows for it
constexpr int kMaxAdapters = 8192;                                        // counters of the grouping launch (LDS)

struct LoraTile { int32_t start, count, adapter; };                       // rows order[start ..) of one adapter; adapter n: rows without one
struct LoraParams {
    LoraArgs a;
    int32_t splits, rp, copies;                                           // copies: rows without an adapter are tiles too (base is another tensor)
    const int32_t *order; const LoraTile *tiles; const int32_t *num_tiles;
    float *v;                                                             // [splits][T][rp]
    bool xw, aw, bw, yw;                                                  // whole 16-byte pieces of x, A, B and base / y
};

__device__ __forceinline__ int adapter_of(const LoraParams &p, int64_t t) {
    const int id = p.a.ids[t];
    return id >= 0 && id < (int)p.a.n ? id : p.copies ? (int)p.a.n : -1;
}

// float16: v may be beyond its range, or far below it, so each row of v is multiplied by the power of two that brings its largest number to 2^13 .. 2^14 (exponents of -100 .. 100)
__device__ __forceinline__ int range_of(unsigned int most) {
    const int e = (int)(most >> 23) - 127;
    return most == 0 || e == 128 ? 0 : min(max(13 - e, -100), 100);
}

// rows of tile `tile` (rows[0 .. count), LDS) and its adapter; count 0: no such tile.  T <= 64, tiles of 16 rows: row t is number rank(t) of its adapter's rows, the rows of rank 0, 16, .. lead a tile,
// tiles go by their leaders.  Every wave for itself, a lane a row (all write the same)
__device__ __forceinline__ int tile_of_small(const LoraParams &p, int tile, int *rows, int &adapter) {
    const int lane = threadIdx.x & 63, id = lane < (int)p.a.T ? adapter_of(p, lane) : -1;
    int rank = 0;
    for (int j0 = 0; j0 < (int)p.a.T; j0 += 8)
#pragma unroll
        for (int j = j0; j < j0 + 8; ++j) rank += __builtin_amdgcn_readlane(id, j) == id && j < lane;      // (T <= 64: j < 64)
    const unsigned long long leads = __ballot(id >= 0 && (rank & 15) == 0);
    const unsigned long long mine = __ballot(((leads >> lane) & 1) && __popcll(leads & ((1ull << lane) - 1)) == tile);
    if (!mine) return 0;
    const int leader = __ffsll((long long)mine) - 1, first = __builtin_amdgcn_readlane(rank, leader);
    adapter = __builtin_amdgcn_readlane(id, leader);
    const bool in = id == adapter && rank >= first && rank < first + 16;
    if (in) rows[rank - first] = lane;
    return __popcll(__ballot(in));
}
// how a workgroup learns of its tile
enum Find { SMALL, MANY, GROUPED };
// rows of tile `tile` (16 rows), as tile_of_small, of up to kMany rows and fewer than 1024 adapters: a workgroup counts each adapter's rows, and the rows of the tile's adapter in their order
template <int THREADS>
__device__ __forceinline__ int tile_of_many(const LoraParams &p, int tile, int *rows, int &adapter) {
    constexpr int PER = kMany / THREADS, OWN = 1024 / THREADS;            // rows and adapters of a thread
    __shared__ int cnt[1024], waves[16], chosen[2];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, T = (int)p.a.T;
    int id[PER];
#pragma unroll
    for (int e = 0; e < PER; ++e) id[e] = e * THREADS + tid < T ? adapter_of(p, e * THREADS + tid) : -1;
#pragma unroll
    for (int e = 0; e < OWN; ++e) cnt[OWN * tid + e] = 0;
    if (tid == 0) chosen[0] = -1;
    __syncthreads();
#pragma unroll
    for (int e = 0; e < PER; ++e) if (id[e] >= 0) atomicAdd(&cnt[id[e]], 1);
    __syncthreads();
    int own = 0;
#pragma unroll
    for (int e = 0; e < OWN; ++e) own += (cnt[OWN * tid + e] + 15) / 16;
    const int upto = scan<int>(own, waves);
    int from = upto - own;
    if (from <= tile && tile < upto) {                                    // (one thread)
        int i = OWN * tid;
        for (int t; from + (t = (cnt[i] + 15) / 16) <= tile; ++i) from += t;
        chosen[0] = i; chosen[1] = (tile - from) * 16;
    }
    __syncthreads();
    if (chosen[0] < 0) return 0;
    adapter = same(chosen[0]);
    const int first = same(chosen[1]), count = same(min(16, cnt[adapter] - first));
    unsigned long long mine[PER];
#pragma unroll
    for (int e = 0; e < PER; ++e) {
        mine[e] = __ballot(id[e] == adapter);
        if (lane == 0) waves[e * (THREADS / 64) + wave] = __popcll(mine[e]);
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < PER; ++e) {
        int rank = __popcll(mine[e] & ((1ull << lane) - 1)) - first;
        for (int w = 0; w < e * (THREADS / 64) + wave; ++w) rank += waves[w];
        if (id[e] == adapter && rank >= 0 && rank < 16) rows[rank] = e * THREADS + tid;
    }
    __syncthreads();
    return count;
}

template <int TR, Find FIND, int THREADS>
__device__ __forceinline__ int tile_rows(const LoraParams &p, int tile, int *rows, int &adapter) {
    if constexpr (FIND == SMALL) return tile_of_small(p, tile, rows, adapter);
    if constexpr (FIND == MANY) return tile_of_many<THREADS>(p, tile, rows, adapter);
    if (tile >= *p.num_tiles) return 0;
    const LoraTile d = p.tiles[tile];
    adapter = d.adapter;
    if (threadIdx.x < d.count) rows[threadIdx.x] = p.order[d.start + threadIdx.x];
    __syncthreads();
    return d.count;
}
}  // namespace

// More than 64 rows, adapter by adapter (their order inside one is of no consequence: a row's sums are its own), and the tiles they make.  One workgroup: 8 us for 8192 rows, 300 for 2^19
__global__ __launch_bounds__(1024) void lora_group_kernel(LoraParams p, int tr, int32_t *order, LoraTile *tiles, int32_t *num_tiles) {
    extern __shared__ int32_t count[];                                    // [n + 1] rows of an adapter, then where its next row goes
    __shared__ int32_t sum_rows[16], sum_tiles[16], base_rows, base_tiles;
    const int n = (int)p.a.n + 1, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    for (int i = tid; i < n; i += 1024) count[i] = 0;
    if (tid == 0) base_rows = base_tiles = 0;
    __syncthreads();
    auto add = [&](int id) {                                              // (returns the row's place; lanes of the first lane's adapter add together: a prompt's rows are all of one)
        int at = 0;
        const unsigned long long have = __ballot(id >= 0);
        if (!have) return at;
        const int first = __ffsll((long long)have) - 1, lead = __shfl(id, first);
        const unsigned long long same = __ballot(id == lead);
        int start = 0;
        if (lane == first) start = atomicAdd(&count[lead], __popcll(same));
        start = __shfl(start, first);
        if (id == lead) at = start + __popcll(same & ((1ull << lane) - 1));
        else if (id >= 0) at = atomicAdd(&count[id], 1);
        return at;
    };
    const int64_t T = p.a.T;
    int id[8];                                                            // (8 rows a thread are asked for together, and kept where there are no more)
    auto ask = [&](int64_t c) {
#pragma unroll
        for (int e = 0; e < 8; ++e) id[e] = c + e * 1024 + tid < T ? p.a.ids[c + e * 1024 + tid] : -1;
#pragma unroll
        for (int e = 0; e < 8; ++e) id[e] = id[e] >= 0 && id[e] < (int)p.a.n ? id[e] : p.copies && c + e * 1024 + tid < T ? (int)p.a.n : -1;
    };
    for (int64_t c = 0; c < T; c += 8192) {
        ask(c);
#pragma unroll
        for (int e = 0; e < 8; ++e) add(id[e]);
    }
    __syncthreads();
    for (int c = 0; c < n; c += 1024) {                                   // exclusive sums of rows and tiles over the adapters
        const int i = c + tid, rows = i < n ? count[i] : 0, mine = (rows + tr - 1) / tr;
        int r = rows, t = mine;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int ur = __shfl_up(r, d), ut = __shfl_up(t, d);
            if (lane >= d) { r += ur; t += ut; }
        }
        if (lane == 63) { sum_rows[wave] = r; sum_tiles[wave] = t; }
        __syncthreads();
        int r0 = base_rows, t0 = base_tiles;
        for (int w = 0; w < wave; ++w) { r0 += sum_rows[w]; t0 += sum_tiles[w]; }
        __syncthreads();
        if (tid == 1023) { base_rows = r0 + r; base_tiles = t0 + t; }
        r0 += r - rows; t0 += t - mine;
        if (i < n) {
            count[i] = r0;
            for (int k = 0; k < mine; ++k) tiles[t0 + k] = LoraTile{r0 + k * tr, min(tr, rows - k * tr), i};
        }
        __syncthreads();
    }
    if (tid == 0) *num_tiles = base_tiles;
    for (int64_t c = 0; c < T; c += 8192) {
        if (T > 8192) ask(c);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int at = add(id[e]);
            if (id[e] >= 0) order[at] = (int32_t)(c + e * 1024 + tid);
        }
    }
}

// Rows come from memory 128 bytes at a time, 8 rows a request, and pass through the wave's own LDS image into the layout of the operands (straight into that layout a request would be 16 rows of 64 bytes,
// and each of its 64 lanes an address of its own: 26 GB/s a CU).
template <class E>
struct Strip {
    static constexpr int CK = 128 / (int)sizeof(typename E::T), STEPS = CK / E::KS;      // numbers of a strip of a row, steps of the product in it
    // piece c (16 bytes) of row r, in an image of 128-byte rows
    static __device__ __forceinline__ int place(int r, int c) { return r * 128 + ((c ^ (r & 7)) << 4); }
};

// D(rank x row) = A . x^T: a lane's 4 sums are neighbours in v.  The waves of a workgroup take the strips of its share of K in turn; the next one is on its way.
// The waves' sums of ranks r0 .. r0 + 16 RT - 1 over share `split` of K are left in smem: [wave][tile of 16 rows x tile of 16 ranks][lane]
template <int MT, int RT>
constexpr int image_bytes() { return (MT + RT) * 16 * 128; }
template <class E, int MT, int RT, int WAVES>
__device__ __forceinline__ void down_sums(const LoraParams &p, const int *rows, int count, int adapter, int r0, int split, char *smem) {
    typedef typename E::T T; typedef typename E::V V;
    typedef Strip<E> S;
    constexpr int XN = MT * 2, AN = RT * 2, IMAGE = image_bytes<MT, RT>();
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, lm = lane & 15, lq = lane >> 4, lr = lane >> 3, lp = lane & 7;
    const int K = (int)p.a.K, R = (int)p.a.R;
    const int strips = (K + S::CK - 1) / S::CK, per = (strips + p.splits - 1) / p.splits, first = split * per, last = min(strips, first + per);
    const T *x[XN], *w[AN];
#pragma unroll
    for (int u = 0; u < XN; ++u) { const int t = u * 8 + lr; x[u] = (const T *)p.a.x + (int64_t)rows[t < count ? t : 0] * p.a.ldx + lp * E::W; }
#pragma unroll
    for (int u = 0; u < AN; ++u) w[u] = (const T *)p.a.A + ((int64_t)adapter * R + min(r0 + u * 8 + lr, R - 1)) * K + lp * E::W;
    char *xi = smem + wave * IMAGE, *ai = xi + MT * 16 * 128;
    V xv[XN], wv[AN];
    const bool aligned = p.xw && p.aw;
    auto request = [&](int s) {
        const int k = s * S::CK, n = K - k - lp * E::W;                   // numbers of the row from this lane's piece on
        if (aligned && k + S::CK <= K) {
#pragma unroll
            for (int u = 0; u < XN; ++u) xv[u] = *reinterpret_cast<const V *>(x[u] + k);
#pragma unroll
            for (int u = 0; u < AN; ++u) wv[u] = *reinterpret_cast<const V *>(w[u] + k);
        } else {
#pragma unroll
            for (int u = 0; u < XN; ++u) xv[u] = n > 0 ? load16<E>(x[u] + k, p.xw, n) : zero16<E>();
#pragma unroll
            for (int u = 0; u < AN; ++u) wv[u] = n > 0 ? load16<E>(w[u] + k, p.aw, n) : zero16<E>();
        }
    };
    float4_t acc[MT][RT];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int r = 0; r < RT; ++r) acc[m][r] = (float4_t){0.f, 0.f, 0.f, 0.f};
    if (first + wave < last) request(first + wave);
    for (int s = first + wave; s < last; s += WAVES) {
#pragma unroll
        for (int u = 0; u < XN; ++u) *reinterpret_cast<V *>(xi + S::place(u * 8 + lr, lp)) = xv[u];
#pragma unroll
        for (int u = 0; u < AN; ++u) *reinterpret_cast<V *>(ai + S::place(u * 8 + lr, lp)) = wv[u];
        asm volatile("" ::: "memory");                                    // (a wave's LDS requests are served in order)
        if (s + WAVES < last) request(s + WAVES);
#pragma unroll
        for (int st = 0; st < S::STEPS; ++st) {
            V xf[MT], wf[RT];
#pragma unroll
            for (int m = 0; m < MT; ++m) xf[m] = *reinterpret_cast<const V *>(xi + S::place(m * 16 + lm, st * 4 + lq));
#pragma unroll
            for (int r = 0; r < RT; ++r) wf[r] = *reinterpret_cast<const V *>(ai + S::place(r * 16 + lm, st * 4 + lq));
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int r = 0; r < RT; ++r) acc[m][r] = E::mma(wf[r], xf[m], acc[m][r]);
        }
        asm volatile("" ::: "memory");
    }
    // the waves' sums, one behind the other
    static_assert(MT * RT * 1024 <= IMAGE, "");
    __syncthreads();
    float4_t *part = reinterpret_cast<float4_t *>(smem);                  // [wave][tile][lane]
#pragma unroll
    for (int i = 0; i < MT * RT; ++i) part[(wave * MT * RT + i) * 64 + lane] = acc[i / RT][i % RT];
    __syncthreads();
}
template <class E, int MT, int RT, Find FIND, int WAVES>
__global__ __launch_bounds__(WAVES * 64) void lora_down_kernel(LoraParams p) {
    constexpr int TR = MT * 16;
    __shared__ int rows[TR];
    __shared__ __attribute__((aligned(16))) char smem[WAVES * image_bytes<MT, RT>()];
    int adapter = -1;
    const int count = tile_rows<TR, FIND, WAVES * 64>(p, blockIdx.x, rows, adapter);
    if (!count || adapter >= (int)p.a.n) return;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, lm = lane & 15, lq = lane >> 4, r0 = blockIdx.z * RT * 16;
    down_sums<E, MT, RT, WAVES>(p, rows, count, adapter, r0, blockIdx.y, smem);
    const float4_t *part = reinterpret_cast<const float4_t *>(smem);
    const float scale = p.a.scales ? p.a.scales[adapter] : 1.f;
    for (int i = wave; i < MT * RT; i += WAVES) {
        const int m = i / RT, r = i % RT, t = m * 16 + lm;
        float4_t v = part[i * 64 + lane];
#pragma unroll
        for (int o = 1; o < WAVES; ++o) v += part[(o * MT * RT + i) * 64 + lane];
        if (t < count && r0 + r * 16 < p.rp) *reinterpret_cast<float4_t *>(p.v + ((int64_t)blockIdx.y * p.a.T + rows[t]) * p.rp + r0 + r * 16 + lq * 4) = v * scale;
    }
}

// D(column x row) = B . v^T: a lane's NT * 4 = W sums are neighbours in y (row m of tile i of B is column (m / 4) W + 4 i + m % 4 of the group).  A wave takes groups of NT * 16 columns, two at a time,
// straight from and to memory: rows of 64 bytes a request, but no wait between.  (Through images as above, requests of whole rows: 93 -> 171 us for 8192 rows of 12288 columns of rank 32.)
// v in LDS: [hi, lo] [rows][ldv], 32 bits: [rows][ldv]; high: float16, bits of a row's largest |v|
template <class E>
constexpr int v_stride(int R) { return (R + E::KS - 1) / E::KS * E::KS + E::W; }      // (16 bytes off a multiple of 64: neighbours lie in other banks)
template <class E, int MT>
__device__ __forceinline__ void up_columns(const LoraParams &p, const int *rows, int count, int adapter, const typename E::T *hi, const unsigned int *high, int ldv, int g0, int groups) {
    typedef typename E::T T; typedef typename E::V V;
    constexpr int TR = MT * 16, W = E::W, NT = W / 4, GN = NT * 16;
    constexpr bool F = sizeof(T) == 4, H = __is_same(E, F16);
    const int lane = threadIdx.x & 63, lm = lane & 15, lq = lane >> 4;
    const int R = (int)p.a.R, N = (int)p.a.N, ks = (R + E::KS - 1) / E::KS;
    const bool real = adapter < (int)p.a.n;
    const T *lo = hi + TR * ldv;
    const int64_t at0 = (int64_t)lq * W;
    int64_t row[MT];
    float back[MT];                                                       // what undoes the row's range
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        const int t = m * 16 + lm;
        row[m] = rows[t < count ? t : 0];
        back[m] = H && real ? __uint_as_float((unsigned)(127 - range_of(high[t])) << 23) : 1.f;
    }
    const T *B = (const T *)p.a.B + (int64_t)adapter * N * R;
    // NB neighbouring groups at a time; whole: all their columns are there, everything in aligned pieces of 16 bytes
    auto go = [&](int64_t n0, auto nb, auto whole) {
        constexpr int NB = decltype(nb)::value;
        constexpr bool WH = decltype(whole)::value;
        V b[NB][MT];
        int left[NB];                                                     // columns of this lane that there are
#pragma unroll
        for (int q = 0; q < NB; ++q) {
            left[q] = WH ? W : (int)max((int64_t)0, min((int64_t)W, N - n0 - q * GN - at0));
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                const T *at = (const T *)p.a.base + row[m] * p.a.ldb + n0 + q * GN + at0;
                b[q][m] = WH ? *reinterpret_cast<const V *>(at) : left[q] > 0 ? load16<E>(at, p.yw, left[q]) : zero16<E>();
            }
        }
        float4_t acc[NB][NT][MT];
#pragma unroll
        for (int q = 0; q < NB; ++q)
#pragma unroll
            for (int i = 0; i < NT; ++i)
#pragma unroll
                for (int m = 0; m < MT; ++m) acc[q][i][m] = (float4_t){0.f, 0.f, 0.f, 0.f};
        if (real) {
            const T *bp[NB][NT];
#pragma unroll
            for (int q = 0; q < NB; ++q)
#pragma unroll
                for (int i = 0; i < NT; ++i) {
                    const int64_t n = n0 + q * GN + (lm >> 2) * W + 4 * i + (lm & 3);
                    bp[q][i] = B + (WH ? n : min(n, (int64_t)N - 1)) * R;
                }
            for (int k = 0; k < ks; ++k) {
                const int r = k * E::KS + lq * W, n = R - r;
                V bv[NB][NT];
#pragma unroll
                for (int q = 0; q < NB; ++q)
#pragma unroll
                    for (int i = 0; i < NT; ++i) bv[q][i] = n >= W && (WH || p.bw) ? *reinterpret_cast<const V *>(bp[q][i] + r) : !WH && n > 0 ? load16<E>(bp[q][i] + r, false, n) : zero16<E>();
#pragma unroll
                for (int m = 0; m < MT; ++m) {
                    const V vh = *reinterpret_cast<const V *>(hi + (m * 16 + lm) * ldv + r);
#pragma unroll
                    for (int q = 0; q < NB; ++q)
#pragma unroll
                        for (int i = 0; i < NT; ++i) acc[q][i][m] = E::mma(bv[q][i], vh, acc[q][i][m]);
                    if constexpr (!F) {
                        const V vl = *reinterpret_cast<const V *>(lo + (m * 16 + lm) * ldv + r);
#pragma unroll
                        for (int q = 0; q < NB; ++q)
#pragma unroll
                            for (int i = 0; i < NT; ++i) acc[q][i][m] = E::mma(bv[q][i], vl, acc[q][i][m]);
                    }
                }
            }
        }
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int q = 0; q < NB; ++q) {
                if (m * 16 + lm >= count || left[q] <= 0) continue;
                V o;
#pragma unroll
                for (int e = 0; e < W; ++e) {
                    const float v = acc[q][e / 4][m][e % 4], x = (float)b[q][m][e];
                    o[e] = real ? (T)(H ? fmaf(v, back[m], x) : x + v) : b[q][m][e];
                }
                T *y = (T *)p.a.y + row[m] * p.a.ldy + n0 + q * GN + at0;
                if (WH || (left[q] == W && p.yw)) *reinterpret_cast<V *>(y) = o;
                else
#pragma unroll
                    for (int e = 0; e < W; ++e) if (e < left[q]) y[e] = o[e];
            }
    };
    const bool aligned = p.yw && p.bw;
    for (int g = g0, end = g + groups; g < end;) {
        const int64_t n0 = (int64_t)g * GN;
        if (n0 >= N) return;
        if (aligned && g + 2 <= end && n0 + 2 * GN <= N) { go(n0, std::integral_constant<int, 2>(), std::true_type()); g += 2; }
        else if (aligned && n0 + GN <= N) { go(n0, std::integral_constant<int, 1>(), std::true_type()); ++g; }
        else { go(n0, std::integral_constant<int, 1>(), std::false_type()); ++g; }
    }
}

template <class E, int MT, Find FIND>
__global__ __launch_bounds__(256, MT == 4 ? 3 : 1) void lora_up_kernel(LoraParams p, int groups) {
    typedef typename E::T T; typedef typename E::V V;
    constexpr int TR = MT * 16;
    constexpr bool F = sizeof(T) == 4, H = __is_same(E, F16);
    extern __shared__ __attribute__((aligned(16))) char smem[];           // v
    __shared__ unsigned int high[TR];
    __shared__ int rows[TR];
    int adapter = -1;
    const int count = tile_rows<TR, FIND, 256>(p, blockIdx.y, rows, adapter);
    if (!count) return;
    const int wave = threadIdx.x >> 6, R = (int)p.a.R, ldv = v_stride<E>(R);
    const bool real = adapter < (int)p.a.n;
    T *hi = reinterpret_cast<T *>(smem), *lo = hi + TR * ldv;
    if (real) {
        const int per = (ldv - E::W) / 4;                                   // pieces of 4 sums; a thread has up to 8 (64 rows of rank 128, 16 of rank 256)
        float4_t v[8];
        if (H && threadIdx.x < TR) high[threadIdx.x] = 0;
        if (H) __syncthreads();
#pragma unroll
        for (int n = 0; n < 8; ++n) {
            const int i = n * 256 + threadIdx.x, t = i / per, r = (i - t * per) * 4;
            v[n] = (float4_t){0.f, 0.f, 0.f, 0.f};
            if (i < TR * per && t < count && r < p.rp) {
                const float *at = p.v + (int64_t)rows[t] * p.rp + r;
                const int64_t next = p.a.T * p.rp;
                int s = 0;
                for (; s + 4 <= p.splits; s += 4, at += 4 * next) {
                    float4_t q[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) q[e] = *reinterpret_cast<const float4_t *>(at + e * next);
                    v[n] += (q[0] + q[1]) + (q[2] + q[3]);
                }
                for (; s < p.splits; ++s, at += next) v[n] += *reinterpret_cast<const float4_t *>(at);
            }
            float most = 0.f;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (r + e >= R) v[n][e] = 0.f;                            // (behind R there are repeats of the last row of A)
                most = fmaxf(most, fabsf(v[n][e]));
            }
            if (H && i < TR * per) atomicMax(&high[t], __float_as_uint(most));
        }
        if (H) __syncthreads();
#pragma unroll
        for (int n = 0; n < 8; ++n) {
            const int i = n * 256 + threadIdx.x, t = i / per, r = (i - t * per) * 4;
            if (i >= TR * per) break;
            const float f = H ? __uint_as_float((unsigned)(127 + range_of(high[t])) << 23) : 1.f;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float x = v[n][e] * f;
                const T h = (T)x;
                hi[t * ldv + r + e] = h;
                if constexpr (!F) lo[t * ldv + r + e] = (T)(fabsf((float)h) < INFINITY ? x - (float)h : 0.f);
            }
        }
    }
    __syncthreads();
    up_columns<E, MT>(p, rows, count, adapter, hi, high, ldv, (blockIdx.x * 4 + wave) * groups, groups);
}
// Both in one launch, where few rows (tiles of 16) meet few ranks (up to kRanks, 16 RT at a time): each workgroup forms v anew for its columns, 8 waves over K, and keeps it in LDS
constexpr int kRanks = 96;
template <class E, int RT, Find FIND>
__global__ __launch_bounds__(512) void lora_both_kernel(LoraParams p) {
    typedef typename E::T T;
    constexpr bool F = sizeof(T) == 4, H = __is_same(E, F16);
    constexpr int MOST = v_stride<E>(RT == 1 ? 16 : kRanks);
    __shared__ int rows[16];
    __shared__ unsigned int high[16];
    __shared__ __attribute__((aligned(16))) char smem[8 * image_bytes<1, RT>()];
    __shared__ __attribute__((aligned(16))) T v[(F ? 1 : 2) * 16 * MOST];
    __shared__ float sums[RT == 1 ? 16 : kRanks][17];                     // [rank][row]
    int adapter = -1;
    const int count = tile_rows<16, FIND, 512>(p, blockIdx.y, rows, adapter);
    if (!count) return;
    const int tid = threadIdx.x, R = (int)p.a.R, ldv = v_stride<E>(R);
    T *hi = v, *lo = v + 16 * ldv;
    if (adapter < (int)p.a.n) {
        for (int i = tid; i < (F ? 1 : 2) * 16 * ldv; i += 512) v[i] = (T)0.f;      // (what the last step of the product reads behind R)
        if (tid < 16) high[tid] = 0;
        const float scale = p.a.scales ? p.a.scales[adapter] : 1.f;
        for (int r0 = 0; r0 < R; r0 += RT * 16) {
            if (r0) __syncthreads();
            down_sums<E, 1, RT, 8>(p, rows, count, adapter, r0, 0, smem);
            if (tid < RT * 64) {
                const int t = tid & 15, r = r0 + (tid >> 6) * 16 + ((tid >> 4) & 3) * 4;
                const float4_t *part = reinterpret_cast<const float4_t *>(smem) + tid;
                float4_t sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int w = 0; w < 8; ++w) sum += part[w * RT * 64];
                sum *= scale;
                float most = 0.f;
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (r + e < R && t < count) { sums[r + e][t] = sum[e]; most = fmaxf(most, fabsf(sum[e])); }      // (behind them are repeats)
                if (H) atomicMax(&high[t], __float_as_uint(most));
            }
        }
        __syncthreads();
        for (int i = tid; i < 16 * R; i += 512) {
            const int t = i & 15, r = i >> 4;
            if (t >= count) continue;
            const float x = sums[r][t] * (H ? __uint_as_float((unsigned)(127 + range_of(high[t])) << 23) : 1.f);
            const T h = (T)x;
            hi[t * ldv + r] = h;
            if constexpr (!F) lo[t * ldv + r] = (T)(fabsf((float)h) < INFINITY ? x - (float)h : 0.f);
        }
    }
    __syncthreads();
    up_columns<E, 1>(p, rows, count, adapter, hi, high, ldv, blockIdx.x * 8 + (tid >> 6), 1);
}

static int lora_splits_most(int64_t T, int64_t K) {                       // (a wave has a strip of 64 at least)
    return (int)std::max<int64_t>(1, std::min<int64_t>(4, K / 512));
}
static int64_t lora_rp(int64_t R) { return (R + 15) / 16 * 16; }
size_t lora_workspace_bytes(int64_t T, int64_t K, int64_t N, int64_t R) {
    (void)N;
    if (T <= 0 || K <= 0 || R <= 0) return 0;
    return (size_t)T * lora_splits_most(T, K) * lora_rp(R) * 4 + (T > kSmall ? ((size_t)T * (4 + sizeof(LoraTile)) + 64) : 0);
}

template <class E, int MT, Find FIND>
static void lora_launch(const LoraParams &p, int64_t tiles, hipStream_t s) {
    const int rt = (int)(p.rp / 16);
    const unsigned t = (unsigned)tiles, z = (unsigned)p.splits;
    constexpr int WAVES = MT == 4 ? 4 : 8;                                // tiles of 16 rows: more waves of a workgroup share K, and v has fewer shares to add up again
    if (rt == 1) lora_down_kernel<E, MT, 1, FIND, WAVES><<<dim3(t, z, 1), WAVES * 64, 0, s>>>(p);
    else lora_down_kernel<E, MT, 2, FIND, WAVES><<<dim3(t, z, (rt + 1) / 2), WAVES * 64, 0, s>>>(p);
    constexpr int GN = E::W / 4 * 16;
    const int64_t all = (p.a.N + GN - 1) / GN;                            // groups of columns: a wave takes 1 to 4, as long as there are workgroups for two rounds of the chip
    int groups = 4;
    while (groups > 1 && (all + 4 * groups - 1) / (4 * groups) * tiles < 512) groups /= 2;
    lora_up_kernel<E, MT, FIND><<<dim3((unsigned)((all + 4 * groups - 1) / (4 * groups)), t), 256, (size_t)MT * 16 * v_stride<E>((int)p.a.R) * 4, s>>>(p, groups);
}

template <class E>
static int lora_of(const LoraArgs &a, hipStream_t s) {
    LoraParams p{};
    p.a = a;
    p.copies = a.base != a.y;
    p.rp = (int)lora_rp(a.R);
    auto whole = [](const void *q, int64_t ld) { return ((uintptr_t)q & 15) == 0 && ld % E::W == 0; };
    p.xw = whole(a.x, a.ldx); p.aw = whole(a.A, a.K); p.bw = whole(a.B, a.R); p.yw = whole(a.y, a.ldy) && whole(a.base, a.ldb);
    // the tiles there can be: full ones, and one begun per adapter (rows without one count as one).  64 rows, which read A and B a quarter as often, where the adapters have 32 and more in the middle and
    // there is enough to do for so few workgroups; else 16.  Rank 64, 4096 -> 4096, us with 16 and 64: 300 rows 16.0 19.7, 1024 25.9 22.8, 8192 99 80; rank 16: 2048 rows 23.5 23.6, 4096 39.7 39.9,
    // 8192 69 65; 8192 rows 4096 -> 12288 of rank 32 145 122
    const int64_t kinds = std::min<int64_t>(a.n + p.copies, a.T);
    const int tr = a.T * p.rp >= 65536 && a.T >= 32 * kinds && a.R <= 128 ? 64 : 16;   // (up: 64 rows of v in LDS, 34 KB at rank 128)
    const int64_t tiles = std::min<int64_t>(a.T, a.T / tr + kinds);
    const int64_t zs = (p.rp / 16 + 1) / 2;
    p.splits = (int)std::max<int64_t>(1, std::min<int64_t>(lora_splits_most(a.T, a.K), ((tr == 64 ? 512 : 256) + tiles * zs - 1) / (tiles * zs)));
    p.v = (float *)a.workspace;
    constexpr int GN = E::W / 4 * 16;
    const int64_t columns = (a.N + 8 * GN - 1) / (8 * GN), row = a.K * (int64_t)sizeof(typename E::T), size = sizeof(typename E::T);
    const char *x0 = (const char *)a.x, *y0 = (const char *)a.y;
    const bool apart = x0 + ((a.T - 1) * a.ldx + a.K) * size <= y0 || y0 + ((a.T - 1) * a.ldy + a.N) * size <= x0;
    const int64_t tiles16 = std::min<int64_t>(a.T, a.T / 16 + kinds);
    // One launch, as long as what its workgroups read again from the L2 caches (x and A of a tile for every 8 GN columns), and the way of one of them along K (for every 32 ranks), take less than the
    // launch spared and, beyond kSmall rows, the search for the tile in it.  us in one launch and in two, 16-bit types: 32 rows of 32 adapters of rank 16, 1024 -> 2048 (17 MB again) 5.3 9.0;
    // 64 x 4096 -> 4096, rank 32 (57 MB) 10.6 10.8; 32 x 4096 -> 4096, rank 16 (134 MB) 11.2 9.6; 32 x 2048 -> 2048, rank 96 (3 x 4 KB along K) 14.2 9.6; 251 x 4096 -> 4096, rank 16 (80 MB) 10.6 12.2,
    // rank 32 (145 MB) 16.4 13.5; 512 x 1024 -> 1024, rank 64 (2 x 24 MB) 9.7 12.4; 512 x 1024 -> 12288, rank 16 (116 MB) 19.0 17.0.  (Each workgroup reads x while others write y: they must not overlap.)
    const int64_t rounds = a.R <= 16 ? 1 : (a.R + 31) / 32, again = rounds * columns * tiles16 * (16 + p.rp) * row;
    const bool found = a.T <= kSmall || (a.T <= kMany && a.n < 1023), little = rounds * row <= 8192 && again <= (a.T <= kSmall ? 64ll : 96ll) << 20;
    if (apart && found && little && a.R <= kRanks) {
        p.splits = 1;
        const dim3 grid((unsigned)columns, (unsigned)tiles16);
        if (a.T <= kSmall) {
            if (a.R <= 16) lora_both_kernel<E, 1, SMALL><<<grid, 512, 0, s>>>(p);
            else lora_both_kernel<E, 2, SMALL><<<grid, 512, 0, s>>>(p);
        } else {
            if (a.R <= 16) lora_both_kernel<E, 1, MANY><<<grid, 512, 0, s>>>(p);
            else lora_both_kernel<E, 2, MANY><<<grid, 512, 0, s>>>(p);
        }
    } else if (a.T <= kSmall) lora_launch<E, 1, SMALL>(p, tiles, s);
    else if (tr == 16 && found) lora_launch<E, 1, MANY>(p, tiles, s);      // (251 x 4096 -> 4096, rank 64: 15.0 us, grouped by a launch 17.0)
    else {
        char *at = (char *)a.workspace + (size_t)a.T * lora_splits_most(a.T, a.K) * p.rp * 4;
        LoraTile *td = (LoraTile *)at;
        int32_t *order = (int32_t *)(at + (size_t)a.T * sizeof(LoraTile)), *nt = order + a.T;
        p.tiles = td; p.order = order; p.num_tiles = nt;
        lora_group_kernel<<<dim3(1), dim3(1024), (size_t)(a.n + 1) * 4, s>>>(p, tr, order, td, nt);
        if (tr == 64) lora_launch<E, 4, GROUPED>(p, tiles, s);
        else lora_launch<E, 1, GROUPED>(p, tiles, s);
    }
    NVR_KX_LAUNCHED("lora_add");
    return 0;
}

int lora_add(int dt, const LoraArgs &a, hipStream_t s) {
    if (a.T < 0 || a.K <= 0 || a.N <= 0 || a.R <= 0 || a.n < 0) return nvr::fail(NVR_ERR_INVALID_ARG, "nvr_lora_add: T=%ld K=%ld N=%ld R=%ld adapters=%ld", (long)a.T, (long)a.K, (long)a.N, (long)a.R, (long)a.n);
    if (a.R > 256 || a.n >= kMaxAdapters || a.K > (1 << 22) || a.N > (1 << 22) || a.T > (1 << 19))       // (tiles and groups of columns are grid axes of 65535)
        return nvr::fail(NVR_ERR_UNSUPPORTED, "nvr_lora_add: ranks up to 256, fewer than %d adapters, 2^19 rows of up to 2^22 numbers (T=%ld K=%ld N=%ld R=%ld adapters=%ld)", kMaxAdapters, (long)a.T, (long)a.K, (long)a.N, (long)a.R, (long)a.n);
    if (a.T == 0) return 0;
    if (!a.x || !a.ids || !a.base || !a.y || !a.workspace || (a.n && (!a.A || !a.B))) return nvr::fail(NVR_ERR_INVALID_ARG, "nvr_lora_add: null argument");
    if (((uintptr_t)a.workspace & 15) != 0) return nvr::fail(NVR_ERR_INVALID_ARG, "nvr_lora_add: the workspace is not aligned to 16 bytes");
    if (a.ldx < a.K || a.ldb < a.N || a.ldy < a.N) return nvr::fail(NVR_ERR_INVALID_ARG, "nvr_lora_add: rows overlap");
    if (a.base == a.y && a.ldb != a.ldy) return nvr::fail(NVR_ERR_INVALID_ARG, "nvr_lora_add: in place with another stride");
    if (a.n == 0 && a.base == a.y) return 0;
    NVR_BY_DTYPE(dt, return lora_of<E>(a, s));
}

}}  // namespace nvr::kx
