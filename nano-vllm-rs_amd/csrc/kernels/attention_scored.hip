// attention_scored.hip — decode attention over the paged cache that also adds each key's attention weight, summed over the query heads of its kv head, to the key's score.
//
//   s_hj = scale q_h . k_j,  w_hj = exp(s_hj - M_h) / L_h,  out_h = sum_j w_hj v_j,  score'_gj = decay score_gj (keys j < scored_lens) + sum over the heads h of g of w_hj
//
// A weight is known when the row's maximum and sum are, that is behind the last key.  So the first launch is a split decode attention that reads K and V once and leaves its scores s in the
// workspace (4 bytes a key and head beside the 4 D bytes of the key's rows), and the second turns them into weights: it merges the partitions' (maximum, sum), updates the scores, and joins the
// partitions' outputs.  Bound by the stream of K and V.
// First launch: as many workgroups as fit the chip at once, each with an equal share of all sequences' keys for one kv head, in units of 128 (a grid of (sequence, part) leaves most of its workgroups empty
// where contexts differ, and a last round half full: 48 contexts of 512 .. 8100 keys 119 us).  A workgroup's four waves take tiles of TK keys on the matrix cores, the heads of the group (up to 16) as
// columns: S^T = K Q^T, O^T += V^T P^T.  Rows come from the pages whole (16 bytes a lane, the next tile's in flight) and pass through the wave's own LDS image into the layout of the operands.  Weights
// enter the second product as two 16-bit numbers, the rounded weight and the rounded rest, so that they have 17 (bfloat16) or 22 bits there: the cores are idle most of the time anyway.
// 48 sequences of 512 .. 8100 keys, 32 heads over 8 of 128, bfloat16: 119 us (107 and 12) for 556 MB, 4.7 TB/s; 32 x 8192 keys of 4 heads a kv head: 220 us, 4.95 TB/s, where the decode attention
// without scores takes 212; one sequence of 2047 keys: 10 us (6 and 4), two launches and their chains of round trips.  float32: the 48 sequences 209 us (196 and 13, 1.1 GB), the one 14.
#include <algorithm>
#include "serving.h"
#include "elem.h"
#include "../common.h"

namespace nvr { namespace kx {

namespace {
constexpr float kLog2e = 1.44269504088896340736f;
constexpr int kUnit = 128;                                                // keys of a unit: a tile of 32 (32 bits: two of 16) for each wave
struct ScoredParams {
    ScoredArgs a;
    int32_t wide;                                                         // WHOLE: scores of a head in LDS
    int32_t shares, lpad;                                                 // workgroups of a kv head, scores of a head in the workspace
    float *s, *ml, *o;                                                    // [B][H][lpad], [shares + B][H][2], [shares + B][H][D]: share w's part of sequence b at w + b
    int32_t *ends;                                                        // [B][2]: the first and the last share of a sequence
    bool qw;
};
// keys that the attention may look at
__device__ __forceinline__ int visible(const ScoredArgs &a, int b) {
    const long long most = (long long)a.max_blocks * a.block_size;
    int n = a.ctx_lens[b];
    n = min(n, a.max_ctx);
    return (int)max(0ll, min((long long)n, most));
}
__device__ __forceinline__ int units_of(const ScoredArgs &a, int b) { return (visible(a, b) + kUnit - 1) / kUnit; }
template <class E, int D>
struct Image {
    static constexpr int TK = sizeof(typename E::T) == 4 ? 16 : 32;                                   // keys of a tile
    static constexpr int ROW = D * (int)sizeof(typename E::T), LPR = ROW / 16, RPI = 64 / LPR, NI = TK / RPI;   // bytes of a row, lanes of it, rows of a request, requests of a tile
    static constexpr int VS = ROW + (sizeof(typename E::T) == 4 ? 16 : 32);                           // V: stride of a row (conflict-free transposed reads)
    static constexpr int KB = TK * ROW, BYTES = KB + TK * VS, OS = D + 4, ALL = 4 * BYTES > 4 * 16 * OS * 4 ? 4 * BYTES : 4 * 16 * OS * 4;                               // K's image, both; numbers of a row of the waves' sums; bytes of either for four waves
};
// operand of O^T += V^T P^T: column (of 16) lm of V, keys 4 lq .. at `a` and 16 further at `b`, by the transposing reads
template <class E>
__device__ __forceinline__ typename E::V transposed(const char *a, const char *b) {
    typename E::V v;
    if constexpr (__is_same(E, BF16)) {
        typedef __bf16 b4 __attribute__((ext_vector_type(4)));
        const b4 x = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((__attribute__((address_space(3))) b4 *)a), y = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((__attribute__((address_space(3))) b4 *)b);
        v = __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
    } else if constexpr (__is_same(E, F16)) {
        typedef __fp16 h4 __attribute__((__vector_size__(4 * sizeof(__fp16))));
        const h4 x = __builtin_amdgcn_ds_read_tr16_b64_v4f16((__attribute__((address_space(3))) h4 *)a), y = __builtin_amdgcn_ds_read_tr16_b64_v4f16((__attribute__((address_space(3))) h4 *)b);
#pragma unroll
        for (int e = 0; e < 4; ++e) { v[e] = (_Float16)x[e]; v[4 + e] = (_Float16)y[e]; }
    }
    return v;
}
}  // namespace

// WHOLE: contexts are short, and a workgroup has a sequence's keys of a kv head and answers by itself, scores in LDS: no second launch, no workspace.  us where it answers and with two launches: 5 sequences
// of up to 60 keys 5.2 10.7, 32 of 20 .. 250 9.1 11.9, 32 of 200 .. 500 16.8 19.9, 64 of 100 .. 500 (4 heads a kv head) 19.7 26.9; 8 of 200 .. 500 14.2 11.6, 32 of 100 .. 1000 24.6 20.0.  (F32 of 128: 3
// registers are spilled)
template <class E, int D, bool WHOLE>
__global__ __launch_bounds__(256, D == 256 ? 1 : 2) void attn_scored_kernel(ScoredParams p) {
    typedef typename E::T T; typedef typename E::V V;
    typedef Image<E, D> I;
    constexpr bool F = sizeof(T) == 4;
    constexpr int MT = I::TK / 16, NKS = D / E::KS, DT = D / 16;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    __shared__ float ml[4][16][2];
    __shared__ int sums[4], at[2];
    __shared__ float big[16], inv[16];
    const int g = blockIdx.x, w = blockIdx.y;                             // (kv heads of the same keys next to each other: their rows are neighbours)
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, lm = lane & 15, lq = lane >> 4;
    const int G = p.a.H / p.a.KVH;
    // ---- this share of all sequences' units, one behind the other: units u0 .. u1 - 1, the first of them number `unit` of sequence b
    int b, unit, u0, u1, shares;                                          // (a share has a unit at least: the second launch counts on it)
    auto shared_out = [&](int all) {
        shares = min(p.shares, all);
        if (w >= shares) return false;
        u0 = (int)((int64_t)w * all / shares); u1 = (int)((int64_t)(w + 1) * all / shares);
        return true;
    };
    if constexpr (WHOLE) {
        b = w; unit = 0; u0 = 0; u1 = units_of(p.a, b);
        if (u1 == 0) {
            T *out = (T *)p.a.out + ((int64_t)b * p.a.H + g * G) * D;
            for (int i = threadIdx.x; i < G * D; i += 256) out[i] = (T)0.f;
            return;
        }
    } else if (p.a.B <= 64) {                                             // a lane a sequence, every wave for itself
        const int mine = lane < p.a.B ? units_of(p.a, lane) : 0;
        int upto = mine;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) { const int o = __shfl_up(upto, d); if (lane >= d) upto += o; }
        if (!shared_out(__builtin_amdgcn_readlane(upto, 63))) return;
        b = __ffsll((long long)__ballot(upto > u0)) - 1;
        unit = u0 - __builtin_amdgcn_readlane(upto - mine, b);
    } else {                                                              // a thread counts those of `per` sequences
        const int per = (p.a.B + 255) / 256, b0 = threadIdx.x * per;
        int mine = 0;
        for (int i = 0; i < per && b0 + i < p.a.B; ++i) mine += units_of(p.a, b0 + i);
        int upto = mine;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) { const int o = __shfl_up(upto, d); if (lane >= d) upto += o; }
        if (lane == 63) sums[wave] = upto;
        __syncthreads();
        int all = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) { if (i < wave) upto += sums[i]; all += sums[i]; }
        if (!shared_out(all)) return;
        if (upto - mine <= u0 && u0 < upto) {
            int u = upto - mine, i = b0;
            for (int n; u + (n = units_of(p.a, i)) <= u0; ++i) u += n;
            at[0] = i; at[1] = u0 - u;
        }
        __syncthreads();
        b = __builtin_amdgcn_readfirstlane(at[0]); unit = __builtin_amdgcn_readfirstlane(at[1]);
    }
    const float scale2 = p.a.scale * kLog2e;
    const int64_t row_elems = (int64_t)p.a.KVH * D;
    const T *kc = (const T *)p.a.k + (int64_t)g * D, *vc = (const T *)p.a.v + (int64_t)g * D;
    char *img = smem + wave * I::BYTES;
    float *kept = reinterpret_cast<float *>(smem + I::ALL);               // WHOLE: scores of the heads, p.wide apart
    const int rl = lane / I::LPR, pl = lane % I::LPR;                     // this lane's row of a request and its piece
    for (int left = u1 - u0; left > 0; ++b, unit = 0) {
        const int ctx = visible(p.a, b), units = (ctx + kUnit - 1) / kUnit, take = min(left, units - unit);
        if (take <= 0) continue;                                              // (a sequence without keys)
        left -= take;
        const int first = unit * kUnit, last = min(ctx, first + take * kUnit);
        if (!WHOLE && g == 0 && threadIdx.x == 0) {
            if (unit == 0) p.ends[2 * b] = w;
            if (unit + take == units) p.ends[2 * b + 1] = w;
        }
        const int32_t *table = p.a.block_tables + (int64_t)b * p.a.max_blocks;
        V qf[NKS];                                                            // column lm: head lm of the group (none behind the last: 0)
        {
            const T *q = (const T *)p.a.q + (int64_t)b * p.a.ldq + (int64_t)(g * G + min(lm, G - 1)) * D + lq * E::W;
#pragma unroll
            for (int ks = 0; ks < NKS; ++ks) qf[ks] = lm < G ? load16<E>(q + ks * E::KS, p.qw) : zero16<E>();
        }
        // key `lane` of a tile: its page is asked for two tiles ahead, its row (< 0: not in the pool) formed one tile ahead.  Keys that are not there take another's row: their scores are -inf, their values 0
        auto page_of = [&](int tile) {
            const int j = min(first + tile * I::TK + (lane & (I::TK - 1)), last - 1);
            return table[(unsigned)j / (unsigned)p.a.block_size];
        };
        auto rows_of = [&](int tile, int page, unsigned int &mask) {
            const int j = first + tile * I::TK + (lane & (I::TK - 1));
            const bool in = j < last && page >= 0 && page < p.a.num_blocks;
            const int r = in ? page * p.a.block_size + (int)((unsigned)j % (unsigned)p.a.block_size) : -1;
            mask = (unsigned int)__ballot(in && lane < I::TK);
            const int other = mask ? __builtin_amdgcn_readlane(r, __ffs(mask) - 1) : -1;      // (in front of the choice: an exchange among the lanes that choose it would ask a lane that is not there)
            return in ? r : other;
        };
        V kx[I::NI], vx[I::NI];
        auto request = [&](int rows) {
#pragma unroll
            for (int u = 0; u < I::NI; ++u) {
                const int64_t o = (int64_t)__shfl(rows, u * I::RPI + rl) * row_elems + pl * E::W;
                kx[u] = __builtin_nontemporal_load(reinterpret_cast<const V *>(kc + o));
                vx[u] = __builtin_nontemporal_load(reinterpret_cast<const V *>(vc + o));
            }
        };
        const int tiles = (last - first + I::TK - 1) / I::TK;
        float m = -INFINITY, l = 0.f;
        float4_t o[DT];
#pragma unroll
        for (int t = 0; t < DT; ++t) o[t] = (float4_t){0.f, 0.f, 0.f, 0.f};
        constexpr unsigned int kAll = I::TK == 32 ? 0xffffffffu : 0xffffu;
        char *vimg = img + I::KB;
        float *sp = WHOLE ? kept + lm * p.wide : p.s + ((int64_t)b * p.a.H + g * G + lm) * p.lpad;
        unsigned int mask = 0;
        int page = 0;
        if (wave < tiles) {
            page = page_of(wave);
            const int rows = rows_of(wave, page, mask);
            page = page_of(wave + 4);
            if (mask) request(rows);
        }
        constexpr int SW = I::LPR >= 16 ? 15 : I::LPR - 1;                    // K: piece c of row r at slot c ^ (r & SW)
        for (int x = wave; x < tiles; x += 4) {
            const int j0 = first + x * I::TK;
            const unsigned int here = mask;
            if (here) {
                if (here != kAll)
#pragma unroll
                    for (int u = 0; u < I::NI; ++u) if (!((here >> (u * I::RPI + rl)) & 1)) vx[u] = zero16<E>();
#pragma unroll
                for (int u = 0; u < I::NI; ++u) { const int r = u * I::RPI + rl; *reinterpret_cast<V *>(img + r * I::ROW + ((pl ^ (r & SW)) << 4)) = kx[u]; }
#pragma unroll
                for (int u = 0; u < I::NI; ++u) *reinterpret_cast<V *>(vimg + (u * I::RPI + rl) * I::VS + pl * 16) = vx[u];
            }
            asm volatile("" ::: "memory");                                    // (a wave's LDS requests are served in order)
            mask = 0;
            if (x + 4 < tiles) {
                const int rows = rows_of(x + 4, page, mask);
                page = page_of(x + 8);
                if (mask) request(rows);
            }
            if (!here) {                                                      // (no page of the tile is in the pool)
                if (lm < G)
#pragma unroll
                    for (int t = 0; t < MT; ++t) *reinterpret_cast<float4_t *>(sp + j0 + t * 16 + lq * 4) = (float4_t){-INFINITY, -INFINITY, -INFINITY, -INFINITY};
                continue;
            }
            float4_t s[MT];
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                s[t] = (float4_t){0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int ks = 0; ks < NKS; ++ks) s[t] = E::mma(*reinterpret_cast<const V *>(img + (t * 16 + lm) * I::ROW + (((ks * 4 + lq) ^ (lm & SW)) << 4)), qf[ks], s[t]);
            }
            float mx = -INFINITY;                                             // scores of head lm: keys j0 + 16 t + 4 lq + e
#pragma unroll
            for (int t = 0; t < MT; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    s[t][e] = ((here >> (t * 16 + lq * 4 + e)) & 1) ? s[t][e] * scale2 : -INFINITY;
                    mx = fmaxf(mx, s[t][e]);
                }
            if (lm < G)
#pragma unroll
                for (int t = 0; t < MT; ++t) *reinterpret_cast<float4_t *>(sp + j0 + t * 16 + lq * 4) = s[t];
            mx = xor32_partner_max(xor16_partner_max(mx));
            const float mn = fmaxf(m, mx), ms = mn == -INFINITY ? 0.f : mn, alpha = __builtin_amdgcn_exp2f(m - ms);
            const bool moved = mn != m;
            m = mn;
            float rs = 0.f;
            V ph, pm;
#pragma unroll
            for (int t = 0; t < MT; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float w = __builtin_amdgcn_exp2f(s[t][e] - ms);
                    rs += w;
                    ph[t * 4 + e] = (T)w;
                    if constexpr (!F) pm[t * 4 + e] = (T)(w - (float)ph[t * 4 + e]);
                }
            l = fmaf(l, alpha, rs);
            if (__any(moved)) {
#pragma unroll
                for (int t = 0; t < DT; ++t) o[t] *= alpha;
            }
#pragma unroll
            for (int t = 0; t < DT; ++t) {
                V a;
                if constexpr (F) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) a[e] = *reinterpret_cast<const float *>(vimg + (lq * 4 + e) * I::VS + (t * 16 + lm) * 4);
                } else {
                    const char *at = vimg + (lq * 4 + (lm >> 2)) * I::VS + t * 32 + (lm & 3) * 8;
                    a = transposed<E>(at, at + 16 * I::VS);
                }
                o[t] = E::mma(a, ph, o[t]);
                if constexpr (!F) o[t] = E::mma(a, pm, o[t]);
            }
            asm volatile("" ::: "memory");
        }
        // ---- the waves' sums
        l = xor32_partner_sum(xor16_partner_sum(l));
        __syncthreads();
        float *so = reinterpret_cast<float *>(smem);
#pragma unroll
        for (int t = 0; t < DT; ++t) *reinterpret_cast<float4_t *>(so + (wave * 16 + lm) * I::OS + t * 16 + lq * 4) = o[t];
        if (lq == 0) { ml[wave][lm][0] = m; ml[wave][lm][1] = l; }
        __syncthreads();
        for (int i = threadIdx.x; i < G * (D / 4); i += 256) {
            const int h = i / (D / 4), c = (i % (D / 4)) * 4;
            float M = ml[0][h][0], L = 0.f;
#pragma unroll
            for (int i = 1; i < 4; ++i) M = fmaxf(M, ml[i][h][0]);
            const float Ms = M == -INFINITY ? 0.f : M;
            float4_t v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float f = __builtin_amdgcn_exp2f(ml[i][h][0] - Ms);
                v += *reinterpret_cast<const float4_t *>(so + (i * 16 + h) * I::OS + c) * f;
                L = fmaf(ml[i][h][1], f, L);
            }
            if constexpr (WHOLE) {
                const float n = L == 0.f ? 0.f : 1.f / L;                 // (no key: output and weights of 0)
                T *out = (T *)p.a.out + ((int64_t)b * p.a.H + g * G + h) * D + c;
#pragma unroll
                for (int e = 0; e < 4; ++e) out[e] = (T)(v[e] * n);
                if (c == 0) { big[h] = Ms; inv[h] = n; }
                continue;
            }
            const int64_t to = (int64_t)(w + b) * p.a.H + g * G + h;
            *reinterpret_cast<float4_t *>(p.o + to * D + c) = v;
            if (c == 0) { p.ml[2 * to] = M; p.ml[2 * to + 1] = L; }
        }
        if constexpr (WHOLE) {
            __syncthreads();
            const int scored = p.a.scored ? p.a.scored[b] : ctx - 1;
            for (int j = threadIdx.x; j < ctx; j += 256) {
                const int block = (int)((unsigned)j / (unsigned)p.a.block_size), page = table[block];
                if (page < 0 || page >= p.a.num_blocks) continue;
                const int64_t to = ((int64_t)page * p.a.KVH + g) * p.a.block_size + (j - block * p.a.block_size);
                float sum = 0.f;
                for (int h = 0; h < G; ++h) sum = fmaf(__builtin_amdgcn_exp2f(kept[h * p.wide + j] - big[h]), inv[h], sum);
                p.a.new_scores[to] = j < scored ? fmaf(p.a.decay, p.a.scores[to], sum) : sum;
            }
            return;
        }
        if (left > 0) __syncthreads();
    }
}

// Weights of 4 keys a thread, and the outputs of the heads that fall to this workgroup (head i of the group to the one of number i % gridDim.x)
// (four waves a workgroup: 48 sequences of up to 8100 keys 120.4 us in all, one wave 118.5)
constexpr int kJoin = 64;
template <class E>
__global__ __launch_bounds__(kJoin) void attn_scored_join_kernel(ScoredParams p) {
    typedef typename E::T T;
    constexpr int THREADS = kJoin;
    __shared__ float big[16], inv[16];
    __shared__ float4_t sums[THREADS];
    const int g = blockIdx.y, b = blockIdx.z, G = p.a.H / p.a.KVH, D = p.a.D, ctx = visible(p.a, b), tid = threadIdx.x;
    // (a sequence without keys has no ends; where none can have any, there is no workspace)
    const int j = (blockIdx.x * THREADS + tid) * 4;
    int from = 0, parts = 0;
    if (ctx > 0) { from = p.ends[2 * b]; parts = p.ends[2 * b + 1] - from + 1; }
    if ((int)blockIdx.x * THREADS * 4 >= ctx && (int)blockIdx.x >= G) return;
    const float *ml = p.ml + ((int64_t)(from + b) * p.a.H + g * G) * 2, *sp = p.s + ((int64_t)b * p.a.H + g * G) * p.lpad;
    const int32_t *table = p.a.block_tables + (int64_t)b * p.a.max_blocks;
    const int scored = p.a.scored ? p.a.scored[b] : ctx - 1, bs = p.a.block_size;
    // what the keys need is asked for first: their page (one for all four where blocks are multiples of 4), their scores, the first heads' s
    const bool one = bs % 4 == 0 && ((uintptr_t)p.a.scores & 15) == 0 && ((uintptr_t)p.a.new_scores & 15) == 0, mine = j < ctx, all = one && j + 4 <= ctx;
    const int block = (int)((unsigned)min(j, ctx - 1) / (unsigned)bs), page = mine ? table[block] : -1;
    const int64_t at = ((int64_t)page * p.a.KVH + g) * bs + (j - block * bs);
    const bool in = page >= 0 && page < p.a.num_blocks;
    float4_t old = {0.f, 0.f, 0.f, 0.f}, s[4];
    if (all && in && j < scored) old = *reinterpret_cast<const float4_t *>(p.a.scores + at);
#pragma unroll
    for (int h = 0; h < 4; ++h) s[h] = mine ? *reinterpret_cast<const float4_t *>(sp + (int64_t)min(h, G - 1) * p.lpad + j) : (float4_t){0.f, 0.f, 0.f, 0.f};
    // (maximum, sum) of each head: 16 lanes a head
    for (int h0 = 0; h0 < G; h0 += THREADS / 16) {
        const int h = h0 + (tid >> 4), n = tid & 15;
        float M = -INFINITY, L = 0.f;
        if (h < G)
            for (int i = n; i < parts; i += 16) {
                const float m = ml[((int64_t)i * p.a.H + h) * 2], l = ml[((int64_t)i * p.a.H + h) * 2 + 1], mn = fmaxf(M, m), ms = mn == -INFINITY ? 0.f : mn;
                L = fmaf(L, __builtin_amdgcn_exp2f(M - ms), l * __builtin_amdgcn_exp2f(m - ms));
                M = mn;
            }
        float mm = M;
        mm = dpp_max<0x128>(mm); mm = dpp_max<0x124>(mm); mm = dpp_max<0x4E>(mm); mm = dpp_max<0xB1>(mm);
        const float ms = mm == -INFINITY ? 0.f : mm;
        L = row_sum<16>(L * __builtin_amdgcn_exp2f(M - ms));
        if (n == 0 && h < G) { big[h] = ms; inv[h] = L == 0.f ? 0.f : 1.f / L; }      // (no key: output and weights of 0)
    }
    __syncthreads();
    if (mine) {
        float4_t w = {0.f, 0.f, 0.f, 0.f};
        for (int h0 = 0; h0 < G; h0 += 4) {
#pragma unroll
            for (int h = 0; h < 4; ++h)
                if (h0 + h < G)
#pragma unroll
                    for (int e = 0; e < 4; ++e) w[e] = fmaf(__builtin_amdgcn_exp2f(s[h][e] - big[h0 + h]), inv[h0 + h], w[e]);
            if (h0 + 4 < G)
#pragma unroll
                for (int h = 0; h < 4; ++h) s[h] = *reinterpret_cast<const float4_t *>(sp + (int64_t)min(h0 + 4 + h, G - 1) * p.lpad + j);
        }
        if (all) {
            if (in) {
                float4_t v;
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = j + e < scored ? fmaf(p.a.decay, old[e], w[e]) : w[e];
                *reinterpret_cast<float4_t *>(p.a.new_scores + at) = v;
            }
        } else
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (j + e >= ctx) break;
                const int k = (int)((unsigned)(j + e) / (unsigned)bs), pg = table[k];
                if (pg < 0 || pg >= p.a.num_blocks) continue;
                const int64_t a = ((int64_t)pg * p.a.KVH + g) * bs + (j + e - k * bs);
                p.a.new_scores[a] = j + e < scored ? fmaf(p.a.decay, p.a.scores[a], w[e]) : w[e];
            }
    }
    // outputs: D / 4 threads a head's columns, the others its parts in turn
    const int cols = D / 4, c = tid % cols, first = tid / cols, teams = THREADS / cols;
    for (int h = blockIdx.x; h < G; h += gridDim.x) {
        const float *m = ml + h * 2, *o = p.o + ((int64_t)(from + b) * p.a.H + g * G + h) * D + c * 4;
        float4_t v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
        for (int i = first; i < parts; i += teams) v += *reinterpret_cast<const float4_t *>(o + (int64_t)i * p.a.H * D) * __builtin_amdgcn_exp2f(m[(int64_t)i * p.a.H * 2] - big[h]);
        sums[tid] = v;
        __syncthreads();
        if (tid < cols) {
            for (int t = 1; t < teams; ++t) v += sums[t * cols + tid];
            T *out = (T *)p.a.out + ((int64_t)b * p.a.H + g * G + h) * D + c * 4;
#pragma unroll
            for (int e = 0; e < 4; ++e) out[e] = (T)(v[e] * inv[h]);
        }
        __syncthreads();
    }
}

namespace {
// workgroups of a kv head: two of them fit a CU (one at heads of 256), and no more than there can be units
int scored_shares(int64_t B, int64_t KVH, int64_t D, int64_t max_ctx) {
    return (int)std::max<int64_t>(1, std::min<int64_t>((D == 256 ? 256 : 512) / KVH, B * ((max_ctx + kUnit - 1) / kUnit)));
}
// one launch: up to 256 keys; up to 512 where there are sequences enough for the chip and two workgroups fit a CU
constexpr size_t kLds = 160 * 1024 - 2048;
template <class E> size_t image_of(int D) { return D == 64 ? Image<E, 64>::ALL : D == 128 ? Image<E, 128>::ALL : Image<E, 256>::ALL; }
bool whole_of(const ScoredArgs &a, int dt, int wide) {
    size_t lds = 0;
    NVR_BY_DTYPE(dt, lds = image_of<E>(a.D));
    lds += (size_t)(a.H / a.KVH) * wide * 4;
    if (a.max_ctx <= 256) return lds <= kLds;
    return a.max_ctx <= 512 && (int64_t)a.B * a.KVH >= 256 && lds <= kLds / 2;
}
struct ScoredSpace { size_t s, o, ml, ends; };
ScoredSpace scored_space(int64_t B, int64_t H, int64_t KVH, int64_t D, int64_t max_ctx, int &shares, int &lpad) {
    shares = scored_shares(B, KVH, D, max_ctx);
    lpad = (int)((max_ctx + kUnit - 1) / kUnit * kUnit);
    return ScoredSpace{(size_t)B * H * lpad * 4, (size_t)(shares + B) * H * D * 4, (size_t)(shares + B) * H * 8, (size_t)B * 8};
}
template <class E, int D, bool WHOLE>
int scored_launch(const ScoredParams &p, hipStream_t s) {
    typedef Image<E, D> I;
    constexpr size_t most = WHOLE ? kLds : I::ALL;
    const size_t lds = I::ALL + (WHOLE ? (size_t)(p.a.H / p.a.KVH) * p.wide * 4 : 0);
    if constexpr (most > 48 * 1024) {
        static std::atomic<uint64_t> allowed{0};
        if (const int rc = allow_lds("nvr_paged_attn_decode_scored", reinterpret_cast<const void *>(&attn_scored_kernel<E, D, WHOLE>), most, allowed)) return rc;
    }
    attn_scored_kernel<E, D, WHOLE><<<dim3((unsigned)p.a.KVH, (unsigned)(WHOLE ? p.a.B : p.shares)), 256, lds, s>>>(p);
    return 0;
}
}  // namespace

size_t paged_attn_scored_workspace_bytes(int64_t B, int64_t H, int64_t KVH, int64_t D, int64_t max_ctx) {
    if (B <= 0 || H <= 0 || KVH <= 0 || D <= 0 || max_ctx <= 0) return 0;
    int a, b;
    const ScoredSpace w = scored_space(B, H, KVH, D, max_ctx, a, b);
    return w.s + w.o + w.ml + w.ends;
}
int paged_attn_scored(int dt, const ScoredArgs &a, hipStream_t s) {
    const char *me = "nvr_paged_attn_decode_scored";
    if (a.B < 0 || a.H <= 0 || a.KVH <= 0 || a.H % a.KVH || a.block_size <= 0 || a.max_blocks < 0 || a.num_blocks < 0 || a.max_ctx < 0)
        return nvr::fail(NVR_ERR_INVALID_ARG, "%s: batch %d, %d heads over %d, blocks of %d", me, a.B, a.H, a.KVH, a.block_size);
    if (a.D != 64 && a.D != 128 && a.D != 256) return nvr::fail(NVR_ERR_UNSUPPORTED, "%s: head_dim %d (64, 128 or 256)", me, a.D);
    if (a.H / a.KVH > 16) return nvr::fail(NVR_ERR_UNSUPPORTED, "%s: %d query heads a kv head (up to 16)", me, a.H / a.KVH);
    if (a.num_blocks * a.block_size > 0x7fffffffll || a.B > 65535 || a.KVH > 65535 || a.max_ctx > (1 << 23)) return nvr::fail(NVR_ERR_UNSUPPORTED, "%s: a pool of 2^31 rows and more, more than 65535 sequences, or contexts beyond 2^23", me);
    if (a.B == 0) return 0;
    if (!a.q || !a.k || !a.v || !a.ctx_lens || !a.block_tables || !a.scores || !a.new_scores || !a.out || (a.max_ctx && !a.workspace))      // (without keys one launch answers, and has no use for it)
        return nvr::fail(NVR_ERR_INVALID_ARG, "%s: null argument", me);
    if (a.ldq < (int64_t)a.H * a.D) return nvr::fail(NVR_ERR_INVALID_ARG, "%s: rows of q overlap", me);
    if ((((uintptr_t)a.k | (uintptr_t)a.v | (uintptr_t)a.workspace) & 15) != 0) return nvr::fail(NVR_ERR_INVALID_ARG, "%s: caches and workspace have to be aligned to 16 bytes", me);
    ScoredParams p{};
    p.a = a;
    p.a.max_ctx = std::max(a.max_ctx, 1);
    const ScoredSpace w = scored_space(a.B, a.H, a.KVH, a.D, p.a.max_ctx, p.shares, p.lpad);
    char *at = (char *)a.workspace;
    p.s = (float *)at; p.o = (float *)(at + w.s); p.ml = (float *)(at + w.s + w.o); p.ends = (int32_t *)(at + w.s + w.o + w.ml);
    p.a.max_ctx = a.max_ctx;
    const int W = dt == DT_F32 ? 4 : 8;
    p.qw = ((uintptr_t)a.q & 15) == 0 && a.ldq % W == 0;
    p.wide = (int)(((int64_t)a.max_ctx + 31) / 32 * 32 + 4);                // (tiles of 32 keys; rows in other banks)
    int rc = 0;
    const bool whole = whole_of(a, dt, p.wide);
    if (whole) NVR_BY_DTYPE(dt, (rc = a.D == 64 ? scored_launch<E, 64, true>(p, s) : a.D == 128 ? scored_launch<E, 128, true>(p, s) : scored_launch<E, 256, true>(p, s)));
    else NVR_BY_DTYPE(dt, (rc = a.D == 64 ? scored_launch<E, 64, false>(p, s) : a.D == 128 ? scored_launch<E, 128, false>(p, s) : scored_launch<E, 256, false>(p, s)));
    if (rc) return rc;
    if (whole) {
        NVR_KX_LAUNCHED("paged_attn_scored");
        return 0;
    }
    const int64_t ctx = a.max_ctx;
    constexpr int keys = 4 * kJoin;
    const int64_t wide = std::max<int64_t>((ctx + keys - 1) / keys, a.H / a.KVH);       // (a head of the group each at least: 5 sequences of up to 60 keys, 8 heads a kv head 13.7 us with one workgroup for all)
    NVR_BY_DTYPE(dt, (attn_scored_join_kernel<E><<<dim3((unsigned)wide, (unsigned)a.KVH, (unsigned)a.B), kJoin, 0, s>>>(p)));
    NVR_KX_LAUNCHED("paged_attn_scored");
    return 0;
}

}}  // namespace nvr::kx
