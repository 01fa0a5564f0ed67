// attention_scored.hip — decode attention over the paged cache that also adds each key's attention weight, summed over the query heads of its kv head, to the key's score.
//
//   s_hj = scale q_h . k_j,  w_hj = exp(s_hj - M_h) / L_h,  out_h = sum_j w_hj v_j,  score'_gj = decay score_gj (keys j < scored_lens) + sum over the heads h of g of w_hj
//
// A weight is known when the row's maximum and sum are, that is behind the last key.  So the first launch is a split decode attention that reads K and V once and leaves its scores s in the
// workspace (4 bytes a key and head beside the 4 D bytes of the key's rows), and the second turns them into weights: it merges the partitions' (maximum, sum), updates the scores, and joins the
// partitions' outputs.  Bound by the stream of K and V.
// First launch: a workgroup of four waves takes a part of one (sequence, kv head)'s keys; a wave takes tiles of TK keys on the matrix cores, the heads of the group (up to 16) as columns:
// S^T = K Q^T, O^T += V^T P^T.  Rows come from the pages whole (16 bytes a lane, the next tile's in flight) and pass through the wave's own LDS image into the layout of the operands.  Weights
// enter the second product as two 16-bit numbers, the rounded weight and the rounded rest, so that they have 17 (bfloat16) or 22 bits there: the cores are idle most of the time anyway.
#include <algorithm>
#include "serving.h"
#include "elem.h"
#include "../common.h"

namespace nvr { namespace kx {

namespace {
constexpr float kLog2e = 1.44269504088896340736f;
struct ScoredParams {
    ScoredArgs a;
    int32_t part, parts, lpad;                                            // keys of a part, parts of the longest context, scores of a head in the workspace
    float *s, *ml, *o;                                                    // [B][H][lpad], [B][H][parts][2], [B][H][parts][D]
    bool qw;
};
// keys that the attention may look at
__device__ __forceinline__ int visible(const ScoredArgs &a, int b) {
    const long long most = (long long)a.max_blocks * a.block_size;
    int n = a.ctx_lens[b];
    n = min(n, a.max_ctx);
    return (int)max(0ll, min((long long)n, most));
}
// row of the pool of key j (< 0: its page is not in the pool)
__device__ __forceinline__ int pool_row(const ScoredArgs &a, const int32_t *table, int j) {
    const int block = (int)((unsigned)j / (unsigned)a.block_size), page = table[block];
    return page >= 0 && page < a.num_blocks ? page * a.block_size + (j - block * a.block_size) : -1;
}
template <class E, int D>
struct Image {
    static constexpr int TK = sizeof(typename E::T) == 4 ? 16 : 32;                                   // keys of a tile
    static constexpr int ROW = D * (int)sizeof(typename E::T), LPR = ROW / 16, RPI = 64 / LPR, NI = TK / RPI;   // bytes of a row, lanes of it, rows of a request, requests of a tile
    static constexpr int VS = ROW + (sizeof(typename E::T) == 4 ? 16 : 32);                           // V: stride of a row (conflict-free transposed reads)
    static constexpr int BYTES = TK * VS, OS = D + 4;
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

template <class E, int D>
__global__ __launch_bounds__(256) void attn_scored_kernel(ScoredParams p) {
    typedef typename E::T T; typedef typename E::V V;
    typedef Image<E, D> I;
    constexpr bool F = sizeof(T) == 4;
    constexpr int MT = I::TK / 16, NKS = D / E::KS, DT = D / 16;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    __shared__ float ml[4][16][2];
    const int part = blockIdx.x, g = blockIdx.y, b = blockIdx.z;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, lm = lane & 15, lq = lane >> 4;
    const int G = p.a.H / p.a.KVH, ctx = visible(p.a, b), first = part * p.part, last = min(ctx, first + p.part);
    if (first >= last) return;                                            // (the second launch looks at the parts that there are)
    const int32_t *table = p.a.block_tables + (int64_t)b * p.a.max_blocks;
    const float scale2 = p.a.scale * kLog2e;
    const int64_t row_elems = (int64_t)p.a.KVH * D;
    const T *kc = (const T *)p.a.k + (int64_t)g * D, *vc = (const T *)p.a.v + (int64_t)g * D;
    char *img = smem + wave * I::BYTES;
    V qf[NKS];                                                            // column lm: head lm of the group (none behind the last: 0)
    {
        const T *q = (const T *)p.a.q + (int64_t)b * p.a.ldq + (int64_t)(g * G + min(lm, G - 1)) * D + lq * E::W;
#pragma unroll
        for (int ks = 0; ks < NKS; ++ks) qf[ks] = lm < G ? load16<E>(q + ks * E::KS, p.qw) : zero16<E>();
    }
    const int rl = lane / I::LPR, pl = lane % I::LPR;                     // this lane's row of a request and its piece
    // a tile's rows of the pool, key `lane` of it; those that are not there take another's row (their scores are -inf and their values 0)
    auto rows_of = [&](int tile, unsigned int &mask) {
        const int j = first + tile * I::TK + (lane & (I::TK - 1));
        const int r = j < last ? pool_row(p.a, table, j) : -1;
        mask = (unsigned int)__ballot(r >= 0 && lane < I::TK);
        return r >= 0 ? r : mask ? __shfl(r, __ffs(mask) - 1) : -1;
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
    unsigned int mask = 0, next_mask = 0;
    constexpr unsigned int kAll = I::TK == 32 ? 0xffffffffu : 0xffffu;
    int rows = wave < tiles ? rows_of(wave, mask) : -1;
    if (mask) request(rows);
    float *sp = p.s + ((int64_t)b * p.a.H + g * G + lm) * p.lpad;
    for (int x = wave; x < tiles; x += 4) {
        const int next = x + 4;
        int next_rows = -1;
        next_mask = 0;
        if (next < tiles) next_rows = rows_of(next, next_mask);
        const int j0 = first + x * I::TK;
        if (!mask) {                                                      // (no page of the tile is in the pool)
            if (lm < G)
#pragma unroll
                for (int t = 0; t < MT; ++t) *reinterpret_cast<float4_t *>(sp + j0 + t * 16 + lq * 4) = (float4_t){-INFINITY, -INFINITY, -INFINITY, -INFINITY};
            rows = next_rows; mask = next_mask;
            if (mask) request(rows);
            continue;
        }
        // K through the image: piece c of row r at slot c ^ (r & 15) (or & 7: rows of eight pieces)
        constexpr int SW = I::LPR >= 16 ? 15 : I::LPR - 1;
#pragma unroll
        for (int u = 0; u < I::NI; ++u) { const int r = u * I::RPI + rl; *reinterpret_cast<V *>(img + r * I::ROW + ((pl ^ (r & SW)) << 4)) = kx[u]; }
        asm volatile("" ::: "memory");                                    // (a wave's LDS requests are served in order)
        float4_t s[MT];
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            s[t] = (float4_t){0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int ks = 0; ks < NKS; ++ks) s[t] = E::mma(*reinterpret_cast<const V *>(img + (t * 16 + lm) * I::ROW + (((ks * 4 + lq) ^ (lm & SW)) << 4)), qf[ks], s[t]);
        }
        asm volatile("" ::: "memory");
        if (mask != kAll)
#pragma unroll
            for (int u = 0; u < I::NI; ++u) if (!((mask >> (u * I::RPI + rl)) & 1)) vx[u] = zero16<E>();
#pragma unroll
        for (int u = 0; u < I::NI; ++u) *reinterpret_cast<V *>(img + (u * I::RPI + rl) * I::VS + pl * 16) = vx[u];
        asm volatile("" ::: "memory");
        if (next_mask) request(next_rows);
        float mx = -INFINITY;                                             // scores of head lm: keys j0 + 16 t + 4 lq + e
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                s[t][e] = ((mask >> (t * 16 + lq * 4 + e)) & 1) ? s[t][e] * scale2 : -INFINITY;
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
                for (int e = 0; e < 4; ++e) a[e] = *reinterpret_cast<const float *>(img + (lq * 4 + e) * I::VS + (t * 16 + lm) * 4);
            } else {
                const char *at = img + (lq * 4 + (lm >> 2)) * I::VS + t * 32 + (lm & 3) * 8;
                a = transposed<E>(at, at + 16 * I::VS);
            }
            o[t] = E::mma(a, ph, o[t]);
            if constexpr (!F) o[t] = E::mma(a, pm, o[t]);
        }
        asm volatile("" ::: "memory");
        rows = next_rows; mask = next_mask;
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
        for (int w = 1; w < 4; ++w) M = fmaxf(M, ml[w][h][0]);
        const float Ms = M == -INFINITY ? 0.f : M;
        float4_t v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float f = __builtin_amdgcn_exp2f(ml[w][h][0] - Ms);
            v += *reinterpret_cast<const float4_t *>(so + (w * 16 + h) * I::OS + c) * f;
            L = fmaf(ml[w][h][1], f, L);
        }
        const int64_t at = ((int64_t)b * p.a.H + g * G + h) * p.parts + part;
        *reinterpret_cast<float4_t *>(p.o + at * D + c) = v;
        if (c == 0) { p.ml[2 * at] = M; p.ml[2 * at + 1] = L; }
    }
}

// Weights of 4 keys a thread, and the outputs of the heads that fall to this workgroup (head i of the group to the one of number i % gridDim.x)
template <class E>
__global__ __launch_bounds__(256) void attn_scored_join_kernel(ScoredParams p, int keys) {
    typedef typename E::T T;
    __shared__ float big[16], inv[16];
    const int g = blockIdx.y, b = blockIdx.z, G = p.a.H / p.a.KVH, D = p.a.D, ctx = visible(p.a, b), tid = threadIdx.x;
    const int parts = (ctx + p.part - 1) / p.part;
    const float *ml = p.ml + ((int64_t)b * p.a.H + g * G) * p.parts * 2;
    const int j0 = blockIdx.x * keys;
    if (j0 >= ctx && (int)blockIdx.x >= G) return;
    // (maximum, sum) of each head: 16 lanes a head
    {
        const int h = tid >> 4, n = tid & 15;
        float M = -INFINITY, L = 0.f;
        if (h < G)
            for (int i = n; i < parts; i += 16) {
                const float m = ml[((int64_t)h * p.parts + i) * 2], l = ml[((int64_t)h * p.parts + i) * 2 + 1], mn = fmaxf(M, m), ms = mn == -INFINITY ? 0.f : mn;
                L = fmaf(L, __builtin_amdgcn_exp2f(M - ms), l * __builtin_amdgcn_exp2f(m - ms));
                M = mn;
            }
#pragma unroll
        for (int d = 8; d > 0; d >>= 1) {
            const float m = __shfl_xor(M, d), l = __shfl_xor(L, d), mn = fmaxf(M, m), ms = mn == -INFINITY ? 0.f : mn;
            L = L * __builtin_amdgcn_exp2f(M - ms) + l * __builtin_amdgcn_exp2f(m - ms);
            M = mn;
        }
        if (n == 0) { big[h] = M == -INFINITY ? 0.f : M; inv[h] = L == 0.f ? 0.f : 1.f / L; }       // (no key: output and weights of 0)
    }
    __syncthreads();
    const int32_t *table = p.a.block_tables + (int64_t)b * p.a.max_blocks;
    const int scored = p.a.scored ? p.a.scored[b] : ctx - 1;
    const float *sp = p.s + ((int64_t)b * p.a.H + g * G) * p.lpad;
    for (int j = j0 + tid * 4; j < min(ctx, j0 + keys); j += 1024) {
        float4_t w = {0.f, 0.f, 0.f, 0.f};
        for (int h = 0; h < G; ++h) {
            const float4_t s = *reinterpret_cast<const float4_t *>(sp + (int64_t)h * p.lpad + j);
#pragma unroll
            for (int e = 0; e < 4; ++e) w[e] = fmaf(__builtin_amdgcn_exp2f(s[e] - big[h]), inv[h], w[e]);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (j + e >= ctx) break;
            const int r = pool_row(p.a, table, j + e);
            if (r < 0) continue;
            const int block = r / p.a.block_size;
            const int64_t at = ((int64_t)block * p.a.KVH + g) * p.a.block_size + (r - block * p.a.block_size);
            p.a.new_scores[at] = j + e < scored ? fmaf(p.a.decay, p.a.scores[at], w[e]) : w[e];
        }
    }
    for (int h = blockIdx.x; h < G; h += gridDim.x) {
        const float *m = ml + (int64_t)h * p.parts * 2, *o = p.o + ((int64_t)b * p.a.H + g * G + h) * p.parts * D;
        for (int c = tid; c < D; c += 256) {
            float v = 0.f;
            for (int i = 0; i < parts; ++i) v = fmaf(o[(int64_t)i * D + c], __builtin_amdgcn_exp2f(m[2 * i] - big[h]), v);
            ((T *)p.a.out)[((int64_t)b * p.a.H + g * G + h) * D + c] = (T)(v * inv[h]);
        }
    }
}

namespace {
// keys of a part: 512, or as few as fill the chip (two workgroups a CU), 128 at least (a tile a wave)
int scored_part(int64_t B, int64_t KVH, int64_t max_ctx) {
    int part = 512;
    while (part > 128 && B * KVH * ((max_ctx + part - 1) / part) < 512) part /= 2;
    return part;
}
struct ScoredSpace { size_t s, ml, o; };
ScoredSpace scored_space(int64_t B, int64_t H, int64_t KVH, int64_t D, int64_t max_ctx, int &part, int &parts, int &lpad) {
    part = scored_part(B, KVH, max_ctx);
    parts = (int)((max_ctx + part - 1) / part);
    lpad = (int)((max_ctx + 31) / 32 * 32);
    return ScoredSpace{(size_t)B * H * lpad * 4, (size_t)((B * H * parts * 8 + 15) / 16 * 16), (size_t)B * H * parts * D * 4};
}
template <class E, int D>
int scored_launch(const ScoredParams &p, hipStream_t s) {
    typedef Image<E, D> I;
    constexpr size_t lds = 4 * I::BYTES > 4 * 16 * I::OS * 4 ? 4 * I::BYTES : 4 * 16 * I::OS * 4;
    if constexpr (lds > 48 * 1024) {
        static const hipError_t opted = hipFuncSetAttribute(reinterpret_cast<const void *>(&attn_scored_kernel<E, D>), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
        if (opted != hipSuccess) return nvr::fail(NVR_ERR_HIP, "nvr_paged_attn_decode_scored: LDS of %zu bytes: %s", lds, hipGetErrorString(opted));
    }
    attn_scored_kernel<E, D><<<dim3((unsigned)p.parts, (unsigned)p.a.KVH, (unsigned)p.a.B), 256, lds, s>>>(p);
    return 0;
}
}  // namespace

size_t paged_attn_scored_workspace_bytes(int64_t B, int64_t H, int64_t KVH, int64_t D, int64_t max_ctx) {
    if (B <= 0 || H <= 0 || KVH <= 0 || D <= 0 || max_ctx <= 0) return 0;
    int a, b, c;
    const ScoredSpace w = scored_space(B, H, KVH, D, max_ctx, a, b, c);
    return w.s + w.ml + w.o;
}
int paged_attn_scored(int dt, const ScoredArgs &a, hipStream_t s) {
    const char *me = "nvr_paged_attn_decode_scored";
    if (a.B < 0 || a.H <= 0 || a.KVH <= 0 || a.H % a.KVH || a.block_size <= 0 || a.max_blocks < 0 || a.num_blocks < 0 || a.max_ctx < 0)
        return nvr::fail(NVR_ERR_INVALID_ARG, "%s: batch %d, %d heads over %d, blocks of %d", me, a.B, a.H, a.KVH, a.block_size);
    if (a.D != 64 && a.D != 128 && a.D != 256) return nvr::fail(NVR_ERR_UNSUPPORTED, "%s: head_dim %d (64, 128 or 256)", me, a.D);
    if (a.H / a.KVH > 16) return nvr::fail(NVR_ERR_UNSUPPORTED, "%s: %d query heads a kv head (up to 16)", me, a.H / a.KVH);
    if (a.num_blocks * a.block_size > 0x7fffffffll || a.B > 65535 || a.KVH > 65535 || a.max_ctx > (1 << 30)) return nvr::fail(NVR_ERR_UNSUPPORTED, "%s: a pool of 2^31 rows and more, or more than 65535 sequences", me);
    if (a.B == 0) return 0;
    if (!a.q || !a.k || !a.v || !a.ctx_lens || !a.block_tables || !a.scores || !a.new_scores || !a.out || !a.workspace) return nvr::fail(NVR_ERR_INVALID_ARG, "%s: null argument", me);
    if (a.ldq < (int64_t)a.H * a.D) return nvr::fail(NVR_ERR_INVALID_ARG, "%s: rows of q overlap", me);
    if ((((uintptr_t)a.k | (uintptr_t)a.v | (uintptr_t)a.workspace) & 15) != 0) return nvr::fail(NVR_ERR_INVALID_ARG, "%s: caches and workspace have to be aligned to 16 bytes", me);
    ScoredParams p{};
    p.a = a;
    p.a.max_ctx = std::max(a.max_ctx, 1);
    const ScoredSpace w = scored_space(a.B, a.H, a.KVH, a.D, p.a.max_ctx, p.part, p.parts, p.lpad);
    p.s = (float *)a.workspace; p.ml = (float *)((char *)a.workspace + w.s); p.o = (float *)((char *)a.workspace + w.s + w.ml);
    p.a.max_ctx = a.max_ctx;
    const int W = dt == DT_F32 ? 4 : 8;
    p.qw = ((uintptr_t)a.q & 15) == 0 && a.ldq % W == 0;
    int rc = 0;
    NVR_BY_DTYPE(dt, rc = a.D == 64 ? scored_launch<E, 64>(p, s) : a.D == 128 ? scored_launch<E, 128>(p, s) : scored_launch<E, 256>(p, s));
    if (rc) return rc;
    const int keys = 1024;
    const dim3 grid((unsigned)((std::max(a.max_ctx, 1) + keys - 1) / keys), (unsigned)a.KVH, (unsigned)a.B);
    NVR_BY_DTYPE(dt, (attn_scored_join_kernel<E><<<grid, 256, 0, s>>>(p, keys)));
    NVR_KX_LAUNCHED("paged_attn_scored");
    return 0;
}

}}  // namespace nvr::kx
