// rope_forms.hip — rotary positions in the forms that models use: pairs of columns half a part apart or side by side, the first `rotary`
// columns of a head alone, angles from any table of turns per position; k and v rows go on into the paged cache.
//
// (y1, y2) = amplitude (x1 cos a - x2 sin a, x1 sin a + x2 cos a), a = 2 pi frac(position * turns[pair]).  The angle is kept in turns and its whole turns are
// dropped in 64 bits: at position 10^6 a product in 32 bits is off by 0.06 radians before the sine sees it.  cos and sin are 64-bit functions rounded once to 32
// bits (a workgroup forms them once per token for all heads: 64 pairs beside 24 or more heads of 128), the rotation is in 32 bits, and the store rounds once.
//
// Bound by memory: a thread takes 16 bytes of either half of a pair, everything is read and written once.  32768 tokens of 16 + 8 + 8 heads of 128, float16: 109 us, 5.5 TB/s (a large copy: 5.1; four tokens a workgroup: 117);
// 1531 tokens of 32 + 8 + 8 heads, float32, half of each head turning: 15 us, 5.5 TB/s; 32 tokens: 3.5 us, a launch's own time.
#include <algorithm>
#include <type_traits>
#include "serving.h"
#include "elem.h"
#include "../common.h"

namespace nvr { namespace kx {

// A unit is two pieces of W numbers that turn together (W pairs), or one piece that is passed on.  Units of a token: q heads, then k heads (each `rotary / 2W` turning ones, then the rest of the
// head), then v pieces.  `tok` tokens a workgroup.
template <class E, int W>
struct Piece { typename E::T v[W]; };
template <class E, int W>
__device__ __forceinline__ void get(const typename E::T *p, float (&x)[W]) {
    if constexpr (W == E::W) {
        const typename E::V v = *reinterpret_cast<const typename E::V *>(p);
#pragma unroll
        for (int e = 0; e < W; ++e) x[e] = (float)v[e];
    } else {
#pragma unroll
        for (int e = 0; e < W; ++e) x[e] = (float)p[e];
    }
}
template <class E, int W>
__device__ __forceinline__ void put(typename E::T *p, const float (&x)[W]) {
    if constexpr (W == E::W) {
        typename E::V v;
#pragma unroll
        for (int e = 0; e < W; ++e) v[e] = (typename E::T)x[e];
        *reinterpret_cast<typename E::V *>(p) = v;
    } else {
#pragma unroll
        for (int e = 0; e < W; ++e) p[e] = (typename E::T)x[e];
    }
}

template <class E, int W, bool PAIRS, bool ONE>
__global__ __launch_bounds__(256) void rope_rotate_store_kernel(RopeArgs a, int several) {
    typedef typename E::T T;
    const int tok = ONE ? 1 : several;                                    // (compiled for one: the divisions are 2 % of large steps)
    extern __shared__ float2 turn[];                                      // [tok][rotary / 2]: cos, sin
    const int half = a.rotary / 2, D = a.D;
    const int64_t t0 = (int64_t)blockIdx.x * tok;
    const int nt = (int)min((int64_t)tok, a.T - t0);
    for (int i = threadIdx.x; i < nt * half; i += 256) {
        const int t = ONE ? 0 : i / half;
        const double at = (double)a.positions[t0 + t], per = a.turns[i - t * half];
        double s, c;
        sincospi(2.0 * fma(at, per, -rint(at * per)), &s, &c);            // (the part of a turn without a rounding of the product)
        turn[i] = make_float2((float)(c * a.amplitude), (float)(s * a.amplitude));
    }
    __syncthreads();
    const int turning = half / W, per_head = turning + (D - a.rotary) / W, hk = (a.H + a.KVH) * per_head, units = hk + (a.v_cache ? a.KVH * (D / W) : 0);
    for (int i = threadIdx.x; i < nt * units; i += 256) {
        const int t = ONE ? 0 : i / units, u = i - t * units;
        const int64_t row = t0 + t;
        int64_t slot = -1;
        if (u >= a.H * per_head && a.k_cache) { slot = a.slots[row]; if (slot >= a.num_slots) slot = -1; }
        if (u >= hk) {                                                    // v: a copy
            if (slot < 0) continue;
            const int at = (u - hk) * W;
            float x[W];
            get<E, W>((const T *)a.v + row * a.ldv + at, x);
            put<E, W>((T *)a.v_cache + slot * ((int64_t)a.KVH * D) + at, x);
            continue;
        }
        const int head = u / per_head, in = u - head * per_head;
        const bool is_k = head >= a.H;
        const int h = is_k ? head - a.H : head;
        const T *src = is_k ? (const T *)a.k + row * a.ldk + (int64_t)h * D : (const T *)a.q + row * a.ldq + (int64_t)h * D;
        T *dst = is_k ? (a.k_out ? (T *)a.k_out + row * a.ldko + (int64_t)h * D : nullptr) : (T *)a.q_out + row * a.ldqo + (int64_t)h * D;
        T *cache = slot >= 0 ? (T *)a.k_cache + (slot * a.KVH + h) * D : nullptr;
        float x[W], y[W];
        if (in < turning) {
            const int at = PAIRS ? 2 * W * in : W * in, two = PAIRS ? at + W : at + half;
            get<E, W>(src + at, x); get<E, W>(src + two, y);
            const float2 *cs = turn + t * half + W * in;
            if constexpr (PAIRS && W > 1) {                               // pairs (2 j, 2 j + 1): W / 2 of them in either piece
#pragma unroll
                for (int e = 0; e < W; e += 2) {
                    const float2 r = cs[e / 2], r2 = cs[W / 2 + e / 2];
                    const float x0 = x[e], x1 = x[e + 1], y0 = y[e], y1 = y[e + 1];
                    x[e] = fmaf(x0, r.x, -(x1 * r.y)); x[e + 1] = fmaf(x0, r.y, x1 * r.x);
                    y[e] = fmaf(y0, r2.x, -(y1 * r2.y)); y[e + 1] = fmaf(y0, r2.y, y1 * r2.x);
                }
            } else {
#pragma unroll
                for (int e = 0; e < W; ++e) {
                    const float2 r = cs[e];
                    const float x0 = x[e], x1 = y[e];
                    x[e] = fmaf(x0, r.x, -(x1 * r.y)); y[e] = fmaf(x0, r.y, x1 * r.x);
                }
            }
            if (dst) { put<E, W>(dst + at, x); put<E, W>(dst + two, y); }
            if (cache) { put<E, W>(cache + at, x); put<E, W>(cache + two, y); }
        } else {
            const int at = a.rotary + (in - turning) * W;
            get<E, W>(src + at, x);
            if (dst) put<E, W>(dst + at, x);
            if (cache) put<E, W>(cache + at, x);
        }
    }
}

template <class E>
static int rope_of(const RopeArgs &a, hipStream_t s) {
    constexpr int W = E::W;
    const uintptr_t bytes = (uintptr_t)a.q | (uintptr_t)a.k | (uintptr_t)a.v | (uintptr_t)a.q_out | (uintptr_t)a.k_out | (uintptr_t)a.k_cache | (uintptr_t)a.v_cache;
    const bool wide = (bytes & 15) == 0 && ((a.H ? a.ldq | a.ldqo : 0) | (a.KVH ? a.ldk : 0) | (a.k_out ? a.ldko : 0) | (a.v_cache ? a.ldv : 0)) % W == 0 && a.D % W == 0 && a.rotary % (2 * W) == 0;
    // tokens of a workgroup: as many as give its threads a unit each, as long as there are two workgroups a CU (8872 tokens of 2 + 2 + 2 heads of 128: 9.8 us, one a workgroup 12.4; 24 heads: 109, four 117)
    const int V = wide ? W : 1, units = (a.H + a.KVH) * (a.rotary / 2 / V + (a.D - a.rotary) / V) + (a.v_cache ? a.KVH * (a.D / V) : 0);
    const int tok = (int)std::max<int64_t>(1, std::min<int64_t>(256 / units, a.T / 512));
    const size_t lds = (size_t)tok * (a.rotary / 2) * sizeof(float2);
    const dim3 grid((unsigned)((a.T + tok - 1) / tok)), block(256);
    auto launch = [&](auto w, auto one) {
        constexpr int N = decltype(w)::value;
        constexpr bool ONE = decltype(one)::value;
        if (a.pairs) rope_rotate_store_kernel<E, N, true, ONE><<<grid, block, lds, s>>>(a, tok);
        else rope_rotate_store_kernel<E, N, false, ONE><<<grid, block, lds, s>>>(a, tok);
    };
    if (!wide) launch(std::integral_constant<int, 1>(), std::false_type());
    else if (tok == 1) launch(std::integral_constant<int, W>(), std::true_type());
    else launch(std::integral_constant<int, W>(), std::false_type());
    NVR_KX_LAUNCHED("rope_rotate_store");
    return 0;
}

int rope_rotate_store(int dt, const RopeArgs &a, hipStream_t s) {
    if (a.T < 0 || a.H < 0 || a.KVH < 0 || a.H + a.KVH <= 0 || a.D <= 0 || a.D > 1024) return nvr::fail(NVR_ERR_INVALID_ARG, "nvr_rope_rotate_store_kv: T=%ld H=%d KVH=%d D=%d", (long)a.T, a.H, a.KVH, a.D);
    if (a.rotary <= 0 || a.rotary % 2 || a.rotary > a.D) return nvr::fail(NVR_ERR_INVALID_ARG, "nvr_rope_rotate_store_kv: rotary_dim %d has to be even, 2 .. head_dim %d", a.rotary, a.D);
    if (a.T > 0x7fffffff) return nvr::fail(NVR_ERR_INVALID_ARG, "nvr_rope_rotate_store_kv: T=%ld", (long)a.T);
    if (a.T > (1 << 23)) return nvr::fail(NVR_ERR_UNSUPPORTED, "nvr_rope_rotate_store_kv: %ld tokens (up to 2^23)", (long)a.T);      // (a launch has fewer than 2^32 threads)
    if (!a.positions || !a.turns || (a.H && (!a.q || !a.q_out)) || (a.KVH && !a.k)) return nvr::fail(NVR_ERR_INVALID_ARG, "nvr_rope_rotate_store_kv: null argument");
    if (!!a.k_cache != !!a.v_cache || (a.k_cache && (!a.slots || !a.v || a.num_slots < 0))) return nvr::fail(NVR_ERR_INVALID_ARG, "nvr_rope_rotate_store_kv: both caches, v and the slots come together");
    if (a.KVH && !a.k_out && !a.k_cache) return nvr::fail(NVR_ERR_INVALID_ARG, "nvr_rope_rotate_store_kv: k goes nowhere (k_out and the caches are null)");
    if ((a.H && (a.ldq < (int64_t)a.H * a.D || a.ldqo < (int64_t)a.H * a.D)) || (a.KVH && a.ldk < (int64_t)a.KVH * a.D) || (a.k_out && a.ldko < (int64_t)a.KVH * a.D) || (a.v_cache && a.ldv < (int64_t)a.KVH * a.D))
        return nvr::fail(NVR_ERR_INVALID_ARG, "nvr_rope_rotate_store_kv: rows overlap");
    if ((a.H && a.q_out == a.q && a.ldqo != a.ldq) || (a.k_out && a.k_out == a.k && a.ldko != a.ldk)) return nvr::fail(NVR_ERR_INVALID_ARG, "nvr_rope_rotate_store_kv: in place with another stride");
    if (a.T == 0) return 0;
    NVR_BY_DTYPE(dt, return rope_of<E>(a, s));
}

}}  // namespace nvr::kx
