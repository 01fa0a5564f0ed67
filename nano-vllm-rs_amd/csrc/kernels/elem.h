// elem.h — the three storage types of the operators that are templates over them (serving.h), 16 bytes of each at a time.
#pragma once
#include <atomic>
#include "device_utils.h"
#include "../common.h"

namespace nvr { namespace kx {

enum Dtype : int { DT_F16 = 0, DT_BF16 = 1, DT_F32 = 2 };

// T: a number in memory; V: 16 bytes of them (W numbers); KS: depth of one mma step (a lane's 16 bytes times the 4 lanes of a column).
// mma: D(16 x 16) += A(16 x KS) . B(KS x 16): lane l holds 16 bytes of row / column l & 15 of A / B, k = W (l >> 4) .. of the step, and of D column l & 15 at rows 4 (l >> 4) + e.
// Both operands take their k's in the same order, so any order will do.
struct F16 {
    typedef _Float16 T;
    typedef _Float16 V __attribute__((ext_vector_type(8)));
    static constexpr int W = 8, KS = 32;
    static __device__ __forceinline__ float4_t mma(V a, V b, float4_t c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
};
struct BF16 {
    typedef __bf16 T;
    typedef __bf16 V __attribute__((ext_vector_type(8)));
    static constexpr int W = 8, KS = 32;
    static __device__ __forceinline__ float4_t mma(V a, V b, float4_t c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
};
struct F32 {
    typedef float T;
    typedef float V __attribute__((ext_vector_type(4)));
    static constexpr int W = 4, KS = 16;
    static __device__ __forceinline__ float4_t mma(V a, V b, float4_t c) {
#pragma unroll
        for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], b[e], c, 0, 0, 0);
        return c;
    }
};

// W numbers at p, the first `n` of them there (the others 0), in one request where `whole` says that the 16 bytes are aligned
template <class E>
__device__ __forceinline__ typename E::V load16(const typename E::T *p, bool whole, int n = E::W) {
    if (whole && n >= E::W) return *reinterpret_cast<const typename E::V *>(p);
    typename E::V v;
#pragma unroll
    for (int e = 0; e < E::W; ++e) v[e] = e < n ? p[e] : (typename E::T)0.f;
    return v;
}
template <class E>
__device__ __forceinline__ typename E::V zero16() {
    typename E::V v;
#pragma unroll
    for (int e = 0; e < E::W; ++e) v[e] = (typename E::T)0.f;
    return v;
}

// Large dynamic LDS has to be allowed for a kernel on each device that runs it.  have: the devices that did (one a kernel); what failed is asked for again by the next call.  (May be captured: nothing is enqueued)
inline int allow_lds(const char *me, const void *kernel, size_t bytes, std::atomic<uint64_t> &have) {
    int device = 0;
    hipError_t e = hipGetDevice(&device);
    const uint64_t bit = 1ull << (device & 63);
    if (e == hipSuccess && (have.load(std::memory_order_acquire) & bit)) return 0;
    if (e == hipSuccess) e = hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
    if (e != hipSuccess) {
        (void)hipGetLastError();
        return nvr::fail(NVR_ERR_HIP, "%s: LDS of %zu bytes: %s", me, bytes, hipGetErrorString(e));
    }
    have.fetch_or(bit, std::memory_order_release);
    return 0;
}

#define NVR_BY_DTYPE(dt, ...)                                           \
    do {                                                                \
        if ((dt) == nvr::kx::DT_F16) { using E = nvr::kx::F16; __VA_ARGS__; }        \
        else if ((dt) == nvr::kx::DT_BF16) { using E = nvr::kx::BF16; __VA_ARGS__; } \
        else { using E = nvr::kx::F32; __VA_ARGS__; }                   \
    } while (0)

#define NVR_KX_LAUNCHED(what)                                                                                                              \
    do { hipError_t e_ = hipGetLastError(); if (e_ != hipSuccess) return nvr::fail(NVR_ERR_HIP, what " launch failed: %s", hipGetErrorString(e_)); } while (0)

}}  // namespace nvr::kx
