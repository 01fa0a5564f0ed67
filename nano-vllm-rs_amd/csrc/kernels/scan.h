// scan.h — prefix sums of a wave and of a workgroup by moves between lanes (DPP): a step is one or two instructions, a shuffle through LDS some 60 cycles.
#pragma once
#include <hip/hip_runtime.h>

namespace nvr { namespace kx {

// x of the lane that CTRL names, 0 where there is none or the row is not in ROWS (32 and 64 bits)
template <int CTRL, int ROWS, class T>
__device__ __forceinline__ T moved(T x) {
    if constexpr (sizeof(T) == 4) {
        return __builtin_bit_cast(T, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, ROWS, 0xf, false));
    } else {
        const long long v = __builtin_bit_cast(long long, x);
        const unsigned int lo = (unsigned int)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xf, false), hi = (unsigned int)__builtin_amdgcn_update_dpp(0, (int)(v >> 32), CTRL, ROWS, 0xf, false);
        return __builtin_bit_cast(T, (long long)(((unsigned long long)hi << 32) | lo));
    }
}
template <class T>
__device__ __forceinline__ T row_scan(T v) {                              // over the lanes of a row of 16 up to and with this one: row_shr 1, 2, 4, 8
    v += moved<0x111, 0xf>(v); v += moved<0x112, 0xf>(v); v += moved<0x114, 0xf>(v); v += moved<0x118, 0xf>(v);
    return v;
}
template <class T>
__device__ __forceinline__ T from_lane(T x, int l) {
    if constexpr (sizeof(T) == 4) return __builtin_bit_cast(T, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), l));
    else {
        const long long v = __builtin_bit_cast(long long, x);
        const unsigned int lo = (unsigned int)__builtin_amdgcn_readlane((int)v, l), hi = (unsigned int)__builtin_amdgcn_readlane((int)(v >> 32), l);
        return __builtin_bit_cast(T, (long long)(((unsigned long long)hi << 32) | lo));
    }
}
template <class T>
__device__ __forceinline__ T wave_scan(T v) {                             // ... of the wave: the rows' last lanes to the rows behind (row_bcast 15 and 31)
    v = row_scan(v);
    v += moved<0x142, 0xa>(v); v += moved<0x143, 0xc>(v);
    return v;
}
// sum over the threads up to and with this one; `waves`: one of LDS a wave (16 at most)
template <class T>
__device__ __forceinline__ T scan(T v, T *waves) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    v = wave_scan(v);
    __syncthreads();
    if (lane == 63) waves[wave] = v;
    __syncthreads();
    return from_lane(row_scan(lane < wave ? waves[lane & 15] : (T)0), 15) + v;
}
// x where every lane has the same: in scalar registers (what comes out of LDS the compiler takes for different ones, and branches on it for a branch a lane)
template <class T>
__device__ __forceinline__ T same(T x) { return from_lane(x, 0); }

}}  // namespace nvr::kx
