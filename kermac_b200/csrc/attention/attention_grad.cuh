// What the gradient kernels share: the factor that keeps float16 in range, and where gradients are written.
#pragma once

#include "attention_mma.cuh"

namespace km {
namespace att {

// What a weight's gradient ds = p (dout v^T - delta) is multiplied by before it is rounded to float16; the sums are divided by it.
// |dout v^T| and |delta| are at most x = D max|dout| max|v|, over the keys that are seen: with 2^13 over the power of two at or below x the product
// stays below 2^15, half of what float16 has, and a ds of 2^-27 x still has all its bits (dout v^T of random signs is some 2^-7 x at 128
// channels, which leaves 2^-20 for p).  From |dout| alone, which this was once, keys of +-1200 in 128 channels became infinite, and v of size 0.01
// before 5000 keys gave four times the error of rounding.
// 1 where x is zero, and for the types that have the range.
template <typename T>
__device__ __forceinline__ float factor_for(float x) {
    if constexpr (!is_f16<T>) return 1.0f;
    const uint32_t e = __float_as_uint(x) >> 23;                         // x is zero or 2^-48 .. 2^40
    return x > 0.0f ? __uint_as_float((267u - e) << 23) : 1.0f;
}
__device__ __forceinline__ float warp_max(float best) {
#pragma unroll
    for (int d = 16; d; d >>= 1) best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, d));
    return best;
}
// The largest |v| among the first `count` keys of a head; 0 for the types that need none.  Called by whole warps, each for itself.
template <typename T>
__device__ __forceinline__ float find_v_peak(const AttentionGradParams& p, int kl, int hk, int count) {
    if constexpr (!is_f16<T>) return 0.0f;
    const float* from = p.v_peaks + (static_cast<long long>(kl) * p.Hk + hk) * p.v_peak_count;
    const int    many = (count + ATT_PEAK_ROWS - 1) / ATT_PEAK_ROWS;
    float        best = 0.0f;
#pragma unroll 4
    for (int i = threadIdx.x & 31; i < many; i += 32) best = fmaxf(best, from[i]);
    return warp_max(best);
}
// For a row of dq, whose sum is its own.
template <typename T>
__device__ __forceinline__ float row_factor(const AttentionGradParams& p, int l, int h, int n, float v_peak) {
    if constexpr (!is_f16<T>) return 1.0f;
    return n < p.N ? factor_for<T>(p.D * p.peaks[(static_cast<long long>(l) * p.H + h) * p.peak_count + n / ATT_PEAK_ROWS] * v_peak) : 1.0f;
}
// One factor for a sum over the queries of entries [l0, l1) and the heads of a group, and `count` keys.
template <typename T>
__device__ __forceinline__ float find_factor(const AttentionGradParams& p, int l0, int l1, int hk, int kl, int count) {
    if constexpr (!is_f16<T>) return 1.0f;
    const int per_l = p.G * p.peak_count;        // neighbours
    float     best  = 0.0f;
#pragma unroll 4
    for (int i = threadIdx.x & 31; i < (l1 - l0) * per_l; i += 32) {
        const int l = i / per_l;
        best = fmaxf(best, p.peaks[(static_cast<long long>(l0 + l) * p.H + hk * p.G) * p.peak_count + i - l * per_l]);
    }
    return factor_for<T>(p.D * warp_max(best) * find_v_peak<T>(p, kl, hk, count));
}

template <typename T>
__device__ __forceinline__ const T* head_of(const Heads& t, int l, int h) {
    return reinterpret_cast<const T*>(t.ptr) + l * t.sl + h * t.sh;
}

// Channels (c, c + 1) of a gradient: into the tensor, or into a slice's 32-bit sums [l][row][head][D].
template <typename T>
__device__ __forceinline__ void put_grad(const Heads& to, float* part, int l, int row, int h, int rows, int heads, int D, int c,
                                         float x, float y) {
    if (c >= D) return;
    if (part) {
        float* o = part + ((static_cast<long long>(l) * rows + row) * heads + h) * D + c;
        o[0] = x;
        if (c + 1 < D) o[1] = y;
    } else {
        T* o = reinterpret_cast<T*>(to.ptr) + l * to.sl + row * to.sr + h * to.sh + c;
        o[0] = Type<T>::to(x);
        if (c + 1 < D) o[1] = Type<T>::to(y);
    }
}

}  // namespace att
}  // namespace km
