// What the gradient kernels share: the factor that keeps float16 in range, and where gradients are written.
#pragma once

#include "attention_mma.cuh"

namespace km {
namespace att {

// float16 weights are multiplied by this before they are rounded: they are at most 1, and float16 ends at 6e-8.
constexpr float F16_WEIGHT = 256.0f, F16_WEIGHT_LOG2 = 8.0f;

template <typename T> constexpr bool is_f16 = std::is_same<T, __half>::value;

// 2^-e with 2^e the power of two at or below the largest of the peaks of entries [l0, l1) and heads [h0, h1); 1 when they are zero,
// infinite or NaN, and for the types that have the range.  Called by whole warps, each for itself.
template <typename T>
__device__ __forceinline__ float find_factor(const AttentionGradParams& p, int l0, int l1, int h0, int h1) {
    if constexpr (!is_f16<T>) {
        return 1.0f;
    } else {
        float     best  = 0.0f;
        const int per_l = (h1 - h0) * p.peak_count;
        for (int l = l0; l < l1; ++l)
            for (int i = threadIdx.x & 31; i < per_l; i += 32)
                best = fmaxf(best, p.peaks[(static_cast<long long>(l) * p.H + h0) * p.peak_count + i]);
#pragma unroll
        for (int d = 16; d; d >>= 1) best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, d));
        const uint32_t e = __float_as_uint(best) >> 23;                  // best is a float16 magnitude: 2^-24 .. 65504
        return (best > 0.0f && e < 255) ? __uint_as_float((254u - e) << 23) : 1.0f;
    }
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
