// Warp-level matrix products (mma.sync) and tile copies of the attention kernels that take any layout and type.
//
// 16-bit inputs: m16n8k16 with fp32 sums.  float32 inputs: every value is split into a tf32 head and a tf32 remainder and
// each product is three m16n8k8 (head x head and the two mixed ones): what is dropped is below 2^-22 of a product.  The tensor
// cores add into their accumulator with the low bits cut off, so the heads' products are summed in chains of 16 terms that are
// added up in fp32, and the mixed products, which are 2^-11 of them, in an accumulator of their own (one chain for all of
// both: gradients 1.3e-6 off where fp32 products give 0.6e-6).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>
#include <type_traits>

#include "../km_common.cuh"
#include "attention_params.h"

namespace km {
namespace att {

constexpr float LN2 = 0.6931471805599453f;
constexpr int   WARPS = 4, THREADS = 128;

template <typename T> struct Type;
template <> struct Type<float> {
    static constexpr int K = 8, CHUNK = 4;
    static __device__ __forceinline__ float to(float v) { return v; }
    static __device__ __forceinline__ float from(float v) { return v; }
};
template <> struct Type<__nv_bfloat16> {
    static constexpr int K = 16, CHUNK = 8;
    static __device__ __forceinline__ __nv_bfloat16 to(float v) { return __float2bfloat16_rn(v); }
    static __device__ __forceinline__ float from(__nv_bfloat16 v) { return __bfloat162float(v); }
    static __device__ __forceinline__ uint32_t pair(float lo, float hi) {
        uint32_t r;
        asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
        return r;
    }
};
template <> struct Type<__half> {
    static constexpr int K = 16, CHUNK = 8;
    static __device__ __forceinline__ __half to(float v) { return __float2half_rn(v); }
    static __device__ __forceinline__ float from(__half v) { return __half2float(v); }
    static __device__ __forceinline__ uint32_t pair(float lo, float hi) {
        uint32_t r;
        asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
        return r;
    }
};

template <typename T> constexpr bool is_f16 = std::is_same<T, __half>::value;

// float16 weights are multiplied by 2^8 before they are rounded, and the sums divided by it: they are at most 1 (in attention_tensor.cu 2^5), and
// float16 ends at 2^-24.  131072 keys of weight 2^-25 beside one of weight 1 are 1/256 of the result and were none of it without.
constexpr float F16_WEIGHT = 256.0f, F16_WEIGHT_LOG2 = 8.0f;
template <typename T> constexpr float weight_log2 = is_f16<T> ? F16_WEIGHT_LOG2 : 0.0f;
template <typename T> constexpr float per_weight  = is_f16<T> ? 1.0f / F16_WEIGHT : 1.0f;

// One fma forms a weight's exponent, (s - top) c.  The rounding of top c is a factor on all of a row's weights, until it leaves the type's range: where
// top c is 2^26 and more the next power of two takes the place of c, whose product with top is exact, and float16 weights stay as they are.  Scores
// there lie 4 and more apart in c, so that only weights of 2^-4 and less change, by less than the last bit of their score does.
template <typename T>
struct Exponent {
    float by, up;            // weight = 2^(s by + up - top by)
    __device__ __forceinline__ void raise(float top, float c) {
        const bool huge = fabsf(top * c) >= 0x1p26f;
        by = huge ? __uint_as_float((__float_as_uint(c) + 0x7fffffu) & 0x7f800000u) : c, up = huge ? 0.0f : weight_log2<T>;
    }
    // what sums are multiplied by at the end
    __device__ __forceinline__ float per() const { return up == 0.0f ? 1.0f : per_weight<T>; }
};

__device__ __forceinline__ uint32_t smem_addr(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }

__device__ __forceinline__ void mma_16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, const __nv_bfloat16*) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, const __half*) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_tf32(float (&d)[4], const uint32_t (&a)[4], const uint32_t (&b)[2]) {
    asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}
// A tf32 head and what it leaves, rounded to tf32.  An infinite value leaves NaN: its products are NaN, as a score of an
// infinite channel is infinite or NaN anyway and a softmax over such scores NaN.
__device__ __forceinline__ void split_tf32(float v, uint32_t& head, uint32_t& rest) {
    asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(head) : "f"(v));
    asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(rest) : "f"(v - __uint_as_float(head)));
}

__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}

// Rows of a tile in shared memory are DP channels and 16 bytes apart, so that eight rows start in different banks.
template <typename T, int DP>
struct Tile {
    static constexpr int LD = DP + Type<T>::CHUNK, CHUNKS = DP / Type<T>::CHUNK;
    static constexpr int bytes(int rows) { return rows * LD * static_cast<int>(sizeof(T)); }
};

// s[j] += A B^T for the 16 rows of A at `a` and the 8 * NT rows of B at `b`, summed over all DP channels.
template <typename T, int DP, int NT>
__device__ __forceinline__ void product_nt(float (&s)[NT][4], const T* a, const T* b) {
    constexpr int LD = Tile<T, DP>::LD;
    const int     lane = threadIdx.x & 31;
    if constexpr (sizeof(T) == 2) {
        static_assert(NT % 2 == 0, "tiles are read in pairs");
        const uint32_t pa = smem_addr(a + (lane & 15) * LD + (lane >> 4) * 8);
        const uint32_t pb = smem_addr(b + ((lane & 7) + (lane >> 4) * 8) * LD + ((lane >> 3) & 1) * 8);
#pragma unroll
        for (int k = 0; k < DP / 16; ++k) {
            uint32_t fa[4];
            ldmatrix4(fa, pa + k * 32);
#pragma unroll
            for (int j = 0; j < NT; j += 2) {
                uint32_t fb[4];
                ldmatrix4(fb, pb + (j * 8 * LD + k * 16) * 2);
                mma_16(s[j], fa, fb[0], fb[1], a);
                mma_16(s[j + 1], fa, fb[2], fb[3], a);
            }
        }
    } else {
        const int g = lane >> 2, t = lane & 3;
        const float* pa = a + g * LD + t;
        const float* pb = b + g * LD + t;
        float mixed[NT][4];
#pragma unroll
        for (int j = 0; j < NT; ++j) mixed[j][0] = mixed[j][1] = mixed[j][2] = mixed[j][3] = 0.0f;
#pragma unroll 2
        for (int k = 0; k < DP / 8; k += 2) {
            uint32_t head[2][4], rest[2][4];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                split_tf32(pa[(k + i) * 8], head[i][0], rest[i][0]);
                split_tf32(pa[(k + i) * 8 + 8 * LD], head[i][1], rest[i][1]);
                split_tf32(pa[(k + i) * 8 + 4], head[i][2], rest[i][2]);
                split_tf32(pa[(k + i) * 8 + 8 * LD + 4], head[i][3], rest[i][3]);
            }
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    uint32_t bh[2], br[2];
                    split_tf32(pb[j * 8 * LD + (k + i) * 8], bh[0], br[0]);
                    split_tf32(pb[j * 8 * LD + (k + i) * 8 + 4], bh[1], br[1]);
                    mma_tf32(mixed[j], rest[i], bh);
                    mma_tf32(mixed[j], head[i], br);
                    mma_tf32(sum, head[i], bh);
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) s[j][e] += sum[e];
            }
        }
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[j][e] += mixed[j][e];
    }
}

// o[c] += P B for the 16 x (8 * NT) values p in the layout that product_nt leaves and the 8 * NT rows of B at `b`,
// channels [0, 8 * CT).
template <typename T, int DP, int NT, int CT>
__device__ __forceinline__ void product_nn(float (&o)[CT][4], const float (&p)[NT][4], const T* b) {
    constexpr int LD = Tile<T, DP>::LD;
    const int     lane = threadIdx.x & 31;
    if constexpr (sizeof(T) == 2) {
        const uint32_t pb = smem_addr(b + (lane & 15) * LD + (lane >> 4) * 8);
#pragma unroll
        for (int j = 0; j < NT; j += 2) {
            // P is rounded to the inputs' 16 bits for the tensor cores: half a step of each weight, independent of the sign
            const uint32_t fa[4] = {Type<T>::pair(p[j][0], p[j][1]), Type<T>::pair(p[j][2], p[j][3]),
                                    Type<T>::pair(p[j + 1][0], p[j + 1][1]), Type<T>::pair(p[j + 1][2], p[j + 1][3])};
#pragma unroll
            for (int c = 0; c < CT; c += 2) {
                uint32_t fb[4];
                ldmatrix4_trans(fb, pb + (j * 8 * LD + c * 8) * 2);
                mma_16(o[c], fa, fb[0], fb[1], b);
                mma_16(o[c + 1], fa, fb[2], fb[3], b);
            }
        }
    } else {
        // The order of a sum's terms is free: fragment column t stands for row 2t of B and column t + 4 for row 2t + 1,
        // which is how product_nt leaves p, so no value changes lanes.
        const int g = lane >> 2, t = lane & 3;
        uint32_t head[NT][4], rest[NT][4];
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            split_tf32(p[j][0], head[j][0], rest[j][0]);
            split_tf32(p[j][2], head[j][1], rest[j][1]);
            split_tf32(p[j][1], head[j][2], rest[j][2]);
            split_tf32(p[j][3], head[j][3], rest[j][3]);
        }
        const float* pb = b + 2 * t * LD + g;
#pragma unroll
        for (int c = 0; c < CT; ++c) {
            float mixed[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int j = 0; j < NT; j += 2) {
                float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int i = j; i < j + 2 && i < NT; ++i) {
                    uint32_t bh[2], br[2];
                    split_tf32(pb[i * 8 * LD + c * 8], bh[0], br[0]);
                    split_tf32(pb[i * 8 * LD + LD + c * 8], bh[1], br[1]);
                    mma_tf32(mixed, rest[i], bh);
                    mma_tf32(mixed, head[i], br);
                    mma_tf32(sum, head[i], bh);
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) o[c][e] += sum[e];
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) o[c][e] += mixed[e];
        }
    }
}

// 16 bytes of shared memory from `src`, or zeros.
__device__ __forceinline__ void copy_async_16(uint32_t dst, const void* src, bool valid) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy_async_4(uint32_t dst, const void* src, bool valid) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(valid ? 4 : 0) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// One 16-byte chunk (channels [c, c + CHUNK)) of a row into shared memory; channels beyond D and rows that are not there
// (row == nullptr) become zeros, and nothing is read for them.
template <typename T>
__device__ __forceinline__ void copy_chunk(T* dst, const T* row, const T* fallback, int c, int D, bool vec) {
    if (vec) {
        const bool valid = row != nullptr && c < D;
        copy_async_16(smem_addr(dst), valid ? static_cast<const void*>(row + c) : static_cast<const void*>(fallback), valid);
    } else {
        T x[Type<T>::CHUNK];
#pragma unroll
        for (int i = 0; i < Type<T>::CHUNK; ++i) x[i] = (row != nullptr && c + i < D) ? row[c + i] : Type<T>::to(0.0f);
        *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(x);
    }
}

// Rows [first, first + rows) of one head into a tile; those from `end` on are zeros and are not read.  Called by `threads`
// threads with their index.
template <typename T, int DP>
__device__ __forceinline__ void copy_rows(T* dst, const T* base, long long stride, int first, int end, int rows, int D, bool vec,
                                          int index, int threads) {
    constexpr int CHUNKS = Tile<T, DP>::CHUNKS, LD = Tile<T, DP>::LD;
    for (int i = index; i < rows * CHUNKS; i += threads) {
        const int r = i / CHUNKS, c = (i % CHUNKS) * Type<T>::CHUNK;
        copy_chunk(dst + r * LD + c, first + r < end ? base + (first + r) * stride : nullptr, base, c, D, vec);
    }
}

__device__ __forceinline__ int key_count(const int* lengths, long long stride, int l, int M) {
    if (!lengths) return M;
    const int n = lengths[l * stride];
    return n < 0 ? 0 : n > M ? M : n;
}

// Sum and maximum over the four lanes that hold one row.
__device__ __forceinline__ float quad_max(float v) {
    v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 1));
    return fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 2));
}
__device__ __forceinline__ float quad_sum(float v) {
    v += __shfl_xor_sync(0xffffffffu, v, 1);
    return v + __shfl_xor_sync(0xffffffffu, v, 2);
}

}  // namespace att
}  // namespace km
