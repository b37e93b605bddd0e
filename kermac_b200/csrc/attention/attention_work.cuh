// What one block of a forward kernel computes, and where its results go.
#pragma once

#include "attention_mma.cuh"

namespace km {
namespace att {

// What one block computes.
struct Work {
    const char *k, *v;            // first key of the head
    long long   k_sr, v_sr;
    int         l, hk;            // l: the batch entry, or -1 for rows of all entries
    int         row0, rows;       // rows of the (l, key head) matrix, and how many there are
    int         first, end;       // keys
    int         length, part;
    bool        causal;
};

// The batch entry with the rank-th longest sequence, so that blocks that start first have the most to do (a tail of long ones costs a
// third of a launch of two rounds).  Called by a whole block of BLOCK threads; more than LPT_MOST entries stay in their order.
constexpr int LPT_MOST = 256;
template <int BLOCK>
__device__ __forceinline__ int longest_first(const int* lengths, long long stride, int L, int M, int rank) {
    if (!lengths || L == 1 || L > LPT_MOST) return rank;
    __shared__ int s_length[LPT_MOST], s_entry;
    for (int i = threadIdx.x; i < L; i += BLOCK) s_length[i] = key_count(lengths, stride, i, M);
    __syncthreads();
    for (int i = threadIdx.x; i < L; i += BLOCK) {
        const int mine = s_length[i];
        int       longer = 0;
#pragma unroll 8
        for (int j = 0; j < L; ++j) longer += s_length[j] > mine || (s_length[j] == mine && j < i);
        if (longer == rank) s_entry = i;
    }
    __syncthreads();
    return s_entry;
}

// ORDERED > 0: entries of the batch longest first, called by a whole block of that many threads.
template <typename T, int ORDERED = 0>
__device__ __forceinline__ Work find_work(const AttentionParams& p, int block, int rows_per_block, int keys_per_tile) {
    Work w;
    const int prefix_blocks = p.Hk * p.prefix_tiles * p.prefix_splits;
    int       tile, split, splits;
    if (block < prefix_blocks) {
        split  = block % p.prefix_splits, block /= p.prefix_splits;
        tile   = block % p.prefix_tiles, w.hk = block / p.prefix_tiles;
        splits = p.prefix_splits;
        w.l = -1, w.rows = p.L * p.N * p.G, w.length = p.P, w.part = split, w.causal = false;
        w.k = p.kp.ptr + w.hk * p.kp.sh * static_cast<long long>(sizeof(T)), w.k_sr = p.kp.sr;
        w.v = p.vp.ptr + w.hk * p.vp.sh * static_cast<long long>(sizeof(T)), w.v_sr = p.vp.sr;
    } else {
        block -= prefix_blocks;
        split = block % p.own_splits, block /= p.own_splits;
        tile  = block % p.own_tiles, block /= p.own_tiles;
        w.hk = block % p.Hk, w.l = block / p.Hk;
        if constexpr (ORDERED > 0) w.l = longest_first<ORDERED>(p.lengths, p.lengths_stride, p.L, p.M, w.l);
        splits = p.own_splits;
        w.rows = p.N * p.G, w.length = key_count(p.lengths, p.lengths_stride, w.l, p.M), w.part = p.prefix_splits + split;
        w.causal = p.causal;
        w.k = p.k.ptr + (w.l * p.k.sl + w.hk * p.k.sh) * static_cast<long long>(sizeof(T)), w.k_sr = p.k.sr;
        w.v = p.v.ptr + (w.l * p.v.sl + w.hk * p.v.sh) * static_cast<long long>(sizeof(T)), w.v_sr = p.v.sr;
    }
    w.row0 = tile * rows_per_block;
    // pieces of whole tiles, from the length that the entry has
    const int tiles = (w.length + keys_per_tile - 1) / keys_per_tile;
    const int each  = (tiles + splits - 1) / splits;
    const long long first = static_cast<long long>(split) * each * keys_per_tile, end = first + static_cast<long long>(each) * keys_per_tile;
    w.first = static_cast<int>(first < w.length ? first : w.length);
    w.end   = static_cast<int>(end < w.length ? end : w.length);
    return w;
}

struct Row { int l, n, h; };
__device__ __forceinline__ Row find_row(const AttentionParams& p, const Work& w, int r) {
    Row row;
    const int q = r / p.G;
    row.h = w.hk * p.G + r - q * p.G;
    row.l = w.l >= 0 ? w.l : q / p.N;
    row.n = w.l >= 0 ? q : q - row.l * p.N;
    return row;
}
// First own key that the row does not see.
__device__ __forceinline__ int row_limit(const AttentionParams& p, const Work& w, int r) {
    return w.causal ? w.length - p.N + r / p.G + 1 : w.length;
}

// The two columns (c, c + 1) of a finished row: into out, or into its part.
template <typename T>
__device__ __forceinline__ void put_pair(const AttentionParams& p, const Work& w, const Row& row, int c, float x, float y) {
    if (c >= p.D) return;
    if (p.parts == 1) {
        T* o = reinterpret_cast<T*>(p.out.ptr) + row.l * p.out.sl + row.n * p.out.sr + row.h * p.out.sh + c;
        if constexpr (sizeof(T) == 2) {
            if (p.vec_out) {
                *reinterpret_cast<uint32_t*>(o) = Type<T>::pair(x, y);
                return;
            }
        }
        o[0] = Type<T>::to(x);
        if (c + 1 < p.D) o[1] = Type<T>::to(y);
    } else {
        float* o = p.part_o + ((((static_cast<long long>(w.part) * p.L + row.l) * p.N + row.n) * p.H) + row.h) * p.D + c;
        if (p.D % 2 == 0) {
            *reinterpret_cast<float2*>(o) = make_float2(x, y);
        } else {
            o[0] = x;
            if (c + 1 < p.D) o[1] = y;
        }
    }
}
// A row's maximum (log2 domain) and its sum of exp2 of what lies below: into its part, or as the logarithm of the whole.  A row without keys
// has the sum 0.  Parts keep the two apart: as one logarithm of some 11, rounded, they would weigh with errors of 3e-7 each, which
// made a float32 token against 3000 keys in 11 pieces 2.6 times as inaccurate as fp32 products.
__device__ __forceinline__ void put_stats(const AttentionParams& p, const Work& w, const Row& row, float top, float sum) {
    if (sum == 0.0f) top = -INFINITY;
    if (p.parts != 1) {
        const long long rows = static_cast<long long>(p.L) * p.N * p.H, at = w.part * rows + (static_cast<long long>(row.l) * p.N + row.n) * p.H + row.h;
        p.part_top[at] = top, p.part_top[p.parts * rows + at] = sum;
    } else if (p.lse) {
        p.lse[row.l * p.lse_sl + row.h * p.lse_sh + row.n] = (top + lg2_approx(sum)) * LN2;
    }
}

}  // namespace att
}  // namespace km
