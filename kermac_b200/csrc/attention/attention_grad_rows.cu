// Gradient of the attention for any layout, type and width up to 256 channels, with mma.sync.
//
// With p = exp(s - lse) recomputed from the forward pass's lse and delta = sum_d dout * out,
//   dv = p^T dout,   ds = p * (dout v^T - delta),   dk = scale ds^T q,   dq = scale ds k.
// Two kinds of blocks, so that every sum has one owner and a fixed order: one holds 64 keys and streams the queries (dk, dv), one holds
// 64 queries and streams the keys (dq).  The price is that s and dout v^T are computed twice, 7 products instead of 5.
//
// One launch has both, so that few rows of either fill the SMs together: a block is four warps, one for each scheduler of an SM, and one
// warp alone issues in 0.38 of the cycles.  float32 gradients, two launches and one: 2 x 300 x 500, 4 heads of 64, 80 and 63 us;
// 2 x 77 x 300, 8 heads of 64, 55 and 35; 300 x 300, 4 heads of 250, 307 and 184.
#include <algorithm>

#include "attention_grad.cuh"

namespace km {
namespace att {
namespace {

// Whether an entry's queries take delta from its own terms, for the reason in attention_grad_tensor.cu: where a block of keys holds all of them.
template <typename T>
__device__ __forceinline__ constexpr bool exact_delta(int count) { return sizeof(T) == 2 && count <= ATT_GRAD_ROWS; }

template <typename T, int DP>
struct GradShape {
    static constexpr int ROWS   = ATT_GRAD_ROWS;
    static constexpr int STREAM = sizeof(T) == 2 && DP <= 128 ? 32 : 16;
    static constexpr int CT     = (DP > 128 ? 128 : DP) / 8;             // channel groups of a block's dk and dv
    static constexpr int HELD   = Tile<T, DP>::bytes(ROWS);
    static constexpr int MOVED  = Tile<T, DP>::bytes(STREAM);
    static constexpr int STATS  = 2 * 2 * STREAM * 4 + WARPS * STREAM * 4;      // two stages of lse and delta; the warps' parts of an exact delta
    static constexpr int SMEM   = 2 * HELD + 2 * 2 * MOVED + STATS;
};

// `block`: (key tile, slice, key head, batch entry of k and v, channel part)
template <typename T, int DP>
__device__ __forceinline__ void gradient_of_keys(const AttentionGradParams& p, int block) {
    typedef GradShape<T, DP> S;
    typedef Tile<T, DP>      TL;
    constexpr int NT = S::STREAM / 8, CT = S::CT;
    extern __shared__ __align__(16) char smem[];
    T* const     held_k = reinterpret_cast<T*>(smem);
    T* const     held_v = reinterpret_cast<T*>(smem + S::HELD);
    char* const  ring   = smem + 2 * S::HELD;
    float* const stats  = reinterpret_cast<float*>(ring + 4 * S::MOVED);
    float* const parts  = stats + 4 * S::STREAM;
    const int    warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;

    const int tiles = (p.M + S::ROWS - 1) / S::ROWS;
    const int key0 = block % tiles * S::ROWS; block /= tiles;
    const int slice = block % p.kv_slices;    block /= p.kv_slices;
    const int hk = block % p.Hk;              block /= p.Hk;
    const int kl = block % p.kv_batch, c0 = block / p.kv_batch * CT * 8;

    // the sum runs over (batch entries of a broadcast k, heads of the group, query tiles): this block's piece of it
    const int l_count = p.kv_batch == 1 ? p.L : 1, l_first = p.kv_batch == 1 ? 0 : kl;
    const int q_tiles = (p.N + S::STREAM - 1) / S::STREAM;
    const int all     = l_count * p.G * q_tiles;
    const int from    = static_cast<int>(static_cast<long long>(all) * slice / p.kv_slices);
    const int to      = static_cast<int>(static_cast<long long>(all) * (slice + 1) / p.kv_slices);
    int longest = 0;                               // keys from here on are in no sum of this block: their gradient is zero
    if (from < to)
        for (int l = l_first + from / (p.G * q_tiles); l <= l_first + (to - 1) / (p.G * q_tiles); ++l) {
            const int n = key_count(p.lengths, p.lengths_stride, l, p.M);
            longest = n > longest ? n : longest;
        }
    const bool  idle   = key0 >= longest;
    const float factor = idle ? 1.0f : find_factor<T>(p, l_first, l_first + l_count, hk, kl, longest);
    const float by     = factor * per_weight<T>;

    float dk[CT][4], dv[CT][4];
#pragma unroll
    for (int c = 0; c < CT; ++c)
        dk[c][0] = dk[c][1] = dk[c][2] = dk[c][3] = dv[c][0] = dv[c][1] = dv[c][2] = dv[c][3] = 0.0f;

    if (!idle) {
        copy_rows<T, DP>(held_k, head_of<T>(p.k, kl, hk), p.k.sr, key0, longest, S::ROWS, p.D, p.vec, threadIdx.x, THREADS);
        copy_rows<T, DP>(held_v, head_of<T>(p.v, kl, hk), p.v.sr, key0, longest, S::ROWS, p.D, p.vec, threadIdx.x, THREADS);
        auto load = [&](int i) {
            if (i < to) {
                const int qt = i % q_tiles, lg = i / q_tiles, h = hk * p.G + lg % p.G, l = l_first + lg / p.G, n0 = qt * S::STREAM;
                T* const  dst = reinterpret_cast<T*>(ring + (i & 1) * 2 * S::MOVED);
                copy_rows<T, DP>(dst, head_of<T>(p.q, l, h), p.q.sr, n0, p.N, S::STREAM, p.D, p.vec, threadIdx.x, THREADS);
                copy_rows<T, DP>(dst + S::STREAM * TL::LD, head_of<T>(p.dout, l, h), p.dout.sr, n0, p.N, S::STREAM, p.D, p.vec,
                                 threadIdx.x, THREADS);
                if (threadIdx.x < 2 * S::STREAM) {
                    const int    r = threadIdx.x % S::STREAM, which = threadIdx.x / S::STREAM;
                    const bool   valid = n0 + r < p.N;
                    const float* src = which == 0 ? p.lse + l * p.lse_sl + h * p.lse_sh : p.delta + (static_cast<long long>(l) * p.H + h) * p.N;
                    copy_async_4(smem_addr(stats + ((i & 1) * 2 + which) * S::STREAM + r), valid ? src + n0 + r : src, valid);
                }
            }
            copy_commit();
        };
        load(from);
        for (int i = from; i < to; ++i) {
            load(i + 1);
            copy_wait<1>();
            __syncthreads();
            const T* const     q     = reinterpret_cast<const T*>(ring + (i & 1) * 2 * S::MOVED);
            const T* const     dout  = q + S::STREAM * TL::LD;
            const float* const lse   = stats + (i & 1) * 2 * S::STREAM;
            float* const       delta = stats + ((i & 1) * 2 + 1) * S::STREAM;
            const int          l     = l_first + i / (q_tiles * p.G), n0 = (i % q_tiles) * S::STREAM;
            const int          count = key_count(p.lengths, p.lengths_stride, l, p.M);
            float s[NT][4], ds[NT][4];
#pragma unroll
            for (int j = 0; j < NT; ++j)
                s[j][0] = s[j][1] = s[j][2] = s[j][3] = ds[j][0] = ds[j][1] = ds[j][2] = ds[j][3] = 0.0f;
            product_nt<T, DP, NT>(s, held_k + warp * 16 * TL::LD, q);
            product_nt<T, DP, NT>(ds, held_v + warp * 16 * TL::LD, dout);
            if (exact_delta<T>(count) && key0 == 0) {          // this block has every key of the entry
#pragma unroll
                for (int j = 0; j < NT; ++j)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const int col  = j * 8 + 2 * t + e;
                        float     part = 0.0f;
#pragma unroll
                        for (int r = 0; r < 2; ++r)
                            if (warp * 16 + g + 8 * r < count)
                                part = fmaf(ex2_approx(fmaf(s[j][e + 2 * r], p.scale_log2, -lse[col] * (1.0f / LN2))), ds[j][e + 2 * r], part);
#pragma unroll
                        for (int d = 4; d <= 16; d <<= 1) part += __shfl_xor_sync(0xffffffffu, part, d);
                        if (g == 0) parts[warp * S::STREAM + col] = part;
                    }
                __syncthreads();
                if (threadIdx.x < S::STREAM) {
                    const float* const of = parts + threadIdx.x;
                    delta[threadIdx.x] = (of[0] + of[S::STREAM]) + (of[2 * S::STREAM] + of[3 * S::STREAM]);
                }
                __syncthreads();
            }
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int   col  = j * 8 + 2 * t + (e & 1);
                    const bool  seen = key0 + warp * 16 + g + 8 * (e >> 1) < count && n0 + col < p.N;
                    const float w    = ex2_approx(fmaf(s[j][e], p.scale_log2, weight_log2<T> - lse[col] * (1.0f / LN2)));
                    ds[j][e] = seen ? w * ((ds[j][e] - delta[col]) * by) : 0.0f;
                    s[j][e]  = seen ? w : 0.0f;
                }
            product_nn<T, DP, NT, CT>(dv, s, dout + c0);
            product_nn<T, DP, NT, CT>(dk, ds, q + c0);
            __syncthreads();
        }
        copy_wait<0>();
    }
    float* const dk_part = p.kv_slices > 1 ? p.dk_part + static_cast<long long>(slice) * p.kv_batch * p.M * p.Hk * p.D : nullptr;
    float* const dv_part = p.kv_slices > 1 ? p.dv_part + static_cast<long long>(slice) * p.kv_batch * p.M * p.Hk * p.D : nullptr;
    const float  k_by = p.scale / factor, v_by = per_weight<T>;
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        const int key = key0 + warp * 16 + g + 8 * r;
        if (key >= p.M) continue;
#pragma unroll
        for (int c = 0; c < CT; ++c) {
            const int at = c0 + c * 8 + 2 * t;
            put_grad<T>(p.dk, dk_part, kl, key, hk, p.M, p.Hk, p.D, at, dk[c][2 * r] * k_by, dk[c][2 * r + 1] * k_by);
            put_grad<T>(p.dv, dv_part, kl, key, hk, p.M, p.Hk, p.D, at, dv[c][2 * r] * v_by, dv[c][2 * r + 1] * v_by);
        }
    }
}

template <typename T, int DP>
__device__ __forceinline__ void gradient_of_queries(const AttentionGradParams& p, int block) {
    typedef GradShape<T, DP> S;
    typedef Tile<T, DP>      TL;
    constexpr int NT = S::STREAM / 8, CT = DP / 8;
    extern __shared__ __align__(16) char smem[];
    T* const    held_q = reinterpret_cast<T*>(smem);
    T* const    held_d = reinterpret_cast<T*>(smem + S::HELD);
    char* const ring   = smem + 2 * S::HELD;
    const int   warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;

    const int tiles = (p.N + S::ROWS - 1) / S::ROWS;
    const int n0 = block % tiles * S::ROWS; block /= tiles;
    const int split = block % p.q_splits;   block /= p.q_splits;
    const int h = block % p.H, l = block / p.H, hk = h / p.G;
    const int   count  = key_count(p.lengths, p.lengths_stride, l, p.M);
    const int   kl     = p.kv_batch == 1 ? 0 : l;
    const float v_peak = find_v_peak<T>(p, kl, hk, count);

    copy_rows<T, DP>(held_q, head_of<T>(p.q, l, h), p.q.sr, n0, p.N, S::ROWS, p.D, p.vec, threadIdx.x, THREADS);
    copy_rows<T, DP>(held_d, head_of<T>(p.dout, l, h), p.dout.sr, n0, p.N, S::ROWS, p.D, p.vec, threadIdx.x, THREADS);
    // this block's piece of the keys
    const int key_tiles = (count + S::STREAM - 1) / S::STREAM;
    const int i_first = static_cast<int>(static_cast<long long>(key_tiles) * split / p.q_splits);
    const int i_end   = static_cast<int>(static_cast<long long>(key_tiles) * (split + 1) / p.q_splits);
    auto load = [&](int i) {
        const int first = i * S::STREAM;
        if (i < i_end) {
            T* const dst = reinterpret_cast<T*>(ring + (i & 1) * 2 * S::MOVED);
            copy_rows<T, DP>(dst, head_of<T>(p.k, kl, hk), p.k.sr, first, count, S::STREAM, p.D, p.vec, threadIdx.x, THREADS);
            copy_rows<T, DP>(dst + S::STREAM * TL::LD, head_of<T>(p.v, kl, hk), p.v.sr, first, count, S::STREAM, p.D, p.vec, threadIdx.x,
                             THREADS);
        }
        copy_commit();
    };
    float lse[2], delta[2], factor[2], dq[CT][4];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        const int n = n0 + warp * 16 + g + 8 * r;
        lse[r]   = n < p.N ? p.lse[l * p.lse_sl + h * p.lse_sh + n] * (1.0f / LN2) : 0.0f;
        delta[r] = n < p.N ? p.delta[(static_cast<long long>(l) * p.H + h) * p.N + n] : 0.0f;
        factor[r] = row_factor<T>(p, l, h, n, v_peak);
    }
#pragma unroll
    for (int c = 0; c < CT; ++c) dq[c][0] = dq[c][1] = dq[c][2] = dq[c][3] = 0.0f;

    if (exact_delta<T>(count)) {
        float sum[2] = {0.0f, 0.0f};
        for (int i = 0; i < key_tiles; ++i) {
            T* const k = reinterpret_cast<T*>(ring);
            copy_rows<T, DP>(k, head_of<T>(p.k, kl, hk), p.k.sr, i * S::STREAM, count, S::STREAM, p.D, p.vec, threadIdx.x, THREADS);
            copy_rows<T, DP>(k + S::STREAM * TL::LD, head_of<T>(p.v, kl, hk), p.v.sr, i * S::STREAM, count, S::STREAM, p.D, p.vec, threadIdx.x, THREADS);
            copy_commit();
            copy_wait<0>();
            __syncthreads();
            float s[NT][4], dp[NT][4];
#pragma unroll
            for (int j = 0; j < NT; ++j)
                s[j][0] = s[j][1] = s[j][2] = s[j][3] = dp[j][0] = dp[j][1] = dp[j][2] = dp[j][3] = 0.0f;
            product_nt<T, DP, NT>(s, held_q + warp * 16 * TL::LD, k);
            product_nt<T, DP, NT>(dp, held_d + warp * 16 * TL::LD, k + S::STREAM * TL::LD);
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (i * S::STREAM + j * 8 + 2 * t + (e & 1) < count)
                        sum[e >> 1] = fmaf(ex2_approx(fmaf(s[j][e], p.scale_log2, -lse[e >> 1])), dp[j][e], sum[e >> 1]);
            __syncthreads();
        }
        delta[0] = quad_sum(sum[0]), delta[1] = quad_sum(sum[1]);
    }
    load(i_first);
    for (int i = i_first; i < i_end; ++i) {
        load(i + 1);
        copy_wait<1>();
        __syncthreads();
        const T* const k = reinterpret_cast<const T*>(ring + (i & 1) * 2 * S::MOVED);
        float s[NT][4], ds[NT][4];
#pragma unroll
        for (int j = 0; j < NT; ++j)
            s[j][0] = s[j][1] = s[j][2] = s[j][3] = ds[j][0] = ds[j][1] = ds[j][2] = ds[j][3] = 0.0f;
        product_nt<T, DP, NT>(s, held_q + warp * 16 * TL::LD, k);
        product_nt<T, DP, NT>(ds, held_d + warp * 16 * TL::LD, k + S::STREAM * TL::LD);
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float w = ex2_approx(fmaf(s[j][e], p.scale_log2, -lse[e >> 1]));
                ds[j][e] = i * S::STREAM + j * 8 + 2 * t + (e & 1) < count ? w * ((ds[j][e] - delta[e >> 1]) * factor[e >> 1]) : 0.0f;
            }
        product_nn<T, DP, NT, CT>(dq, ds, k);
        __syncthreads();
    }
    copy_wait<0>();
    // partial sums [slice][entry of q][n][h][D]: a broadcast q has one entry and a slice for each l and piece
    const bool   one_q = p.q_slices > p.q_splits;
    float* const part = p.q_slices > 1 ? p.dq_part + static_cast<long long>(one_q ? l * p.q_splits + split : split * p.L) * p.N * p.H * p.D : nullptr;
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        const int   n  = n0 + warp * 16 + g + 8 * r;
        const float by = p.scale / factor[r];
        if (n >= p.N) continue;
#pragma unroll
        for (int c = 0; c < CT; ++c)
            put_grad<T>(p.dq, part, one_q ? 0 : l, n, h, p.N, p.H, p.D, c * 8 + 2 * t, dq[c][2 * r] * by, dq[c][2 * r + 1] * by);
    }
}

// float32 with up to 64 channels: three blocks an SM (1000 x 1500, 8 heads: 415 -> 380 us); 16-bit types are
// slower with a limit (140 us against 136 at 2 x 500 x 700, 8 heads of 100).
template <typename T, int DP>
__global__ void __launch_bounds__(THREADS, sizeof(T) == 2 ? 0 : DP == 64 ? 3 : 1) attention_grad_rows_kernel(const AttentionGradParams p, const int key_blocks) {
    after_previous_grid();
    const int block = static_cast<int>(blockIdx.x);
    if (block < key_blocks)                  // four products a tile first, then three
        gradient_of_keys<T, DP>(p, block);
    else
        gradient_of_queries<T, DP>(p, block - key_blocks);
}

// The largest of a block.
__device__ __forceinline__ float block_peak(float peak, float* of_warp) {
    peak = warp_max(peak);
    if ((threadIdx.x & 31) == 0) of_warp[threadIdx.x >> 5] = peak;
    __syncthreads();
    return fmaxf(fmaxf(of_warp[0], of_warp[1]), fmaxf(of_warp[2], of_warp[3]));
}
// What is infinite or no number, like the results that it enters, says nothing of the others.
__device__ __forceinline__ float finite_size(float v) { return fabsf(v) < INFINITY ? fabsf(v) : 0.0f; }
// Lanes of a row, which take its 16-byte units in turn: a warp has 32 / lanes rows at a time.
__device__ __forceinline__ int row_lanes(int units) { return units > 16 ? 32 : units > 8 ? 16 : 8; }

// float16: v_peaks of ATT_PEAK_ROWS keys of a head; rows behind the longest sequence hold whatever the memory holds.
__device__ __forceinline__ void find_v_peaks(const AttentionGradParams& p, int block, float* of_warp) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int group = block % p.v_peak_count; block /= p.v_peak_count;
    const int hk = block % p.Hk, kl = block / p.Hk;
    int       there = p.M;
    if (p.lengths != nullptr) {
        there = 0;
        if (p.kv_batch == p.L) {
            there = key_count(p.lengths, p.lengths_stride, kl, p.M);
        } else {
            for (int l = lane; l < p.L; l += 32) there = max(there, key_count(p.lengths, p.lengths_stride, l, p.M));
            there = __reduce_max_sync(0xffffffffu, there);
        }
    }
    const __half* v    = head_of<__half>(p.v, kl, hk);
    float         peak = 0.0f;
    // as in attention_delta_kernel
    const int units = (p.D + 7) / 8, lanes = row_lanes(units), sub = lane & (lanes - 1);
#pragma unroll 4
    for (int r = (warp * 32 + lane) / lanes; r < ATT_PEAK_ROWS; r += THREADS / lanes) {
        const int key = group * ATT_PEAK_ROWS + r;
        for (int u = sub; u < units; u += lanes) {
            alignas(16) __half x[8];
            if (key < there && p.vec) {
                *reinterpret_cast<uint4*>(x) = *reinterpret_cast<const uint4*>(v + key * p.v.sr + u * 8);
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = key < there && u * 8 + e < p.D ? v[key * p.v.sr + u * 8 + e] : Type<__half>::to(0.0f);
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) peak = fmaxf(peak, finite_size(__half2float(x[e])));
        }
    }
    peak = block_peak(peak, of_warp);
    if (threadIdx.x == 0) p.v_peaks[(static_cast<long long>(kl) * p.Hk + hk) * p.v_peak_count + group] = peak;
}

// delta[l][h][n], and for float16 the peaks of dout.  One block for ATT_PEAK_ROWS queries of a head; those from `query_blocks` on
// find the peaks of v.
template <typename T>
__global__ void __launch_bounds__(THREADS) attention_delta_kernel(const AttentionGradParams p, const int query_blocks) {
    __shared__ float of_warp[WARPS];
    after_previous_grid();
    int block = blockIdx.x;
    if constexpr (is_f16<T>)
        if (block >= query_blocks) {
            find_v_peaks(p, block - query_blocks, of_warp);
            return;
        }
    const int groups = (p.N + ATT_PEAK_ROWS - 1) / ATT_PEAK_ROWS, group = block % groups;
    block /= groups;
    const int h = block % p.H, l = block / p.H, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const T * out = head_of<T>(p.out, l, h), *dout = head_of<T>(p.dout, l, h);
    float     peak = 0.0f;
    constexpr int CHUNK = Type<T>::CHUNK;
    const int units = (p.D + CHUNK - 1) / CHUNK, lanes = row_lanes(units), sub = lane & (lanes - 1);
#pragma unroll 4
    for (int r = (warp * 32 + lane) / lanes; r < ATT_PEAK_ROWS; r += THREADS / lanes) {     // uniform: a multiple of lanes rows
        const int n = group * ATT_PEAK_ROWS + r;
        float sum = 0.0f;
        for (int u = sub; u < units; u += lanes) {
            alignas(16) T x[CHUNK], y[CHUNK];
            if (n < p.N && p.vec_out) {
                *reinterpret_cast<uint4*>(x) = *reinterpret_cast<const uint4*>(dout + n * p.dout.sr + u * CHUNK);
                *reinterpret_cast<uint4*>(y) = *reinterpret_cast<const uint4*>(out + n * p.out.sr + u * CHUNK);
            } else {
#pragma unroll
                for (int e = 0; e < CHUNK; ++e) {
                    const bool there = n < p.N && u * CHUNK + e < p.D;
                    x[e] = there ? dout[n * p.dout.sr + u * CHUNK + e] : Type<T>::to(0.0f);
                    y[e] = there ? out[n * p.out.sr + u * CHUNK + e] : Type<T>::to(0.0f);
                }
            }
#pragma unroll
            for (int e = 0; e < CHUNK; ++e) {
                sum = fmaf(Type<T>::from(x[e]), Type<T>::from(y[e]), sum);
                if constexpr (is_f16<T>) peak = fmaxf(peak, finite_size(Type<T>::from(x[e])));
            }
        }
        for (int d = lanes >> 1; d; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
        if (sub == 0 && n < p.N) p.delta[(static_cast<long long>(l) * p.H + h) * p.N + n] = sum;
    }
    if constexpr (is_f16<T>) {
        peak = block_peak(peak, of_warp);
        if (threadIdx.x == 0) p.peaks[(static_cast<long long>(l) * p.H + h) * p.peak_count + group] = peak;
    }
}

// A thread adds up V neighbouring channels: 4 where rows allow it and single ones would be more than four blocks an SM (all three gradients of
// 300 x 500, 4 heads of 64 in pieces: 8.6 -> 4.4 us; but 16 queries of 4 heads in 62 pieces, a few threads with long sums, take 5 us more).
template <typename T, int V>
__global__ void __launch_bounds__(THREADS) attention_reduce_kernel(const SliceSums sums) {
    after_previous_grid();
    const long long all = sums.first[sums.count];
    for (long long at = (static_cast<long long>(blockIdx.x) * THREADS + threadIdx.x) * V; at < all; at += static_cast<long long>(gridDim.x) * THREADS * V) {
        int which = 0;
        while (which + 1 < sums.count && at >= sums.first[which + 1]) ++which;
        const SliceSum& j = sums.job[which];
        const long long i = at - sums.first[which], total = sums.first[which + 1] - sums.first[which];
        float sum[V];
#pragma unroll
        for (int e = 0; e < V; ++e) sum[e] = 0.0f;
#pragma unroll 4
        for (int s = 0; s < j.slices; ++s) {
            if constexpr (V == 4) {
                const float4 x = *reinterpret_cast<const float4*>(j.src + s * total + i);
                sum[0] += x.x, sum[1] += x.y, sum[2] += x.z, sum[3] += x.w;
            } else {
                sum[0] += j.src[s * total + i];
            }
        }
        const long long rest = i / j.D;
        const int       c = static_cast<int>(i - rest * j.D);
        const int       h = static_cast<int>(rest % j.heads), row = static_cast<int>(rest / j.heads % j.rows), l = static_cast<int>(rest / j.heads / j.rows);
        T* const        to = reinterpret_cast<T*>(j.dst.ptr) + l * j.dst.sl + row * j.dst.sr + h * j.dst.sh + c;
        if constexpr (V == 4 && sizeof(T) == 2)
            *reinterpret_cast<uint2*>(to) = make_uint2(Type<T>::pair(sum[0], sum[1]), Type<T>::pair(sum[2], sum[3]));
        else if constexpr (V == 4)
            *reinterpret_cast<float4*>(to) = make_float4(sum[0], sum[1], sum[2], sum[3]);
        else
            *to = Type<T>::to(sum[0]);
    }
}

int check_blocks(long long blocks) {
    return blocks > 0x7fffffffLL ? fail(KM_ERR_TOO_LARGE, "attention: more than 2^31 - 1 blocks") : 0;
}

template <typename T, int DP>
int launch_grad(const AttentionGradParams& p, cudaStream_t st) {
    typedef GradShape<T, DP> S;
    static_assert(S::SMEM <= 227 * 1024, "more shared memory than a block has");
    auto* const kernel = &attention_grad_rows_kernel<T, DP>;
    if (int rc = cuda_status(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM), "cudaFuncSetAttribute")) return rc;
    const long long keys    = ceil_div_ll(p.M, S::ROWS) * p.kv_slices * p.Hk * p.kv_batch * (DP / (S::CT * 8));
    const long long queries = ceil_div_ll(p.N, S::ROWS) * p.q_splits * p.H * p.L;
    if (int rc = check_blocks(keys + queries)) return rc;
    return cuda_status(launch_overlapped(kernel, dim3(static_cast<unsigned>(keys + queries)), THREADS, S::SMEM, st, p, static_cast<int>(keys)),
                       "attention_grad_rows_kernel");
}
template <typename T>
int launch_type(const AttentionGradParams& p, cudaStream_t st) {
    switch (padded_channels(p.D)) {
        case 64: return launch_grad<T, 64>(p, st);
        case 128: return launch_grad<T, 128>(p, st);
        default: return launch_grad<T, 256>(p, st);
    }
}

}  // namespace
}  // namespace att

int attention_grad_rows_launch(const AttentionGradParams& p, int type, cudaStream_t st) {
    using namespace att;
    if (type == ATT_F32) return launch_type<float>(p, st);
    return type == ATT_BF16 ? launch_type<__nv_bfloat16>(p, st) : launch_type<__half>(p, st);
}

int attention_delta_launch(const AttentionGradParams& p, int type, cudaStream_t st) {
    using namespace att;
    const long long queries = ceil_div_ll(p.N, ATT_PEAK_ROWS) * p.H * p.L, blocks = queries + static_cast<long long>(p.v_peak_count) * p.Hk * p.kv_batch;
    if (int rc = check_blocks(blocks)) return rc;
    const dim3 grid(static_cast<unsigned>(blocks));
    const int  query_blocks = static_cast<int>(queries);
    const cudaError_t e = type == ATT_F32    ? launch_overlapped(&attention_delta_kernel<float>, grid, THREADS, 0, st, p, query_blocks)
                          : type == ATT_BF16 ? launch_overlapped(&attention_delta_kernel<__nv_bfloat16>, grid, THREADS, 0, st, p, query_blocks)
                                             : launch_overlapped(&attention_delta_kernel<__half>, grid, THREADS, 0, st, p, query_blocks);
    return cuda_status(e, "attention_delta_kernel");
}

namespace att {
namespace {
template <typename T, int V>
cudaError_t launch_reduce(const SliceSums& sums, cudaStream_t st) {
    const long long blocks = std::min(ceil_div_ll(sums.first[sums.count], THREADS * V), 65536LL);       // the kernel strides over the rest
    return launch_overlapped(&attention_reduce_kernel<T, V>, dim3(static_cast<unsigned>(blocks)), THREADS, 0, st, sums);
}
template <typename T>
cudaError_t launch_reduce(const SliceSums& sums, bool vec, cudaStream_t st) {
    return vec && sums.first[sums.count] > 4LL * THREADS * sm_count() ? launch_reduce<T, 4>(sums, st) : launch_reduce<T, 1>(sums, st);
}
}  // namespace
}  // namespace att

int attention_reduce_launch(const SliceSums& sums, int type, bool vec, cudaStream_t st) {
    using namespace att;
    if (sums.first[sums.count] == 0) return 0;
    return cuda_status(type == ATT_F32    ? launch_reduce<float>(sums, vec, st)
                       : type == ATT_BF16 ? launch_reduce<__nv_bfloat16>(sums, vec, st)
                                          : launch_reduce<__half>(sums, vec, st),
                       "attention_reduce_kernel");
}

}  // namespace km
