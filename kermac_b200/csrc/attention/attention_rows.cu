// Attention for any layout, type and width up to 256 channels: softmax(scale Q K^T) V with mma.sync, and the kernel that joins
// the parts of a split.
//
// One pass over the keys with a running maximum m and sum l per row: a tile's scores S = Q K^T raise m, what was summed under
// the old one is scaled by exp2(m_old - m_new), and P = exp2(S - m) is multiplied with V straight from the registers it was
// computed in (the accumulator layout of one product is the operand layout of the next).
#include "attention_mma.cuh"
#include "attention_work.cuh"

namespace km {
namespace att {
namespace {

// How a block works.  FEW: one tile of 16 rows, the four warps take key tiles of their own in turn and add up at the end
// (decoding steps: bound by reading the keys, so the warps wait for no one and have three tiles each under way).  Otherwise:
// 64 rows, 16 a warp, and one key tile for all.
template <typename T, int DP, bool FEW>
struct Shape {
    static constexpr int ROWS   = FEW ? ATT_FEW_ROWS : ATT_TILE_ROWS;
    static constexpr int KEYS   = sizeof(T) == 2 ? (FEW ? (DP > 128 ? 16 : 32) : (DP > 128 ? 32 : 64))
                                                 : (FEW ? (DP > 128 ? 8 : 16) : (DP > 128 ? 16 : 32));
    static constexpr int STAGES = FEW ? 3 : 2;
    static constexpr int GROUPS = FEW ? WARPS : 1;                 // sets of threads with key tiles of their own
    static constexpr int TILE   = Tile<T, DP>::bytes(KEYS);
    static constexpr int Q      = Tile<T, DP>::bytes(ROWS);
    static constexpr int MERGE  = FEW ? WARPS * ROWS * (DP + 2) * 4 : 0;
    static constexpr int RING   = GROUPS * STAGES * 2 * TILE;
    static constexpr int SMEM   = Q + (RING > MERGE ? RING : MERGE);
};

template <typename T, int DP, bool FEW>
__global__ void __launch_bounds__(THREADS) attention_rows_kernel(const AttentionParams p) {
    typedef Shape<T, DP, FEW> S;
    typedef Tile<T, DP>       TL;
    constexpr int NT = S::KEYS / 8, CT = DP / 8;
    extern __shared__ __align__(16) char smem[];
    T* const  tile_q = reinterpret_cast<T*>(smem);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    after_previous_grid();

    const Work w = find_work<T>(p, blockIdx.x, S::ROWS, S::KEYS);
    const T *  k = reinterpret_cast<const T*>(w.k), *v = reinterpret_cast<const T*>(w.v);

    for (int i = threadIdx.x; i < S::ROWS * TL::CHUNKS; i += THREADS) {
        const int r = i / TL::CHUNKS, c = (i % TL::CHUNKS) * Type<T>::CHUNK;
        const T*  q = nullptr;
        if (w.row0 + r < w.rows) {
            const Row row = find_row(p, w, w.row0 + r);
            q = reinterpret_cast<const T*>(p.q.ptr) + row.l * p.q.sl + row.n * p.q.sr + row.h * p.q.sh;
        }
        copy_chunk(tile_q + r * TL::LD + c, q, reinterpret_cast<const T*>(p.q.ptr), c, p.D, p.vec);
    }
    copy_commit();

    // the key tiles of this group: `step` tiles apart
    const int group = FEW ? warp : 0, index = FEW ? lane : static_cast<int>(threadIdx.x), members = FEW ? 32 : THREADS;
    char* const ring  = smem + S::Q + group * S::STAGES * 2 * S::TILE;
    const int   tiles = (w.end - w.first + S::KEYS - 1) / S::KEYS;
    const int   mine  = (tiles - group + S::GROUPS - 1) / S::GROUPS;
    auto load = [&](int i) {
        if (i < mine) {
            T* const  dst   = reinterpret_cast<T*>(ring + (i % S::STAGES) * 2 * S::TILE);
            const int first = w.first + (i * S::GROUPS + group) * S::KEYS;
            copy_rows<T, DP>(dst, k, w.k_sr, first, w.end, S::KEYS, p.D, p.vec, index, members);
            copy_rows<T, DP>(dst + S::KEYS * TL::LD, v, w.v_sr, first, w.end, S::KEYS, p.D, p.vec, index, members);
        }
        copy_commit();
    };
    auto group_sync = [] {
        if (FEW) __syncwarp(); else __syncthreads();
    };

    float o[CT][4], top[2] = {-INFINITY, -INFINITY}, sum[2] = {0.0f, 0.0f};
#pragma unroll
    for (int c = 0; c < CT; ++c) o[c][0] = o[c][1] = o[c][2] = o[c][3] = 0.0f;
    const int my_row = (FEW ? 0 : warp * 16) + g;
    int       limit[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        limit[i] = row_limit(p, w, w.row0 + my_row + 8 * i);
        limit[i] = limit[i] < w.end ? limit[i] : w.end;
    }

#pragma unroll
    for (int i = 0; i < S::STAGES - 1; ++i) load(i);
    copy_wait<S::STAGES - 1>();              // Q has arrived
    __syncthreads();
    const T* const my_q = tile_q + (FEW ? 0 : warp * 16) * TL::LD;

    for (int i = 0; i < mine; ++i) {
        load(i + S::STAGES - 1);
        copy_wait<S::STAGES - 1>();
        group_sync();
        const T* const tile_k = reinterpret_cast<const T*>(ring + (i % S::STAGES) * 2 * S::TILE);
        const int      first  = w.first + (i * S::GROUPS + group) * S::KEYS;
        float s[NT][4];
#pragma unroll
        for (int j = 0; j < NT; ++j) s[j][0] = s[j][1] = s[j][2] = s[j][3] = 0.0f;
        product_nt<T, DP, NT>(s, my_q, tile_k);

        float best[2] = {top[0], top[1]};
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int key = first + j * 8 + 2 * t + (e & 1);
                s[j][e] = key < limit[e >> 1] ? s[j][e] * p.scale_log2 : -INFINITY;
                best[e >> 1] = fmaxf(best[e >> 1], s[j][e]);
            }
        float base[2];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            best[r] = quad_max(best[r]);
            base[r] = best[r] == -INFINITY ? 0.0f : best[r];     // a row that has seen no key yet: exp2(-inf - 0) = 0
            const float shrink = ex2_approx(top[r] - base[r]);
            top[r] = best[r];
            sum[r] *= shrink;
#pragma unroll
            for (int c = 0; c < CT; ++c) o[c][2 * r] *= shrink, o[c][2 * r + 1] *= shrink;
        }
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                s[j][e] = ex2_approx(s[j][e] - base[e >> 1] + weight_log2<T>);
                sum[e >> 1] += s[j][e];
            }
        product_nn<T, DP, NT, CT>(o, s, tile_k + S::KEYS * TL::LD);
        group_sync();
    }
    sum[0] = quad_sum(sum[0]) * per_weight<T>, sum[1] = quad_sum(sum[1]) * per_weight<T>;

    if constexpr (!FEW) {
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const int at = w.row0 + my_row + 8 * r;
            if (at >= w.rows) continue;
            const Row   row = find_row(p, w, at);
            const float by  = sum[r] == 0.0f ? 0.0f : per_weight<T> / sum[r];
            if (t == 0) put_stats(p, w, row, top[r], sum[r]);
#pragma unroll
            for (int c = 0; c < CT; ++c) put_pair<T>(p, w, row, c * 8 + 2 * t, o[c][2 * r] * by, o[c][2 * r + 1] * by);
        }
    } else {
        copy_wait<0>();
        __syncthreads();                     // the ring is free: the warps' sums go there
        float* const sums = reinterpret_cast<float*>(smem + S::Q);
        constexpr int W = DP + 2;            // DP channels, the maximum and the sum
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            float* const mine_at = sums + (warp * S::ROWS + g + 8 * r) * W;
#pragma unroll
            for (int c = 0; c < CT; ++c)
                *reinterpret_cast<float2*>(mine_at + c * 8 + 2 * t) = make_float2(o[c][2 * r] * per_weight<T>, o[c][2 * r + 1] * per_weight<T>);
            if (t == 0) mine_at[DP] = top[r], mine_at[DP + 1] = sum[r];
        }
        __syncthreads();
        for (int i = threadIdx.x; i < S::ROWS * (DP / 2); i += THREADS) {
            const int r = i / (DP / 2), c = (i % (DP / 2)) * 2;
            if (w.row0 + r >= w.rows || c >= p.D) continue;
            float best = -INFINITY, total = 0.0f, x = 0.0f, y = 0.0f;
#pragma unroll
            for (int j = 0; j < WARPS; ++j) best = fmaxf(best, sums[(j * S::ROWS + r) * W + DP]);
            const float base = best == -INFINITY ? 0.0f : best;
#pragma unroll
            for (int j = 0; j < WARPS; ++j) {
                const float* const from   = sums + (j * S::ROWS + r) * W;
                const float        weight = ex2_approx(from[DP] - base);
                total += weight * from[DP + 1], x += weight * from[c], y += weight * from[c + 1];
            }
            const Row   row = find_row(p, w, w.row0 + r);
            const float by  = total == 0.0f ? 0.0f : 1.0f / total;
            if (c == 0) put_stats(p, w, row, best, total);
            put_pair<T>(p, w, row, c, x * by, y * by);
        }
    }
}

// Adds up the parts of a row, in a fixed order: out = sum_i 2^(top_i) sum_i o_i / sum_i 2^(top_i) sum_i.  One warp a row, or WIDE four that take every fourth
// part each (48 rows of 72 parts, 3 sequences below a prefix of 18192: 28 us with one warp; 4096 rows of 10 parts: 9 us more with four).
// A lane has four neighbouring channels, or single ones 32 apart where rows are no multiple of four (V = 1); loads are predicated,
// not branched around, so that those of eight parts are under way at once (4096 rows of 10 parts of 128 channels: 16 -> 11 us).
template <typename T, bool WIDE, int V>
__global__ void __launch_bounds__(THREADS) attention_join_kernel(const AttentionParams p) {
    constexpr int STEP = WIDE ? WARPS : 1, SETS = 256 / (32 * V);
    __shared__ float s_sum[WARPS][256], s_total[WARPS];
    after_previous_grid();
    const int       lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const long long rows = static_cast<long long>(p.L) * p.N * p.H, row = static_cast<long long>(blockIdx.x) * (WARPS / STEP) + (WIDE ? 0 : warp);
    if (row >= rows) return;                 // WIDE: a block has one row, which is there
    float best = -INFINITY;
    for (int i = lane; i < p.parts; i += 32) best = fmaxf(best, p.part_top[i * rows + row]);
#pragma unroll
    for (int d = 16; d; d >>= 1) best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, d));
    const float base = best == -INFINITY ? 0.0f : best;
    float total = 0.0f, x[SETS][V];
#pragma unroll
    for (int c = 0; c < SETS; ++c)
#pragma unroll
        for (int e = 0; e < V; ++e) x[c][e] = 0.0f;
    for (int i0 = WIDE ? warp : 0; i0 < p.parts; i0 += 32 * STEP) {
        // a lane's part; one without keys has weight 0 and has written no sum
        const int   part = i0 + lane * STEP;
        const float mine = part < p.parts ? ex2_approx(p.part_top[part * rows + row] - base) * p.part_top[(p.parts + part) * rows + row] : 0.0f;
        total += mine;
        const int    many = min(32, (p.parts - i0 + STEP - 1) / STEP);
        const float* from = p.part_o + (i0 * rows + row) * p.D + lane * V;
#pragma unroll 8
        for (int i = 0; i < many; ++i, from += STEP * rows * p.D) {
            const float weight = __shfl_sync(0xffffffffu, mine, i);
#pragma unroll
            for (int c = 0; c < SETS; ++c) {
                const bool there = weight != 0.0f && (c * 32 + lane) * V < p.D;
                if constexpr (V == 4) {
                    const float4 v = there ? *reinterpret_cast<const float4*>(from + c * 32 * V) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    x[c][0] = fmaf(weight, v.x, x[c][0]), x[c][1] = fmaf(weight, v.y, x[c][1]);
                    x[c][2] = fmaf(weight, v.z, x[c][2]), x[c][3] = fmaf(weight, v.w, x[c][3]);
                } else {
                    x[c][0] = fmaf(weight, there ? from[c * 32] : 0.0f, x[c][0]);
                }
            }
        }
    }
#pragma unroll
    for (int d = 16; d; d >>= 1) total += __shfl_xor_sync(0xffffffffu, total, d);
    if constexpr (WIDE) {
#pragma unroll
        for (int c = 0; c < SETS; ++c)
#pragma unroll
            for (int e = 0; e < V; ++e) s_sum[warp][(c * 32 + lane) * V + e] = x[c][e];
        if (lane == 0) s_total[warp] = total;
        __syncthreads();
        if (warp != 0) return;
        total = (s_total[0] + s_total[1]) + (s_total[2] + s_total[3]);
#pragma unroll
        for (int c = 0; c < SETS; ++c)
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const int at = (c * 32 + lane) * V + e;
                x[c][e] = (s_sum[0][at] + s_sum[1][at]) + (s_sum[2][at] + s_sum[3][at]);
            }
    }
    const int       h = static_cast<int>(row % p.H);
    const long long ln = row / p.H;
    const int       l = static_cast<int>(ln / p.N), n = static_cast<int>(ln - static_cast<long long>(l) * p.N);
    const float     by = total == 0.0f ? 0.0f : 1.0f / total;
    T* const        o  = reinterpret_cast<T*>(p.out.ptr) + l * p.out.sl + n * p.out.sr + h * p.out.sh;
#pragma unroll
    for (int c = 0; c < SETS; ++c) {
        const int at = (c * 32 + lane) * V;
        if (at >= p.D) continue;
        alignas(16) T y[V];
#pragma unroll
        for (int e = 0; e < V; ++e) y[e] = Type<T>::to(x[c][e] * by);
        if (V == 4 && p.vec_out) {
            if constexpr (V == 4 && sizeof(T) == 2) *reinterpret_cast<uint2*>(o + at) = *reinterpret_cast<const uint2*>(y);
            if constexpr (V == 4 && sizeof(T) == 4) *reinterpret_cast<uint4*>(o + at) = *reinterpret_cast<const uint4*>(y);
        } else {
#pragma unroll
            for (int e = 0; e < V; ++e) o[at + e] = y[e];
        }
    }
    if (p.lse && lane == 0) p.lse[l * p.lse_sl + h * p.lse_sh + n] = (best + lg2_approx(total)) * LN2;
}

template <typename T, int DP, bool FEW>
int launch_rows(const AttentionParams& p, cudaStream_t st) {
    constexpr int smem = Shape<T, DP, FEW>::SMEM;
    static_assert(smem <= 227 * 1024, "more shared memory than a block has");
    auto* const kernel = &attention_rows_kernel<T, DP, FEW>;
    int rc = cuda_status(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem), "cudaFuncSetAttribute");
    if (rc) return rc;
    unsigned blocks;
    if ((rc = count_blocks(p, &blocks))) return rc;
    return cuda_status(launch_overlapped(kernel, dim3(blocks), THREADS, smem, st, p), "attention_rows_kernel");
}
template <typename T>
int launch_type(const AttentionParams& p, bool few, cudaStream_t st) {
    switch (padded_channels(p.D)) {
        case 64: return few ? launch_rows<T, 64, true>(p, st) : launch_rows<T, 64, false>(p, st);
        case 128: return few ? launch_rows<T, 128, true>(p, st) : launch_rows<T, 128, false>(p, st);
        default: return few ? launch_rows<T, 256, true>(p, st) : launch_rows<T, 256, false>(p, st);
    }
}

}  // namespace
}  // namespace att

int attention_rows_launch(const AttentionParams& p, int type, bool few, cudaStream_t st) {
    using namespace att;
    if (type == ATT_F32) return launch_type<float>(p, few, st);
    return type == ATT_BF16 ? launch_type<__nv_bfloat16>(p, few, st) : launch_type<__half>(p, few, st);
}

namespace att {
namespace {
template <typename T, int V>
cudaError_t launch_join(const AttentionParams& p, cudaStream_t st) {
    const long long rows = static_cast<long long>(p.L) * p.N * p.H;              // below 2^31: checked
    if (p.parts > 16) return launch_overlapped(&attention_join_kernel<T, true, V>, dim3(static_cast<unsigned>(rows)), THREADS, 0, st, p);
    return launch_overlapped(&attention_join_kernel<T, false, V>, dim3(static_cast<unsigned>(ceil_div_ll(rows, WARPS))), THREADS, 0, st, p);
}
template <typename T>
cudaError_t launch_join(const AttentionParams& p, cudaStream_t st) {
    return p.D % 4 == 0 ? launch_join<T, 4>(p, st) : launch_join<T, 1>(p, st);
}
}  // namespace
}  // namespace att

int attention_join_launch(const AttentionParams& p, int type, cudaStream_t st) {
    using namespace att;
    return cuda_status(type == ATT_F32    ? launch_join<float>(p, st)
                       : type == ATT_BF16 ? launch_join<__nv_bfloat16>(p, st)
                                          : launch_join<__half>(p, st),
                       "attention_join_kernel");
}

}  // namespace km
