// Attention of few 16-bit queries (decoding steps): bound by reading the keys and values once.
//
// Up to 16 rows share a block; its four warps take tiles of 32 keys in turn, each with a ring of its own that TMA fills, so that no
// warp waits for another, and add up at the end.  Products are transposed, S^T = K Q^T and O^T = V^T P^T (mma.sync m16n8k16): the rows
// are the narrow side of an instruction, eight at a time, where the other way round 16 rows would be computed for one
// token.  Q stays in registers; P^T passes from accumulator to operand layout by movmatrix.
//
// Measured at 64 sequences x 1 x 4096 keys (ragged), 32 heads of 128, 8 key heads, float16, 674 MB, back-to-back passes over three sets of
// inputs: 110 to 114 us, 5.9 to 6.1 TB/s, 91 to 94 % of a plain copy.  While it was written, one pass at a time: copies by the lanes (cp.async, 480 of some 700
// instructions a tile) with 16 rows an instruction 294 us, this 105; two warps a block and two blocks an SM 118.
//
// Two blocks an SM hide what a block does before its first and behind its last tile.  Up to 64 channels they fit; above, tiles of 16
// keys make room for them: attention_few_tile().  It goes by the keys that an entry may have, M, because lengths are on the device.  With tiles of 32 and
// of 16, us, one token of 4 query heads to each of 8 key heads of 128 (of 80):
//     keys              512          1024          2048          3000          4096          8192
//     4 sequences       6.9   7.4    8.3  10.8    11.6  13.7    14.7  17.6    17.1  20.1    27.6  30.7
//     16                9.6  10.4   14.7  16.2    24.4  26.3    33.3  35.7    43.2  46.1    80.0  86.2
//     32               18.7  14.5   27.8  24.7    45.4  44.5    62.6  62.9    81.0  84.3     154   162
//     64               34.6  27.1   52.2  45.4    88.8  80.9     124   116     162   155     309   302
//     32, 80 channels  16.6  12.4   24.3  18.9    38.7  31.5    52.8  43.3    67.3  56.4     124   106
// Tiles of 16 gain up to 26 % where there are more blocks than SMs, up to some 2500 keys (ragged 64 x 4096: 110.4 and 113.9), and lose up to 30 % where there
// are fewer and their keys are divided.  Taking 32 there as well is not the better rule: one block an SM leaves room for fewer clusters, and 8 pieces of 1081
// keys, 16 heads, went from 9.7 to 15.6 us, 5 pieces of 1718 keys, 40 heads, from 18.5 to 10.6.
#include <algorithm>

#include "attention_tcgen05.cuh"

namespace km {
namespace att {
namespace {

__device__ int g_attention_few_wait_expired = 0;


// KEYS: 32 or 16 keys a tile.
template <int DP, int NR, int KEYS>
struct FewShape {
    static constexpr int ROWS   = 8 * NR, STAGES = 3;
    static constexpr int SLAB   = KEYS * 128, TILE = DP / 64 * SLAB;      // one tile of K or V
    static constexpr int RING   = STAGES * 2 * TILE;                          // of one warp
    static constexpr int W      = DP + 2;                                     // channels, maximum and sum of a row
    static constexpr int MERGE  = WARPS * ROWS * W * 4;
    static constexpr int SMEM   = 1024 + (WARPS * RING > MERGE ? WARPS * RING : MERGE);
};

__device__ __forceinline__ uint32_t transposed(uint32_t v) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
__device__ __forceinline__ float column_max(float v) {       // over the eight lanes that hold one row's keys
    v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 4));
    v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 8));
    return fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 16));
}
__device__ __forceinline__ float column_sum(float v) {
    v += __shfl_xor_sync(0xffffffffu, v, 4);
    v += __shfl_xor_sync(0xffffffffu, v, 8);
    return v + __shfl_xor_sync(0xffffffffu, v, 16);
}

// Blocks of a cluster: arrive and wait (all of them always do), and read each other's shared memory.
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t address_in(uint32_t addr, int rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
__device__ __forceinline__ float load_cluster(uint32_t addr) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ float load_own(uint32_t addr) {
    float v;
    asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
    return v;
}

template <typename T, int DP, int NR, int KEYS>
__global__ void __launch_bounds__(THREADS) attention_few_kernel(const __grid_constant__ AttentionParams p, const __grid_constant__ TensorMaps maps) {
    typedef FewShape<DP, NR, KEYS> S;
    constexpr int BLOCKS = KEYS / 16;              // operands of 16 keys in a tile
    extern __shared__ unsigned char smem_raw[];
    __shared__ __align__(8) unsigned long long s_bars[WARPS * S::STAGES];
    __shared__ int s_expired;
    const int      warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const uint32_t raw = smem_addr(smem_raw), base = (raw + 1023u) & ~1023u, ring = base + warp * S::RING;
    const uint32_t bars = smem_addr(s_bars) + warp * S::STAGES * 8;
    if (threadIdx.x == 0) s_expired = 0;
    if (lane == 0) {
        for (int st = 0; st < S::STAGES; ++st) mbar_init(bars + 8 * st, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        tc::fence_smem_to_async();
    }
    __syncthreads();
    after_previous_grid();

    const Work w      = find_work<T>(p, blockIdx.x, S::ROWS, KEYS);
    const bool prefix = w.l < 0;
    const int  tiles = (w.end - w.first + KEYS - 1) / KEYS, mine = (tiles - warp + WARPS - 1) / WARPS;
    const CUtensorMap *mk = prefix ? &maps.kp : &maps.k, *mv = prefix ? &maps.vp : &maps.v;
    const int lk = prefix || p.k.sl == 0 ? 0 : w.l, lv = prefix || p.v.sl == 0 ? 0 : w.l;
    auto load = [&](int i) {                                  // by lane 0
        const int      st = i % S::STAGES, first = w.first + (i * WARPS + warp) * KEYS;
        const uint32_t to = ring + st * 2 * S::TILE, bar = bars + 8 * st;
        mbar_expect_tx(bar, 2 * S::TILE);
#pragma unroll
        for (int d = 0; d < DP / 64; ++d) {
            tma_load_rows(to + d * S::SLAB, mk, d * 64, first, w.hk, lk, bar);
            tma_load_rows(to + S::TILE + d * S::SLAB, mv, d * 64, first, w.hk, lv, bar);
        }
    };
    if (lane == 0)
        for (int i = 0; i < S::STAGES && i < mine; ++i) load(i);

    // Q^T as the second operand: channels 2t, 2t + 1 (+ 8) of row g
    uint32_t q[NR][DP / 16][2];
    int      limit[NR][2];
#pragma unroll
    for (int r = 0; r < NR; ++r) {
        const int   at = w.row0 + r * 8 + g;
        const char* from = nullptr;
        if (at < w.rows) {
            const Row row = find_row(p, w, at);
            from = p.q.ptr + (row.l * p.q.sl + row.n * p.q.sr + row.h * p.q.sh) * 2;
        }
#pragma unroll
        for (int k = 0; k < DP / 16; ++k)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int c = k * 16 + e * 8 + 2 * t;
                q[r][k][e] = from != nullptr && c < p.D ? *reinterpret_cast<const uint32_t*>(from + c * 2) : 0;
            }
#pragma unroll
        for (int e = 0; e < 2; ++e) limit[r][e] = min(row_limit(p, w, w.row0 + r * 8 + 2 * t + e), w.end);
    }
    // keys in front of it are seen by every row
    const int all_see = min(w.causal ? w.length - p.N + 1 : w.length, w.end), held = prefix ? p.P : p.M;

    float o[DP / 16][NR][4], top[NR][2], sum[NR][2];
    Exponent<T> exponent[NR][2];
#pragma unroll
    for (int r = 0; r < NR; ++r) {
        top[r][0] = top[r][1] = -INFINITY, sum[r][0] = sum[r][1] = 0.0f;
        exponent[r][0] = exponent[r][1] = {p.scale_log2, weight_log2<T>};
#pragma unroll
        for (int d = 0; d < DP / 16; ++d) o[d][r][0] = o[d][r][1] = o[d][r][2] = o[d][r][3] = 0.0f;
    }
    bool expired = false;
    for (int i = 0; i < mine; ++i) {
        const int      st = i % S::STAGES, first = w.first + (i * WARPS + warp) * KEYS;
        const uint32_t tile_k = ring + st * 2 * S::TILE, tile_v = tile_k + S::TILE;
        // every copy is waited for, with a short limit once a wait has run out
        if (!mbar_wait_bounded(bars + 8 * st, (i / S::STAGES) & 1, expired ? 1 << 16 : MBAR_WAIT_TRIES)) expired = true;
        float s[BLOCKS][NR][4];
#pragma unroll
        for (int m = 0; m < BLOCKS; ++m)
#pragma unroll
            for (int r = 0; r < NR; ++r) s[m][r][0] = s[m][r][1] = s[m][r][2] = s[m][r][3] = 0.0f;
#pragma unroll
        for (int k = 0; k < DP / 16; ++k)
#pragma unroll
            for (int m = 0; m < BLOCKS; ++m) {
                const int row = m * 16 + (lane & 15), chunk = k * 2 + (lane >> 4);
                uint32_t  a[4];
                ldmatrix4(a, tile_k + (chunk >> 3) * S::SLAB + row * 128 + ((chunk ^ row) & 7) * 16);
#pragma unroll
                for (int r = 0; r < NR; ++r) mma_16(s[m][r], a, q[r][k][0], q[r][k][1], static_cast<const T*>(nullptr));
            }
        if (first + KEYS > all_see) {
#pragma unroll
            for (int m = 0; m < BLOCKS; ++m)
#pragma unroll
                for (int r = 0; r < NR; ++r)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (first + m * 16 + g + 8 * (e >> 1) >= limit[r][e & 1]) s[m][r][e] = -INFINITY;
            if (first + KEYS > w.end && w.end < held) {
                // rows of V behind the length hold whatever the memory holds, and 0 * NaN is NaN
                if (lane < KEYS && first + lane >= w.end) {
#pragma unroll
                    for (int c = 0; c < DP / 8; ++c)
                        asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(tile_v + (c >> 3) * S::SLAB + lane * 128 + (c & 7) * 16), "r"(0) : "memory");
                }
                __syncwarp();
            }
        }
        float base_m[NR][2];
        bool  grown = false;
#pragma unroll
        for (int r = 0; r < NR; ++r)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                float best = fmaxf(s[0][r][e], s[0][r][e + 2]);
                if (BLOCKS > 1) best = fmaxf(best, fmaxf(s[BLOCKS - 1][r][e], s[BLOCKS - 1][r][e + 2]));
                best = column_max(best);
                grown      = grown || best > top[r][e];
                base_m[r][e] = fmaxf(best, top[r][e]);
            }
        if (__any_sync(0xffffffffu, grown)) {
#pragma unroll
            for (int r = 0; r < NR; ++r) {
                float shrink[2];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    // (-inf) - (-inf) of a row that has seen nothing yet must not become NaN
                    shrink[e] = top[r][e] == -INFINITY ? 0.0f : ex2_approx((top[r][e] - base_m[r][e]) * p.scale_log2);
                    exponent[r][e].raise(base_m[r][e], p.scale_log2);
                    top[r][e] = base_m[r][e];
                    sum[r][e] *= shrink[e];
                }
#pragma unroll
                for (int d = 0; d < DP / 16; ++d)
                    o[d][r][0] *= shrink[0], o[d][r][1] *= shrink[1], o[d][r][2] *= shrink[0], o[d][r][3] *= shrink[1];
            }
        }
        uint32_t weights[BLOCKS][NR][2];
#pragma unroll
        for (int r = 0; r < NR; ++r) {
            // float16 takes the maximum off beforehand, which is as good (Exponent for both: 64 x 4096 keys, float16, 107.9 -> 110.1 us; this for both:
            // 128 sequences below a prefix, bfloat16, 134.9 -> 136.3)
            float minus[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) minus[e] = top[r][e] == -INFINITY ? 0.0f : -top[r][e] * (is_f16<T> ? 1.0f : exponent[r][e].by);
#pragma unroll
            for (int m = 0; m < BLOCKS; ++m) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    s[m][r][e] = ex2_approx(is_f16<T> ? fmaf(s[m][r][e] + minus[e & 1], p.scale_log2, weight_log2<T>)
                                                      : fmaf(s[m][r][e], exponent[r][e & 1].by, minus[e & 1]));
                    sum[r][e & 1] += s[m][r][e];
                }
                weights[m][r][0] = transposed(Type<T>::pair(s[m][r][0], s[m][r][1]));
                weights[m][r][1] = transposed(Type<T>::pair(s[m][r][2], s[m][r][3]));
            }
        }
#pragma unroll
        for (int m = 0; m < BLOCKS; ++m)
#pragma unroll
            for (int d = 0; d < DP / 16; ++d) {
                const int row = m * 16 + (lane & 7) + ((lane >> 4) << 3), chunk = d * 2 + ((lane >> 3) & 1);
                uint32_t  a[4];
                ldmatrix4_trans(a, tile_v + (chunk >> 3) * S::SLAB + row * 128 + ((chunk ^ row) & 7) * 16);
#pragma unroll
                for (int r = 0; r < NR; ++r) mma_16(o[d][r], a, weights[m][r][0], weights[m][r][1], static_cast<const T*>(nullptr));
            }
        __syncwarp();                        // every lane has read the stage
        if (lane == 0 && i + S::STAGES < mine) load(i + S::STAGES);
    }
    if (expired) *reinterpret_cast<volatile int*>(&s_expired) = 1;
    __syncthreads();                         // the rings are free: the warps' sums go there
    float* const sums = reinterpret_cast<float*>(smem_raw + (base - raw));
#pragma unroll
    for (int r = 0; r < NR; ++r)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            float* const at = sums + (warp * S::ROWS + r * 8 + 2 * t + e) * S::W;
#pragma unroll
            for (int d = 0; d < DP / 16; ++d) at[d * 16 + g] = o[d][r][e] * per_weight<T>, at[d * 16 + g + 8] = o[d][r][e + 2] * per_weight<T>;
            const float total = column_sum(sum[r][e]) * per_weight<T>;
            if (g == 0) at[DP] = top[r][e] == -INFINITY ? -INFINITY : top[r][e] * p.scale_log2, at[DP + 1] = total;
        }
    __syncthreads();
    // The pieces of a row's keys are a cluster where they are few: its blocks share out the row's channels and read one another's sums.
    // (With a kernel of its own for that: a token against 4 x 1000 states, 16 heads of 64, 8.3 us a pass; this way 7.0.)
    const int pieces = p.cluster, rank = pieces > 1 ? static_cast<int>(blockIdx.x) % pieces : 0;
    if (pieces > 1) cluster_sync();
    const uint32_t at_sums = smem_addr(sums);
    bool           good = s_expired == 0;
    if (!good && threadIdx.x == 0) g_attention_few_wait_expired = 1;
    // reading through the cluster's window costs a lone block 1 % of a pass over 1024 short sequences
    auto finish = [&](auto load, auto place) {
        for (int i = rank * THREADS + threadIdx.x; good && i < S::ROWS * (DP / 2); i += pieces * THREADS) {
            const int r = i / (DP / 2), c = (i % (DP / 2)) * 2;
            if (w.row0 + r >= w.rows || c >= p.D) continue;
            float best = -INFINITY, total = 0.0f, x = 0.0f, y = 0.0f;
            for (int k = 0; k < pieces; ++k)
#pragma unroll
                for (int j = 0; j < WARPS; ++j) best = fmaxf(best, load(place(at_sums + ((j * S::ROWS + r) * S::W + DP) * 4, k)));
            const float from_m = best == -INFINITY ? 0.0f : best;
            for (int k = 0; k < pieces; ++k)
#pragma unroll
                for (int j = 0; j < WARPS; ++j) {
                    const uint32_t from   = place(at_sums + (j * S::ROWS + r) * S::W * 4, k);
                    const float    weight = ex2_approx(load(from + DP * 4) - from_m);
                    total += weight * load(from + DP * 4 + 4);
                    x += weight * load(from + c * 4), y += weight * load(from + c * 4 + 4);
                }
            const Row   row = find_row(p, w, w.row0 + r);
            const float by  = total == 0.0f ? 0.0f : 1.0f / total;
            if (c == 0) put_stats(p, w, row, best, total);
            put_pair<T>(p, w, row, c, x * by, y * by);
        }
    };
    if (pieces > 1) {
        for (int k = 0; k < pieces; ++k) good = good && __float_as_int(load_cluster(address_in(smem_addr(&s_expired), k))) == 0;
        finish([](uint32_t a) { return load_cluster(a); }, [](uint32_t a, int k) { return address_in(a, k); });
    } else {
        finish([](uint32_t a) { return load_own(a); }, [](uint32_t a, int) { return a; });
    }
    if (pieces > 1) cluster_sync();          // nobody reads this block's shared memory any more
}

// launch_overlapped() with clusters of `size` blocks.
template <typename... Params, typename... Args>
cudaError_t launch_clusters(void (*fn)(Params...), unsigned blocks, int size, int threads, size_t smem_bytes, cudaStream_t stream,
                            const Args&... args) {
    cudaLaunchAttribute attributes[2];
    attributes[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attributes[0].val.programmaticStreamSerializationAllowed = 1;
    attributes[1].id = cudaLaunchAttributeClusterDimension;
    attributes[1].val.clusterDim.x = static_cast<unsigned>(size), attributes[1].val.clusterDim.y = 1, attributes[1].val.clusterDim.z = 1;
    cudaLaunchConfig_t config = {};
    config.gridDim          = dim3(blocks);
    config.blockDim         = dim3(static_cast<unsigned>(threads), 1, 1);
    config.dynamicSmemBytes = smem_bytes;
    config.stream           = stream;
    config.attrs            = attributes;
    config.numAttrs         = 2;
    return cudaLaunchKernelEx(&config, fn, static_cast<Params>(args)...);
}

template <typename T, int DP, int NR, int KEYS>
int launch_few(const AttentionParams& p, const TensorMaps& maps, cudaStream_t st) {
    constexpr int smem = FewShape<DP, NR, KEYS>::SMEM;
    static_assert(smem <= 227 * 1024, "more shared memory than a block has");
    auto* const kernel = &attention_few_kernel<T, DP, NR, KEYS>;
    if (int rc = cuda_status(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem), "cudaFuncSetAttribute")) return rc;
    unsigned blocks;
    if (int rc = count_blocks(p, &blocks)) return rc;
    if (p.cluster == 1) return cuda_status(launch_overlapped(kernel, dim3(blocks), THREADS, smem, st, p, maps), "attention_few_kernel");
    return cuda_status(launch_clusters(kernel, blocks, p.cluster, THREADS, smem, st, p, maps), "attention_few_kernel");
}
template <typename T>
int launch_few_type(const AttentionParams& p, const TensorMaps& maps, int rows, int keys, cudaStream_t st) {
    if (p.D <= 64) return rows <= 8 ? launch_few<T, 64, 1, 32>(p, maps, st) : launch_few<T, 64, 2, 32>(p, maps, st);
    if (keys == 16) return rows <= 8 ? launch_few<T, 128, 1, 16>(p, maps, st) : launch_few<T, 128, 2, 16>(p, maps, st);
    return rows <= 8 ? launch_few<T, 128, 1, 32>(p, maps, st) : launch_few<T, 128, 2, 32>(p, maps, st);
}

}  // namespace
}  // namespace att

int attention_few_launch(const AttentionParams& p, int type, int rows, cudaStream_t st) {
    using namespace att;
    TensorMaps maps = {};
    const int  keys = attention_few_tile(p.D, p.own_tiles > 0 ? p.M : 0, p.prefix_tiles > 0 ? p.P : 0);
    if (int rc = encode_forward(&maps, p, type, keys)) return rc;
    return type == ATT_BF16 ? launch_few_type<__nv_bfloat16>(p, maps, rows, keys, st) : launch_few_type<__half>(p, maps, rows, keys, st);
}

int attention_few_take_wait_flag() { return att::take_wait_flag(att::g_attention_few_wait_expired); }

}  // namespace km
