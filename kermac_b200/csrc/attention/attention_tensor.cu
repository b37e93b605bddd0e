// Attention of many 16-bit queries on the tensor cores (tcgen05), head widths up to 128: softmax(scale Q K^T) V.
//
// A block holds two tiles of 128 rows.  Q, and K and V as TMA brings them, lie in shared memory; S = Q K^T goes to tensor memory,
// the thread that owns a row reads it from there, writes the weights P back over it as the 16-bit operand of O += P V, and
// O stays in tensor memory.  While one tile's warps work on their weights the tensor cores multiply for the other tile.
//
// The running maximum that weights are taken against may lag: it is raised, and O scaled, only where a row's maximum has grown by more
// than 2^8, so that weights are at most 256 (the first tile sets it; after that it seldom happens).  float16 weights, which are 2^8 times as large, see
// attention_mma.cuh, have 2^5, an eighth of that type's range.
//
// 4 x 4096 x 8192, 16 heads of 128, bf16: 1006 to 1025 us, 1.08 PFLOP/s, in passes that follow one another, 947 to 1024 in single ones, by the clock that
// the power limit leaves.  In one run at 1.65 GHz, which the figures below are from, 887, and the products alone, without a softmax, 783.  A step (two tiles of rows, 128 keys) is 3440 cycles for products of 2048.  Tried: two threads a row (eight
// warps a tile, 960 us), 2 to 5 of 8 pairs of exponentials on the FP32 pipe (952 to 1023), polling waits, K and V in one slot (no gain).
#include <algorithm>

#include "attention_tcgen05.cuh"

namespace km {
namespace att {
namespace {

__device__ int g_attention_wait_expired = 0;

template <int DP>
struct TensorShape {
    static constexpr int TILE   = DP / 64 * TC_SLAB;
    static constexpr int STAGES = DP == 128 ? 4 : 6;       // tiles of K and V under way (3 and 5: the same time)
    static constexpr int SMEM   = 1024 + (2 + STAGES) * TILE;
    static constexpr int GROUPS = 2;                       // row tiles, a warpgroup each
    static constexpr int LOAD_WARP = 4 * GROUPS, MMA_WARP = LOAD_WARP + 1, THREADS = 128 * (GROUPS + 1);
    // of the 168 registers that 384 threads are launched with, the last warpgroup gives up what the other two take: 2 * 224 + 56 = 3 * 168
    static constexpr int REGS_SOFTMAX = 224, REGS_OTHERS = 56;
    // tensor memory: S of both tiles (P over its first half), O of both tiles
    static constexpr int S_COL = 0, O_COL = GROUPS * 128;
};

template <typename T, int DP>
__global__ void __launch_bounds__(TensorShape<DP>::THREADS, 1)
attention_tensor_kernel(const __grid_constant__ AttentionParams p, const __grid_constant__ TensorMaps maps,
                        const __grid_constant__ QueryMaps queries, const int query_boxes) {
    typedef TensorShape<DP> S;
    extern __shared__ unsigned char smem_raw[];
    constexpr int BARS = 2 * S::STAGES + 4 * S::GROUPS;
    __shared__ __align__(8) unsigned long long s_bars[BARS];
    __shared__ uint32_t s_tmem;
    __shared__ int s_expired;

    const uint32_t raw  = smem_addr(smem_raw), base = (raw + 1023u) & ~1023u;
    char* const    tiles = reinterpret_cast<char*>(smem_raw) + (base - raw);
    const int      warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t bars = smem_addr(s_bars);
    auto full   = [&](int st) { return bars + 8u * st; };
    auto empty  = [&](int st) { return bars + 8u * (S::STAGES + st); };
    auto q_full = [&](int t) { return bars + 8u * (2 * S::STAGES + t); };
    auto s_full = [&](int t) { return bars + 8u * (2 * S::STAGES + S::GROUPS + t); };
    auto p_full = [&](int t) { return bars + 8u * (2 * S::STAGES + 2 * S::GROUPS + t); };
    auto o_full = [&](int t) { return bars + 8u * (2 * S::STAGES + 3 * S::GROUPS + t); };
    if (threadIdx.x == 0) {
        for (int st = 0; st < S::STAGES; ++st) mbar_init(full(st), 1), mbar_init(empty(st), 1);
        const bool boxes = query_boxes & (static_cast<int>(blockIdx.x) < p.Hk * p.prefix_tiles * p.prefix_splits ? QUERIES_PREFIX : QUERIES_OWN);
        for (int t = 0; t < S::GROUPS; ++t) mbar_init(q_full(t), boxes ? 1 : 4), mbar_init(s_full(t), 1), mbar_init(p_full(t), 4), mbar_init(o_full(t), 1);
        s_expired = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        tc::fence_smem_to_async();
    }
    after_previous_grid();
    if (warp == S::MMA_WARP) tc::tmem_alloc(smem_addr(&s_tmem), 512);
    tc::fence_before_sync();
    __syncthreads();
    tc::fence_after_sync();
    const uint32_t tmem = s_tmem;
    bool expired = false;
    // once a wait has run out this warp stops waiting: a stuck barrier costs one limit, not one per tile
    auto wait = [&](uint32_t bar, int parity) {
        if (!expired && !mbar_wait_bounded(bar, parity)) {
            expired = true;
            *reinterpret_cast<volatile int*>(&s_expired) = 1;
        }
    };

    // what is in flight at the end is waited for (with a limit) also when an earlier wait has run out
    auto drain = [&](uint32_t bar, int parity) {
        if (!mbar_wait_bounded(bar, parity, expired ? 1 << 16 : MBAR_WAIT_TRIES)) *reinterpret_cast<volatile int*>(&s_expired) = 1;
    };

    const Work w       = find_work<T, S::THREADS>(p, blockIdx.x, S::GROUPS * TC_ROWS, TC_ROWS);
    const int  n_tiles = (w.end - w.first + TC_ROWS - 1) / TC_ROWS;
    const int  groups  = w.row0 + TC_ROWS < w.rows ? 2 : 1;
    const bool prefix  = w.l < 0;
    const bool boxes   = query_boxes & (prefix ? QUERIES_PREFIX : QUERIES_OWN);      // Q comes by TMA
    const uint32_t ring = base + S::GROUPS * S::TILE;

    if (warp < S::LOAD_WARP) {
        // ------------------------------------------------------------------ softmax: thread = row
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(S::REGS_SOFTMAX));
        const int t = warp >> 2, r = threadIdx.x & 127, at = w.row0 + t * TC_ROWS + r;
        const uint32_t lane_base = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
        const uint32_t s_col = lane_base + S::S_COL + t * 128, o_col = lane_base + S::O_COL + t * DP;
        if (t < groups && n_tiles > 0) {
            const Row row = find_row(p, w, min(at, w.rows - 1));
            if (!boxes) {
                const char* q = at < w.rows ? p.q.ptr + (row.l * p.q.sl + row.n * p.q.sr + row.h * p.q.sh) * 2 : nullptr;
                fill_row<DP>(tiles + t * S::TILE, r, q, p.D);
                tc::fence_smem_to_async();
                __syncwarp();
                if (lane == 0) mbar_arrive(q_full(t));
            }

            // -inf times the scale of 0 would be NaN; the launcher passes at least 2^-149
            const float c = p.scale_log2;
            const int   limit = min(row_limit(p, w, at < w.rows ? at : w.rows - 1), w.end);
            const int   all_see = w.causal ? w.length - p.N + 1 : w.length;     // keys in front of it are seen by every row
            // slack: how far a row's maximum may grow; -inf where nothing but scores of -inf has come, whose maximum of 0 any other replaces
            constexpr float SLACK = is_f16<T> ? 5.0f : 8.0f;
            float top = 0.0f, sum = 0.0f, slack = SLACK;
            Exponent<T> exponent = {c, weight_log2<T>};
            for (int i = 0; i < n_tiles; ++i) {
                const int first = w.first + i * TC_ROWS;
                wait(s_full(t), i & 1);
                tc::fence_after_sync();
                uint32_t x[128];
#pragma unroll
                for (int j = 0; j < 4; ++j) tmem_load32(s_col + j * 32, x + j * 32);
                tmem_wait_load();
#pragma unroll
                for (int j = 0; j < 4; ++j) tmem_loaded32(x + j * 32);
                if (first + TC_ROWS > min(all_see, w.end)) {
#pragma unroll
                    for (int j = 0; j < 128; ++j) x[j] = first + j < limit ? x[j] : 0xff800000u;
                }
                float best[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int j = 0; j < 128; j += 8)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        best[e] = fmaxf(fmaxf(best[e], __uint_as_float(x[j + e])), __uint_as_float(x[j + 4 + e]));
                const float high = fmaxf(fmaxf(best[0], best[1]), fmaxf(best[2], best[3]));
                if (i == 0) {
                    if (high == -INFINITY) slack = -INFINITY; else top = high, exponent.raise(top, c);      // a row that sees nothing: exp2(-inf - 0) = 0
                } else {
                    const bool grown = (high - top) * c > slack;
                    if (__any_sync(0xffffffffu, grown)) {
                        // the products into O that were issued before this S are complete
                        const float from = top, up = exponent.up;
                        if (grown) top = high, exponent.raise(top, c);
                        const float shrink = grown && slack > 0.0f ? ex2_approx((from - high) * c + (exponent.up - up)) : 1.0f;
                        if (grown) slack = SLACK;
                        sum *= shrink;
#pragma unroll
                        for (int j = 0; j < DP; j += 32) {
                            uint32_t o[32];
                            tmem_load32(o_col + j, o);
                            tmem_wait_load();
                            tmem_loaded32(o);
#pragma unroll
                            for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * shrink);
                            tmem_store32(o_col + j, o);
                        }
                    }
                }
                const float minus = exponent.up - top * exponent.by;
                const u64 c2 = pack2(exponent.by, exponent.by), m2 = pack2(minus, minus);
                u64 total[2] = {0, 0};
#pragma unroll
                for (int j = 0; j < 64; j += 32) {
                    uint32_t y[32];
#pragma unroll
                    for (int e = 0; e < 32; ++e) {
                        const int at2 = 2 * (j + e);
                        float lo, hi;
                        unpack2(fma2(pack2(__uint_as_float(x[at2]), __uint_as_float(x[at2 + 1])), c2, m2), lo, hi);
                        lo = ex2_approx(lo), hi = ex2_approx(hi);
                        total[e & 1] = add2(total[e & 1], pack2(lo, hi));
                        y[e] = Type<T>::pair(lo, hi);
                    }
                    tmem_store32(s_col + (j ? 64 : 0), y);
                }
                float a0, a1, a2, a3;
                unpack2(total[0], a0, a1);
                unpack2(total[1], a2, a3);
                sum += (a0 + a1) + (a2 + a3);
                // Rows of the last V tile behind the length hold whatever the memory holds, and 0 * NaN is NaN.
                const int held = prefix ? p.P : p.M;
                if (t == 0 && first + TC_ROWS > w.end && w.end < held) {
                    const int st = (2 * i + 1) % S::STAGES;
                    wait(full(st), ((2 * i + 1) / S::STAGES) & 1);
                    for (int e = (w.end - first) * 8 + r; e < TC_ROWS * 8; e += 128)
#pragma unroll
                        for (int d = 0; d < DP / 64; ++d)
                            *reinterpret_cast<uint4*>(tiles + (S::GROUPS + st) * S::TILE + d * TC_SLAB + e * 16) = make_uint4(0, 0, 0, 0);
                    tc::fence_smem_to_async();
                }
                tc::wait_st();
                tc::fence_before_sync();
                __syncwarp();
                if (lane == 0) mbar_arrive(p_full(t));
            }
            wait(o_full(t), 0);
            tc::fence_after_sync();
            const bool  good = *reinterpret_cast<volatile int*>(&s_expired) == 0 && at < w.rows;
            sum *= exponent.per();
            const float by  = sum == 0.0f ? 0.0f : exponent.per() / sum;
            if (good) put_stats(p, w, row, top * c, sum);
            if (p.parts > 1 || p.vec_out) {
                // the warp's rows of Q have been used for the last time
                char* const stage = tiles + t * S::TILE + (warp & 3) * 4096;
                char* const to    = p.out.ptr + (row.l * p.out.sl + row.n * p.out.sr + row.h * p.out.sh) * 2;
                float* const part = p.part_o + ((((static_cast<long long>(w.part) * p.L + row.l) * p.N + row.n) * p.H) + row.h) * p.D;
                store_sums<T, DP>(o_col, stage, good && p.parts == 1 ? to : nullptr, good && p.parts > 1 ? reinterpret_cast<char*>(part) : nullptr,
                                  p.parts > 1, p.D, by);
            } else {
#pragma unroll
                for (int j = 0; j < DP; j += 32) {
                    uint32_t o[32];
                    tmem_load32(o_col + j, o);
                    tmem_wait_load();
                    tmem_loaded32(o);
                    if (!good) continue;
#pragma unroll
                    for (int e = 0; e < 32; e += 2)
                        put_pair<T>(p, w, row, j + e, __uint_as_float(o[e]) * by, __uint_as_float(o[e + 1]) * by);
                }
            }
        } else if (t < groups && at < w.rows) {          // no keys
            const Row row = find_row(p, w, at);
            put_stats(p, w, row, -INFINITY, 0.0f);
            if (p.parts == 1)
                for (int j = 0; j < p.D; j += 2) put_pair<T>(p, w, row, j, 0.0f, 0.0f);
        }
    } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(S::REGS_OTHERS));
    if (warp == S::LOAD_WARP) {
        // ------------------------------------------------------------------ copies: K and V tiles in turn
        if (tc::elect_one()) {
            const CUtensorMap *mk = prefix ? &maps.kp : &maps.k, *mv = prefix ? &maps.vp : &maps.v;
            const int lk = prefix || p.k.sl == 0 ? 0 : w.l, lv = prefix || p.v.sl == 0 ? 0 : w.l;
            if (n_tiles > 0 && boxes)
                for (int t = 0; t < groups; ++t) {
                    const CUtensorMap* const mq = prefix ? &queries.prefix : &queries.own;
                    mbar_expect_tx(q_full(t), S::TILE);
#pragma unroll
                    for (int d = 0; d < DP / 64; ++d)
                        tma_load_box(base + t * S::TILE + d * TC_SLAB, mq, d * 64, w.hk * p.G, (w.row0 + t * TC_ROWS) / p.G,
                                     prefix || p.q.sl == 0 ? 0 : w.l, q_full(t));
                }
            for (int j = 0; j < 2 * n_tiles; ++j) {
                const int st = j % S::STAGES;
                if (j >= S::STAGES) wait(empty(st), (j / S::STAGES - 1) & 1);
                mbar_expect_tx(full(st), S::TILE);
#pragma unroll
                for (int d = 0; d < DP / 64; ++d)
                    tma_load_rows(ring + st * S::TILE + d * TC_SLAB, (j & 1) ? mv : mk, d * 64, w.first + (j >> 1) * TC_ROWS, w.hk,
                                  (j & 1) ? lv : lk, full(st));
            }
            for (int t = 0; t < groups && n_tiles > 0 && boxes; ++t) drain(q_full(t), 0);
            // copies still in flight must land before the block's shared memory goes to another
            for (int j = max(0, 2 * n_tiles - S::STAGES); j < 2 * n_tiles; ++j) drain(full(j % S::STAGES), (j / S::STAGES) & 1);
        }
        __syncwarp();
    } else if (warp == S::MMA_WARP) {
        // ------------------------------------------------------------------ products
        auto scores = [&](int t, int st) {
            issue_channels<T, DP>(p.D, tmem + S::S_COL + t * 128, desc_channels(base + t * S::TILE), desc_channels(ring + st * S::TILE), s_full(t));
        };
        if (n_tiles > 0) {
            wait(full(0), 0);
            for (int t = 0; t < groups; ++t) {
                wait(q_full(t), 0);
                tc::fence_after_sync();
                scores(t, 0);
            }
            issue_commit(empty(0));
            for (int i = 0; i < n_tiles; ++i) {
                const int jv = 2 * i + 1, jk = 2 * i + 2, sv = jv % S::STAGES, sk = jk % S::STAGES;
                wait(full(sv), (jv / S::STAGES) & 1);
                for (int t = 0; t < groups; ++t) {
                    wait(p_full(t), i & 1);
                    tc::fence_after_sync();
                    issue_rows<T, DP>(p.D, tmem + S::O_COL + t * DP, tmem + S::S_COL + t * 128, desc_rows(ring + sv * S::TILE), i > 0);
                    if (t == groups - 1) issue_commit(empty(sv));
                    if (i == n_tiles - 1) issue_commit(o_full(t));
                    if (i + 1 < n_tiles) {
                        if (t == 0) wait(full(sk), (jk / S::STAGES) & 1);
                        scores(t, sk);
                        if (t == groups - 1) issue_commit(empty(sk));
                    }
                }
            }
            // every product has ended before tensor memory is given back
            for (int t = 0; t < groups; ++t) drain(o_full(t), 0);
        }
    }
    }
    tc::fence_before_sync();
    __syncthreads();
    tc::fence_after_sync();
    if (warp == S::MMA_WARP) tc::tmem_dealloc(tmem, 512);
    if (threadIdx.x == 0 && s_expired) g_attention_wait_expired = 1;
}

template <typename T, int DP>
int launch_tensor(const AttentionParams& p, const TensorMaps& maps, const QueryMaps& queries, int boxes, cudaStream_t st) {
    typedef TensorShape<DP> S;
    static_assert(S::SMEM <= 227 * 1024 && S::SMEM > 114 * 1024, "one block an SM: a second would wait for its tensor memory");
    auto* const kernel = &attention_tensor_kernel<T, DP>;
    int rc = cuda_status(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM), "cudaFuncSetAttribute");
    if (rc) return rc;
    unsigned blocks;
    if ((rc = count_blocks(p, &blocks))) return rc;
    return cuda_status(launch_overlapped(kernel, dim3(blocks), S::THREADS, S::SMEM, st, p, maps, queries, boxes),
                       "attention_tensor_kernel");
}

}  // namespace
}  // namespace att

int attention_tensor_launch(const AttentionParams& p, int type, cudaStream_t st) {
    using namespace att;
    TensorMaps maps = {};
    if (int rc = encode_forward(&maps, p, type, TC_ROWS)) return rc;
    QueryMaps queries = {};
    int boxes = 0;
    if (int rc = encode_queries(&queries, &boxes, p, type)) return rc;
    if (type == ATT_BF16) return p.D <= 64 ? launch_tensor<__nv_bfloat16, 64>(p, maps, queries, boxes, st) : launch_tensor<__nv_bfloat16, 128>(p, maps, queries, boxes, st);
    return p.D <= 64 ? launch_tensor<__half, 64>(p, maps, queries, boxes, st) : launch_tensor<__half, 128>(p, maps, queries, boxes, st);
}

int attention_tensor_take_wait_flag() { return att::take_wait_flag(att::g_attention_wait_expired); }

}  // namespace km
