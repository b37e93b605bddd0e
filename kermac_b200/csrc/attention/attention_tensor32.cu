// Attention of many float32 queries on the tensor cores (tcgen05), head widths up to 64, to the accuracy of fp32.
//
// A float32 value is the sum of three bf16 ones (8 significant bits each), and a product of two such sums the six of their
// products that are not below 2^-24 of it.  One kernel writes the planes of Q, K and V (zeros for channels behind the last and
// for keys behind a sequence's length), the other is attention_tensor.cu with six products for one:
//   S = q3 k1 + q1 k3 + q2 k2 + q2 k1 + q1 k2 + q1 k1,   O_i = p3 v1 + p1 v3 + p2 v2 + p2 v1 + p1 v2 + p1 v1
// in this order, because the tensor cores add with the low bits cut off: only the last, large chain (4 or 8 instructions) loses
// bits that matter.  For the same reason a tile's O_i starts from zero, and the sum over the tiles is kept in registers, rounded.
//
// Two threads share a row, 64 keys and 32 channels each.  2 x 1000 x 1500 (8 heads of 64, ragged): the form on mma.sync
// (attention_rows.cu), whose warps split every value they read, takes 220 us a pass, this 53 (7 of them for the planes).  A call has
// to have more than 32 keys: 4 x 2000 queries (8 heads) with 33 take 28.1 us this way and 48.3 the other, 1024 queries 12.9 and 12.7, 17 of
// 4 heads 10.6 and 11.5; with 14 keys 28.0 and 32.1, 12.9 and 9.7, 10.5 and 8.4.
#include <algorithm>

#include "../km_build_tma.cuh"
#include "attention_tcgen05.cuh"

namespace km {
namespace att {
namespace {

__device__ int g_attention_tensor32_wait_expired = 0;

constexpr int P32_GROUPS = 2, P32_PLANES = 3, P32_OPERAND = P32_PLANES * TC_SLAB;      // 128 rows of 64 channels, three planes
constexpr int P32_SMEM = 1024 + (P32_GROUPS + 2) * P32_OPERAND;                        // Q of both row tiles, K, V
constexpr int P32_LOAD_WARP = 8 * P32_GROUPS, P32_MMA_WARP = P32_LOAD_WARP + 1, P32_BLOCK = 256 * P32_GROUPS + 128;
// of the 96 registers that 640 threads are launched with, the last four warps give up what the others take: 512 * 104 + 128 * 56
constexpr int P32_REGS_SOFTMAX = 104, P32_REGS_OTHERS = 56;
// tensor memory of a row tile: S, with the first two planes of P for 32 keys over these, the third plane, O
constexpr int P32_COLS = 256, P32_P3 = 128, P32_O = 192;

struct PlaneMaps { CUtensorMap q, qp, k, v, kp, vp; };

__device__ __forceinline__ void tile_sync(int t) { asm volatile("barrier.cta.sync %0, 256;" ::"r"(t + 1) : "memory"); }

// Takes the upper eight bits of a pair as bf16 (rounded) and leaves the rest.
__device__ __forceinline__ uint32_t take_plane(float& x, float& y) {
    const uint32_t plane = Type<__nv_bfloat16>::pair(x, y);
    x -= __uint_as_float(plane << 16), y -= __uint_as_float(plane & 0xffff0000u);
    return plane;
}

// planes[plane][index of the row][64]; PACKED (queries): rows (key head, l, n, head of the group), else (l, key head, row).
struct PlaneJob {
    Heads     src;
    uint16_t* planes;
    int       L, rows, heads, G, D, M, packed, vec;
    const int* lengths; long long lengths_stride;      // keys: rows behind the length are zeros
};
struct PlaneJobs { PlaneJob job[5]; int count; long long first[6]; };

// One thread for 8 channels of a row.
__global__ void __launch_bounds__(256) attention_planes_kernel(const PlaneJobs jobs) {
    after_previous_grid();
    const long long at = (static_cast<long long>(blockIdx.x) * 256 + threadIdx.x);
    if (at >= jobs.first[jobs.count]) return;
    int which = 0;
    while (which + 1 < jobs.count && at >= jobs.first[which + 1]) ++which;
    const PlaneJob& j = jobs.job[which];
    const long long unit = at - jobs.first[which], index = unit >> 3, total = static_cast<long long>(j.L) * j.rows * j.heads;
    const int       c = static_cast<int>(unit & 7) * 8;
    int l, row, h;
    if (j.packed) {
        const int g = static_cast<int>(index % j.G);
        long long rest = index / j.G;
        row = static_cast<int>(rest % j.rows), rest /= j.rows;
        l = static_cast<int>(rest % j.L);
        h = static_cast<int>(rest / j.L) * j.G + g;
    } else {
        row = static_cast<int>(index % j.rows);
        const long long rest = index / j.rows;
        h = static_cast<int>(rest % j.heads), l = static_cast<int>(rest / j.heads);
    }
    const bool   there = j.lengths == nullptr || row < key_count(j.lengths, j.lengths_stride, l, j.M);
    const float* src = reinterpret_cast<const float*>(j.src.ptr) + l * j.src.sl + row * j.src.sr + h * j.src.sh + c;
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; e += 4) {
        if (j.vec && there && c + e < j.D) {
            const float4 v = *reinterpret_cast<const float4*>(src + e);
            x[e] = v.x, x[e + 1] = v.y, x[e + 2] = v.z, x[e + 3] = v.w;
        } else {
#pragma unroll
            for (int f = 0; f < 4; ++f) x[e + f] = there && c + e + f < j.D ? src[e + f] : 0.0f;
        }
    }
#pragma unroll
    for (int plane = 0; plane < P32_PLANES; ++plane) {
        uint32_t y[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = take_plane(x[2 * e], x[2 * e + 1]);
        *reinterpret_cast<uint4*>(j.planes + (plane * total + index) * 64 + c) = make_uint4(y[0], y[1], y[2], y[3]);
    }
}

// Pairs of planes, the small products first.
__device__ __forceinline__ constexpr int left_plane(int i) { return i == 0 ? 2 : i == 1 ? 0 : i == 2 ? 1 : i == 3 ? 1 : 0; }
__device__ __forceinline__ constexpr int right_plane(int i) { return i == 0 ? 0 : i == 1 ? 2 : i == 2 ? 1 : i == 3 ? 0 : i == 4 ? 1 : 0; }

__global__ void __launch_bounds__(P32_BLOCK, 1)
attention_tensor32_kernel(const __grid_constant__ AttentionParams p, const __grid_constant__ PlaneMaps maps) {
    typedef __nv_bfloat16 T;
    extern __shared__ unsigned char smem_raw[];
    __shared__ __align__(8) unsigned long long s_bars[4 + 4 * P32_GROUPS];
    __shared__ uint32_t s_tmem;
    __shared__ int s_expired;
    __shared__ float s_half[P32_GROUPS][2][TC_ROWS];      // what the two threads of a row tell each other
    const uint32_t raw = smem_addr(smem_raw), base = (raw + 1023u) & ~1023u, bars = smem_addr(s_bars);
    const int      warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t k_full = bars, k_empty = bars + 8, v_full = bars + 16, v_empty = bars + 24;
    auto q_full = [&](int t) { return bars + 32 + 8u * t; };
    auto s_full = [&](int t) { return bars + 32 + 8u * (P32_GROUPS + t); };
    auto p_full = [&](int t) { return bars + 32 + 8u * (2 * P32_GROUPS + t); };
    auto o_full = [&](int t) { return bars + 32 + 8u * (3 * P32_GROUPS + t); };
    if (threadIdx.x == 0) {
        mbar_init(k_full, 1), mbar_init(k_empty, 1), mbar_init(v_full, 1), mbar_init(v_empty, 1);
        for (int t = 0; t < P32_GROUPS; ++t) mbar_init(q_full(t), 1), mbar_init(s_full(t), 1), mbar_init(p_full(t), 8), mbar_init(o_full(t), 1);
        s_expired = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        tc::fence_smem_to_async();
    }
    after_previous_grid();
    if (warp == P32_MMA_WARP) tc::tmem_alloc(smem_addr(&s_tmem), 512);
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
    const Work w = find_work<float, P32_BLOCK>(p, blockIdx.x, P32_GROUPS * TC_ROWS, TC_ROWS);
    const int  n_tiles = (w.end - w.first + TC_ROWS - 1) / TC_ROWS, groups = w.row0 + TC_ROWS < w.rows ? 2 : 1;
    const bool prefix = w.l < 0;
    const uint32_t tile_k = base + P32_GROUPS * P32_OPERAND, tile_v = tile_k + P32_OPERAND;

    if (warp < P32_LOAD_WARP) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(P32_REGS_SOFTMAX));
        // ------------------------------------------------------------------ softmax: thread = half a row
        const int t = warp >> 3, half = (warp >> 2) & 1, r = threadIdx.x & 127, at = w.row0 + t * TC_ROWS + r;
        const uint32_t mine = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16) + t * P32_COLS, s_col = mine + half * 64;
        const Row      row = find_row(p, w, min(at, w.rows - 1));
        if (t < groups) {
            const float c = p.scale_log2;                // at least 2^-149: -inf stays -inf
            const int   limit = min(row_limit(p, w, min(at, w.rows - 1)), w.end) - half * 64;
            const int   all_see = min(w.causal ? w.length - p.N + 1 : w.length, w.end);     // keys in front of it are seen by every row
            float top = -INFINITY, sum = 0.0f, o[32];
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = 0.0f;
            auto add_tile = [&] {                        // the products of a tile's weights with V
                uint32_t y[32];
                tmem_load32(mine + P32_O + half * 32, y);
                tmem_wait_load();
                tmem_loaded32(y);
#pragma unroll
                for (int e = 0; e < 32; ++e) o[e] += __uint_as_float(y[e]);
            };
            for (int i = 0; i < n_tiles; ++i) {
                const int first = w.first + i * TC_ROWS;
                wait(s_full(t), i & 1);
                tc::fence_after_sync();
                if (i > 0) add_tile();                   // issued before this S, so complete
                // S is read twice, 32 keys at a time: 64 of its values beside o and the planes of P do not fit the registers
                // (spilled: 56 us for the case above, this way 40)
                uint32_t   x[32];
                const bool masked = first + TC_ROWS > all_see;
                auto load = [&](int chunk) {
                    tmem_load32(s_col + chunk * 32, x);
                    tmem_wait_load();
                    tmem_loaded32(x);
                    if (masked) {
#pragma unroll
                        for (int j = 0; j < 32; ++j) x[j] = first + chunk * 32 + j < limit ? x[j] : 0xff800000u;
                    }
                };
                float best[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int chunk = 0; chunk < 2; ++chunk) {
                    load(chunk);
#pragma unroll
                    for (int j = 0; j < 32; j += 8)
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            best[e] = fmaxf(fmaxf(best[e], __uint_as_float(x[j + e])), __uint_as_float(x[j + 4 + e]));
                }
                tile_sync(t);                            // the other thread has read what the last tile left
                s_half[t][half][r] = fmaxf(fmaxf(best[0], best[1]), fmaxf(best[2], best[3]));
                tile_sync(t);
                const float high = fmaxf(top, fmaxf(s_half[t][0][r], s_half[t][1][r]));
                const float from = high == -INFINITY ? 0.0f : high;           // a row that sees nothing: exp2(-inf - 0) = 0
                const float shrink = top == -INFINITY ? 0.0f : ex2_approx((top - from) * c);
                top = high;
                sum *= shrink;
#pragma unroll
                for (int e = 0; e < 32; ++e) o[e] *= shrink;
                const u64 c2 = pack2(c, c), m2 = pack2(-from, -from);
                u64 total[2] = {0, 0};
#pragma unroll
                for (int chunk = 0; chunk < 2; ++chunk) {
                    load(chunk);
#pragma unroll
                    for (int j = 0; j < 16; j += 8) {
                        uint32_t y[P32_PLANES][8];
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            float lo, hi;
                            unpack2(mul2(add2(pack2(__uint_as_float(x[2 * (j + e)]), __uint_as_float(x[2 * (j + e) + 1])), m2), c2), lo, hi);
                            lo = ex2_approx(lo), hi = ex2_approx(hi);
                            total[e & 1] = add2(total[e & 1], pack2(lo, hi));
#pragma unroll
                            for (int plane = 0; plane < P32_PLANES; ++plane) y[plane][e] = take_plane(lo, hi);
                        }
                        // over the keys that were just read
                        tmem_store8(s_col + chunk * 32 + j, y[0]);
                        tmem_store8(s_col + chunk * 32 + 16 + j, y[1]);
                        tmem_store8(mine + P32_P3 + half * 32 + chunk * 16 + j, y[2]);
                    }
                }
                float a0, a1, a2, a3;
                unpack2(total[0], a0, a1);
                unpack2(total[1], a2, a3);
                sum += (a0 + a1) + (a2 + a3);
                tc::wait_st();
                tc::fence_before_sync();
                __syncwarp();
                if (lane == 0) mbar_arrive(p_full(t));
            }
            if (n_tiles > 0) {
                wait(o_full(t), 0);
                tc::fence_after_sync();
                add_tile();
            }
            tile_sync(t);
            s_half[t][half][r] = sum;
            tile_sync(t);
            sum = s_half[t][0][r] + s_half[t][1][r];
            const bool  good = *reinterpret_cast<volatile int*>(&s_expired) == 0 && at < w.rows;
            const float by   = sum == 0.0f ? 0.0f : 1.0f / sum;
            if (good && half == 0) put_stats(p, w, row, top == -INFINITY ? top : top * c, sum);
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] *= by;
            float* const out  = reinterpret_cast<float*>(p.out.ptr) + row.l * p.out.sl + row.n * p.out.sr + row.h * p.out.sh + half * 32;
            float* const part = p.part_o + ((((static_cast<long long>(w.part) * p.L + row.l) * p.N + row.n) * p.H) + row.h) * p.D + half * 32;
            float* const to   = p.parts > 1 ? part : out;
            if (p.parts > 1 ? p.D % 4 == 0 : p.vec_out) {
                // the warp's part of Q has been used for the last time (without keys nothing was copied there)
                char* const stage = reinterpret_cast<char*>(smem_raw) + (base - raw) + t * P32_OPERAND + (warp & 7) * 4096;
                store_rows(stage, reinterpret_cast<const uint32_t*>(o), good ? reinterpret_cast<char*>(to) : nullptr, (p.D - half * 32) / 4);
            } else if (good) {
#pragma unroll
                for (int e = 0; e < 32; ++e)
                    if (half * 32 + e < p.D) to[e] = o[e];
            }
        }
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(P32_REGS_OTHERS));
        if (warp == P32_LOAD_WARP) {
            // -------------------------------------------------------------- copies
            if (tc::elect_one() && n_tiles > 0) {
                const CUtensorMap *mq = prefix ? &maps.qp : &maps.q, *mk = prefix ? &maps.kp : &maps.k, *mv = prefix ? &maps.vp : &maps.v;
                const int kl = prefix || p.k.sl == 0 ? 0 : w.l, entries = prefix || p.k.sl == 0 ? 1 : p.L;
                auto load = [&](uint32_t to, const CUtensorMap* map, int first, uint32_t bar) {
                    mbar_expect_tx(bar, P32_OPERAND);
#pragma unroll
                    for (int plane = 0; plane < P32_PLANES; ++plane)
                        tma_load_box(to + plane * TC_SLAB, map, 0, first, w.hk, plane * entries + kl, bar);
                };
                for (int t = 0; t < groups; ++t) {
                    mbar_expect_tx(q_full(t), P32_OPERAND);
#pragma unroll
                    for (int plane = 0; plane < P32_PLANES; ++plane)
                        tma_load_box(base + t * P32_OPERAND + plane * TC_SLAB, mq, 0, w.row0 + t * TC_ROWS, prefix ? 0 : w.l, plane * p.Hk + w.hk,
                                     q_full(t));
                }
                for (int i = 0; i < n_tiles; ++i) {
                    if (i > 0) wait(k_empty, (i - 1) & 1);
                    load(tile_k, mk, w.first + i * TC_ROWS, k_full);
                    if (i > 0) wait(v_empty, (i - 1) & 1);
                    load(tile_v, mv, w.first + i * TC_ROWS, v_full);
                }
                for (int t = 0; t < groups; ++t) drain(q_full(t), 0);
                drain(k_full, (n_tiles - 1) & 1);
                drain(v_full, (n_tiles - 1) & 1);
            }
            __syncwarp();
        } else if (warp == P32_MMA_WARP && n_tiles > 0) {
            // -------------------------------------------------------------- products
            const uint64_t k_desc = desc_channels(tile_k), v_desc = desc_rows(tile_v);
            auto scores = [&](int t) {
                const uint64_t q_desc = desc_channels(base + t * P32_OPERAND);
                if (tc::elect_one()) {
#pragma unroll
                    for (int i = 0; i < 6; ++i)
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            mma_ss(tmem + t * P32_COLS, q_desc + left_plane(i) * (TC_SLAB >> 4) + k * 2, k_desc + right_plane(i) * (TC_SLAB >> 4) + k * 2,
                                   instr_desc<T>(128, false), i > 0 || k > 0);
                    tc::commit(s_full(t));
                }
                __syncwarp();
            };
            wait(k_full, 0);
            for (int t = 0; t < groups; ++t) {
                wait(q_full(t), 0);
                tc::fence_after_sync();
                scores(t);
            }
            issue_commit(k_empty);
            for (int i = 0; i < n_tiles; ++i) {
                wait(v_full, i & 1);
                for (int t = 0; t < groups; ++t) {
                    wait(p_full(t), i & 1);
                    tc::fence_after_sync();
                    if (tc::elect_one()) {
#pragma unroll
                        for (int j = 0; j < 6; ++j)
#pragma unroll
                            for (int k = 0; k < 8; ++k) {
                                const int plane = left_plane(j), at = plane == 2 ? P32_P3 + k * 8 : plane * 16 + (k >> 1) * 32 + (k & 1) * 8;
                                mma_ts(tmem + t * P32_COLS + P32_O, tmem + t * P32_COLS + at, v_desc + right_plane(j) * (TC_SLAB >> 4) + k * 128,
                                       instr_desc<T>(64, true), j > 0 || k > 0);
                            }
                        if (i == n_tiles - 1) tc::commit(o_full(t));
                    }
                    __syncwarp();
                }
                issue_commit(v_empty);
                if (i + 1 < n_tiles) {
                    wait(k_full, (i + 1) & 1);
                    tc::fence_after_sync();
                    for (int t = 0; t < groups; ++t) scores(t);
                    issue_commit(k_empty);
                }
            }
            // every product has ended before tensor memory is given back
            for (int t = 0; t < groups; ++t) drain(o_full(t), 0);
        }
    }
    tc::fence_before_sync();
    __syncthreads();
    tc::fence_after_sync();
    if (warp == P32_MMA_WARP) tc::tmem_dealloc(tmem, 512);
    if (threadIdx.x == 0 && s_expired) g_attention_tensor32_wait_expired = 1;
}

long long plane_bytes(long long rows) { return rows * 64 * 2 * P32_PLANES; }

}  // namespace
}  // namespace att

// Bytes of planes of a call: queries, and those keys and values that it has.
long long attention_planes_bytes(const AttentionParams& p) {
    using namespace att;
    return plane_bytes(static_cast<long long>(p.L) * p.N * p.H) + 2 * plane_bytes(static_cast<long long>(p.k.sl == 0 ? 1 : p.L) * p.M * p.Hk) +
           2 * plane_bytes(static_cast<long long>(p.P) * p.Hk);
}

int attention_tensor32_launch(const AttentionParams& p, void* planes, cudaStream_t st) {
    using namespace att;
    PlaneJobs jobs = {};
    PlaneMaps maps = {};
    char*     at = static_cast<char*>(planes);
    auto add = [&](const Heads& src, int L, int rows, int heads, int G, bool packed, const int* lengths) {
        PlaneJob& j = jobs.job[jobs.count];
        j.src = src, j.planes = reinterpret_cast<uint16_t*>(at), j.L = L, j.rows = rows, j.heads = heads, j.G = G, j.D = p.D, j.M = p.M;
        j.packed = packed, j.vec = p.vec, j.lengths = lengths, j.lengths_stride = p.lengths_stride;
        const long long index = static_cast<long long>(L) * rows * heads;
        jobs.first[jobs.count + 1] = jobs.first[jobs.count] + index * 8;
        ++jobs.count;
        at += plane_bytes(index);
        return static_cast<void*>(j.planes);
    };
    // planes as a rank-4 tensor of rows of 64 channels: y rows, z and w the two indexes above
    auto encode = [&](CUtensorMap* map, void* base, long long y, long long z, long long w) {
        const cuuint64_t dims[4]    = {64, static_cast<cuuint64_t>(y), static_cast<cuuint64_t>(z), static_cast<cuuint64_t>(w)};
        const cuuint64_t strides[3] = {128, static_cast<cuuint64_t>(128 * y), static_cast<cuuint64_t>(128 * y * z)};
        const cuuint32_t box[4]     = {64, TC_ROWS, 1, 1};
        return encode_tma_16bit(map, base, true, dims, strides, box);
    };
    int rc = 0;
    void* const q = add(p.q, p.L, p.N, p.H, p.G, true, nullptr);
    const long long rows = static_cast<long long>(p.N) * p.G;
    if (p.own_tiles > 0 && p.M > 0) {
        // (k and v that are broadcast over entries of different lengths are not taken: one set of planes cannot have zeros for each)
        const int entries = p.k.sl == 0 ? 1 : p.L;
        rc = encode(&maps.q, q, rows, p.L, 3LL * p.Hk);
        if (!rc) rc = encode(&maps.k, add(p.k, entries, p.M, p.Hk, 1, false, p.lengths), p.M, p.Hk, 3LL * entries);
        if (!rc) rc = encode(&maps.v, add(p.v, entries, p.M, p.Hk, 1, false, p.lengths), p.M, p.Hk, 3LL * entries);
    }
    if (!rc && p.prefix_tiles > 0) {
        rc = encode(&maps.qp, q, rows * p.L, 1, 3LL * p.Hk);
        if (!rc) rc = encode(&maps.kp, add(p.kp, 1, p.P, p.Hk, 1, false, nullptr), p.P, p.Hk, 3);
        if (!rc) rc = encode(&maps.vp, add(p.vp, 1, p.P, p.Hk, 1, false, nullptr), p.P, p.Hk, 3);
    }
    if (!rc) rc = cuda_status(cudaFuncSetAttribute(attention_tensor32_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, P32_SMEM), "cudaFuncSetAttribute");
    const long long plane_blocks = ceil_div_ll(jobs.first[jobs.count], 256);
    unsigned        blocks;
    if (!rc) rc = count_blocks(p, &blocks);
    if (!rc && plane_blocks > 0x7fffffffLL) rc = fail(KM_ERR_TOO_LARGE, "attention: more than 2^31 - 1 blocks");
    if (!rc)
        rc = cuda_status(launch_overlapped(&attention_planes_kernel, dim3(static_cast<unsigned>(plane_blocks)), 256, 0, st, jobs),
                         "attention_planes_kernel");
    if (!rc)
        rc = cuda_status(launch_overlapped(&attention_tensor32_kernel, dim3(blocks), P32_BLOCK, P32_SMEM, st, p, maps), "attention_tensor32_kernel");
    return rc;
}

int attention_tensor32_take_wait_flag() { return att::take_wait_flag(att::g_attention_tensor32_wait_expired); }

}  // namespace km
