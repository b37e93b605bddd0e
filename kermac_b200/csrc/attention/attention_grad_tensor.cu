// Gradient of the attention of 16-bit tensors on the tensor cores (tcgen05), head widths up to 128.
//
// Two kinds of blocks, like the two kernels of attention_grad_rows.cu: one holds 128 keys and streams query tiles (dk, dv), one holds 128 queries and streams
// key tiles (dq).  One launch has both, the longer ones first, so that the SMs that have finished those go on with the others
// (two launches: a training step of 8 x 512 x 1030 waited twice for its last blocks, 140 of 195 us).
//
// delta from the output as the forward pass rounded it is off by up to half a step of the output's terms, which shows where few keys
// share a query: dq and dk had 1.9 times the error of rounding the weights' gradients and the results with 2 keys, 1.36 with 5, 1.2 with 11, 1.04
// with 128.  Entries of the batch whose keys are in one tile, however far they are padded, form it from its own terms, sum_m p (dout v^T), which
// both kinds of blocks have at hand (1.0 then); where no entry can have more there is no pass over out and dout.  Scores and dout v^T are in
// tensor memory, the weights and their gradients are written back over them as 16-bit operands.  The keys' kernel computes both transposed, so that its operands need no transposition either: a
// lane is a key there and a query in the other kernel.
//
// Tensor memory has no room for a second set of both products beside the 128-channel sums dk and dv, and needs none: what the tensor
// cores do is cut in two, and the weights' warps (eight, 64 columns each) work on the other half meanwhile,
//   tensor cores:  dv(i), s(i + 1)   | dk(i), dp(i + 1)
//   warps:         ds(i)             | p(i + 1)
#include <algorithm>

#include "attention_grad.cuh"
#include "attention_tcgen05.cuh"

namespace km {
namespace att {
namespace {

__device__ int g_attention_grad_wait_expired = 0;

template <int DP>
struct GradTensorShape {
    static constexpr int TILE = DP / 64 * TC_SLAB;
    static constexpr int WARPS_ON_WEIGHTS = 8, LOAD_WARP = 8, MMA_WARP = 9, STATS_WARP = 10, BLOCK = 384;
    static constexpr int KEYS_STAGES = 2;                                   // keys' kernel: tiles of q, and of dout, under way
    static constexpr int K_STAGES = 3, V_STAGES = 2;                        // queries' kernel: k is needed again for dq
    static constexpr int KEYS_SMEM    = 1024 + (2 + 2 * KEYS_STAGES) * TILE + (2 * 2 + 4) * TC_ROWS * 4;      // with lse and delta, and parts of an exact delta
    static constexpr int QUERIES_SMEM = 1024 + (2 + K_STAGES + V_STAGES) * TILE;
    // more than half of an SM's shared memory: a second block would wait inside tcgen05.alloc
    static constexpr int at_least_half(int n) { return n > 115 * 1024 ? n : 115 * 1024; }
};

struct GradMaps { CUtensorMap q, k, v, dout; };

// Bounded waits of one warp; once one has run out the warp stops waiting, and the block writes nothing.
struct Waits {
    int* flag;
    bool expired = false;
    __device__ __forceinline__ void operator()(uint32_t bar, int parity) {
        if (!expired && !mbar_wait_bounded(bar, parity)) {
            expired = true;
            *reinterpret_cast<volatile int*>(flag) = 1;
        }
    }
    // what is in flight at the end is waited for (with a limit) in any case
    __device__ __forceinline__ void drain(uint32_t bar, int parity) {
        if (!mbar_wait_bounded(bar, parity, expired ? 1 << 16 : MBAR_WAIT_TRIES)) *reinterpret_cast<volatile int*>(flag) = 1;
    }
};

template <int DP>
__device__ __forceinline__ void load_tile(uint32_t dst, const CUtensorMap* map, int row, int head, int l, uint32_t bar) {
#pragma unroll
    for (int d = 0; d < DP / 64; ++d) tma_load_rows(dst + d * TC_SLAB, map, d * 64, row, head, l, bar);
}

// Columns [0, DP) of a warp's rows of sums, times `by`, into a gradient or a slice's 32-bit sums (part).  `stage`: 4 KB.
template <typename T, int DP>
__device__ __forceinline__ void put_sums(uint32_t columns, char* stage, const Heads& to, float* part, bool vec, bool good, int l, int row, int h,
                                         int rows, int heads, int D, float by) {
    if (part || vec) {
        char* const at   = to.ptr + (l * to.sl + row * to.sr + h * to.sh) * 2;
        char* const sums = reinterpret_cast<char*>(part + ((static_cast<long long>(l) * rows + row) * heads + h) * D);
        store_sums<T, DP>(columns, stage, good && !part ? at : nullptr, good && part ? sums : nullptr, part != nullptr, D, by);
    } else {
#pragma unroll
        for (int j = 0; j < DP; j += 32) {
            uint32_t x[32];
            tmem_load32(columns + j, x);
            tmem_wait_load();
            tmem_loaded32(x);
            if (!good) continue;
#pragma unroll
            for (int e = 0; e < 32; e += 2)
                put_grad<T>(to, part, l, row, h, rows, heads, D, j + e, __uint_as_float(x[e]) * by, __uint_as_float(x[e + 1]) * by);
        }
    }
}
// Zeros instead.
template <typename T>
__device__ __forceinline__ void put_zeros(const Heads& to, float* part, bool vec, bool good, int l, int row, int h, int rows, int heads, int D) {
    if (part || vec) {
        char* const at   = to.ptr + (l * to.sl + row * to.sr + h * to.sh) * 2;
        char* const sums = reinterpret_cast<char*>(part + ((static_cast<long long>(l) * rows + row) * heads + h) * D);
        const u64   mine = good ? reinterpret_cast<u64>(part ? sums : at) : 0;
        const int   lane = threadIdx.x & 31, chunks = part ? D / 4 : D / 8;
#pragma unroll 8
        for (int i = 0; i < 32; ++i) {
            char* const row_at = reinterpret_cast<char*>(__shfl_sync(0xffffffffu, mine, i));
            if (row_at != nullptr)
                for (int c = lane; c < chunks; c += 32) *reinterpret_cast<uint4*>(row_at + c * 16) = make_uint4(0, 0, 0, 0);
        }
    } else if (good) {
        for (int c = 0; c < D; c += 2) put_grad<T>(to, part, l, row, h, rows, heads, D, c, 0.0f, 0.0f);
    }
}

// dk and dv of 128 keys.
template <typename T, int DP>
__device__ __forceinline__ void gradient_of_keys(const AttentionGradParams& p, const GradMaps& maps, int block) {
    typedef GradTensorShape<DP> S;
    constexpr int ST = S::KEYS_STAGES;
    extern __shared__ unsigned char smem_raw[];
    __shared__ __align__(8) unsigned long long s_bars[6 * ST + 6];
    __shared__ uint32_t s_tmem;
    __shared__ int s_expired;
    const uint32_t raw = smem_addr(smem_raw), base = (raw + 1023u) & ~1023u, bars = smem_addr(s_bars);
    const int      warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    auto q_full  = [&](int st) { return bars + 8u * st; };
    auto q_empty = [&](int st) { return bars + 8u * (ST + st); };
    auto d_full  = [&](int st) { return bars + 8u * (2 * ST + st); };
    auto d_empty = [&](int st) { return bars + 8u * (3 * ST + st); };
    auto t_full  = [&](int st) { return bars + 8u * (4 * ST + st); };       // lse and delta of a query tile
    auto t_empty = [&](int st) { return bars + 8u * (5 * ST + st); };
    const uint32_t held_full = bars + 8u * (6 * ST), s_full = held_full + 8, dp_full = held_full + 16, p_ready = held_full + 24,
                   ds_ready = held_full + 32, done = held_full + 40;
    if (threadIdx.x == 0) {
        for (int st = 0; st < ST; ++st) {
            mbar_init(q_full(st), 1), mbar_init(q_empty(st), 1), mbar_init(d_full(st), 1), mbar_init(d_empty(st), 1);
            mbar_init(t_full(st), 1), mbar_init(t_empty(st), S::WARPS_ON_WEIGHTS);
        }
        mbar_init(held_full, 1), mbar_init(s_full, 1), mbar_init(dp_full, 1), mbar_init(done, 1);
        mbar_init(p_ready, S::WARPS_ON_WEIGHTS), mbar_init(ds_ready, S::WARPS_ON_WEIGHTS);
        s_expired = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        tc::fence_smem_to_async();
    }
    if (warp == S::MMA_WARP) tc::tmem_alloc(smem_addr(&s_tmem), 512);

    // (key tile, slice, key head, batch entry of k and v)
    const int tiles = (p.M + TC_ROWS - 1) / TC_ROWS;
    const int key0 = block % tiles * TC_ROWS; block /= tiles;
    const int slice = block % p.kv_slices;    block /= p.kv_slices;
    const int hk = block % p.Hk, kl = block / p.Hk;
    const int l_count = p.kv_batch == 1 ? p.L : 1, l_first = p.kv_batch == 1 ? 0 : kl;
    const int q_tiles = (p.N + TC_ROWS - 1) / TC_ROWS;
    const int all     = l_count * p.G * q_tiles;
    const int each = all / p.kv_slices, more = all % p.kv_slices;       // the first `more` pieces have one item more
    const int from = slice * each + min(slice, more), to = from + each + (slice < more);
    int longest = 0;                               // keys from here on are in no sum of this block: their gradient is zero
    if (from < to)
        for (int l = l_first + from / (p.G * q_tiles); l <= l_first + (to - 1) / (p.G * q_tiles); ++l)
            longest = max(longest, key_count(p.lengths, p.lengths_stride, l, p.M));
    const int n_items = key0 < longest ? to - from : 0;
    // asked for by the warps that need it, while the copies are under way
    auto find_this_factor = [&] { return n_items > 0 ? find_factor<T>(p, l_first, l_first + l_count, hk, kl, longest) : 1.0f; };

    tc::fence_before_sync();
    __syncthreads();
    tc::fence_after_sync();
    const uint32_t tmem = s_tmem, s_col = tmem, dp_col = tmem + 128, dv_col = tmem + 256, dk_col = tmem + 256 + DP;
    const uint32_t held_k = base, held_v = base + S::TILE, ring_q = base + 2 * S::TILE, ring_d = ring_q + ST * S::TILE;
    float* const   stats = reinterpret_cast<float*>(smem_raw + (base - raw) + (2 + 2 * ST) * S::TILE);
    float* const   parts = stats + 2 * 2 * TC_ROWS;        // [4][128]: the sums of 32 keys each
    Waits wait{&s_expired};

    if (warp < S::WARPS_ON_WEIGHTS) {
        // ------------------------------------------------------------------ weights: lane = key, 64 queries of a tile
        const float    factor = find_this_factor(), by = factor * per_weight<T>;
        const int      half = warp >> 2, key = key0 + (threadIdx.x & 127);
        const uint32_t at   = (static_cast<uint32_t>((warp & 3) * 32) << 16) + half * 64;
        const u64      c2 = pack2(p.scale_log2, p.scale_log2), by2 = pack2(by, by);
        for (int i = 0; i < n_items; ++i) {
            const int  st   = i % ST;
            const int  count = key_count(p.lengths, p.lengths_stride, l_first + (from + i) / (p.G * q_tiles), p.M);
            const bool seen = key < count;
            const ulonglong2* const lse   = reinterpret_cast<const ulonglong2*>(stats + st * 2 * TC_ROWS + half * 64);
            const ulonglong2* const delta = reinterpret_cast<const ulonglong2*>(stats + st * 2 * TC_ROWS + TC_ROWS + half * 64);
            uint32_t w[64];
            wait(t_full(st), (i / ST) & 1);
            wait(s_full, i & 1);
            tc::fence_after_sync();
            tmem_load32(s_col + at, w);
            tmem_load32(s_col + at + 32, w + 32);
            tmem_wait_load();
            tmem_loaded32(w);
            tmem_loaded32(w + 32);
            uint32_t y[32];
#pragma unroll
            for (int j = 0; j < 64; j += 4) {
                const ulonglong2 shift = lse[j / 4];       // -lse * log2(e), -inf behind the last query
                float x[4];
                unpack2(fma2(pack2(__uint_as_float(w[j]), __uint_as_float(w[j + 1])), c2, shift.x), x[0], x[1]);
                unpack2(fma2(pack2(__uint_as_float(w[j + 2]), __uint_as_float(w[j + 3])), c2, shift.y), x[2], x[3]);
#pragma unroll
                for (int e = 0; e < 4; ++e) x[e] = ex2_approx(x[e]), w[j + e] = __float_as_uint(x[e]);
                y[j / 2]     = seen ? Type<T>::pair(x[0], x[1]) : 0;
                y[j / 2 + 1] = seen ? Type<T>::pair(x[2], x[3]) : 0;
            }
            tmem_store32(s_col + at, y);
            tc::wait_st();
            tc::fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive(p_ready);

            wait(dp_full, i & 1);
            tc::fence_after_sync();
            if (count <= TC_ROWS && key0 == 0) {
                // every key of the entry is here: delta = sum_m p (dout v^T), over the lanes
#pragma unroll
                for (int j = 0; j < 64; j += 32) {
                    uint32_t g[32];
                    tmem_load32(dp_col + at + j, g);
                    tmem_wait_load();
                    tmem_loaded32(g);
                    float x[32];
#pragma unroll
                    for (int e = 0; e < 32; ++e) x[e] = seen ? __uint_as_float(w[j + e]) * __uint_as_float(g[e]) : 0.0f;
                    // each step halves the columns that a lane has and adds those of its partner; column `lane` is left
#pragma unroll
                    for (int d = 16; d; d >>= 1)
#pragma unroll
                        for (int e = 0; e < d; ++e) {
                            const bool  upper = lane & d;
                            const float other = __shfl_xor_sync(0xffffffffu, upper ? x[e] : x[e + d], d);
                            x[e] = (upper ? x[e + d] : x[e]) + other;
                        }
                    parts[(warp & 3) * TC_ROWS + half * 64 + j + lane] = x[0] * per_weight<T>;
                }
                asm volatile("barrier.cta.sync 1, 256;" ::: "memory");
                if (half == 0) {
                    const int n = threadIdx.x & 127;
                    stats[st * 2 * TC_ROWS + TC_ROWS + n] = -((parts[n] + parts[TC_ROWS + n]) + (parts[2 * TC_ROWS + n] + parts[3 * TC_ROWS + n])) * by;
                }
                asm volatile("barrier.cta.sync 1, 256;" ::: "memory");
            }
#pragma unroll
            for (int j = 0; j < 64; j += 32) {
                uint32_t g[32];
                tmem_load32(dp_col + at + j, g);
                tmem_wait_load();
                tmem_loaded32(g);
#pragma unroll
                for (int e = 0; e < 32; e += 4) {
                    const ulonglong2 d = delta[(j + e) / 4];       // -delta * by
                    float x[4];
                    unpack2(mul2(pack2(__uint_as_float(w[j + e]), __uint_as_float(w[j + e + 1])),
                                 fma2(pack2(__uint_as_float(g[e]), __uint_as_float(g[e + 1])), by2, d.x)), x[0], x[1]);
                    unpack2(mul2(pack2(__uint_as_float(w[j + e + 2]), __uint_as_float(w[j + e + 3])),
                                 fma2(pack2(__uint_as_float(g[e + 2]), __uint_as_float(g[e + 3])), by2, d.y)), x[2], x[3]);
                    y[(j + e) / 2]     = seen ? Type<T>::pair(x[0], x[1]) : 0;
                    y[(j + e) / 2 + 1] = seen ? Type<T>::pair(x[2], x[3]) : 0;
                }
            }
            tmem_store32(dp_col + at, y);
            tc::wait_st();
            tc::fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive(t_empty(st)), mbar_arrive(ds_ready);
        }
        if (n_items > 0) {
            wait(done, 0);
            tc::fence_after_sync();
        }
        const bool good = key < p.M && *reinterpret_cast<volatile int*>(&s_expired) == 0;
        // the first half of the warps writes dv, the second dk
        const Heads& dst   = half == 0 ? p.dv : p.dk;
        float* const whole = half == 0 ? p.dv_part : p.dk_part;
        float* const part  = p.kv_slices > 1 ? whole + static_cast<long long>(slice) * p.kv_batch * p.M * p.Hk * p.D : nullptr;
        const float  times = half == 0 ? per_weight<T> : p.scale / factor;
        const uint32_t sums = (half == 0 ? dv_col : dk_col) + (static_cast<uint32_t>((warp & 3) * 32) << 16);
        if (n_items > 0) {
            // q and dout tiles have been used for the last time
            char* const stage = reinterpret_cast<char*>(smem_raw) + (ring_q - raw) + warp * 4096;
            put_sums<T, DP>(sums, stage, dst, part, p.vec_grad, good, kl, key, hk, p.M, p.Hk, p.D, times);
        } else {
            put_zeros<T>(dst, part, p.vec_grad, good, kl, key, hk, p.M, p.Hk, p.D);
        }
    } else if (warp == S::LOAD_WARP) {
        // ------------------------------------------------------------------ copies
        if (tc::elect_one() && n_items > 0) {
            const int l_kv = p.k.sl == 0 ? 0 : kl, l_v = p.v.sl == 0 ? 0 : kl;
            mbar_expect_tx(held_full, 2 * S::TILE);
            load_tile<DP>(held_k, &maps.k, key0, hk, l_kv, held_full);
            load_tile<DP>(held_v, &maps.v, key0, hk, l_v, held_full);
            for (int i = 0; i < n_items; ++i) {
                const int st = i % ST, item = from + i, lg = item / q_tiles, l = l_first + lg / p.G, h = hk * p.G + lg % p.G;
                const int n0 = item % q_tiles * TC_ROWS;
                if (i >= ST) wait(q_empty(st), (i / ST - 1) & 1);
                mbar_expect_tx(q_full(st), S::TILE);
                load_tile<DP>(ring_q + st * S::TILE, &maps.q, n0, h, p.q.sl == 0 ? 0 : l, q_full(st));
                if (i >= ST) wait(d_empty(st), (i / ST - 1) & 1);
                mbar_expect_tx(d_full(st), S::TILE);
                load_tile<DP>(ring_d + st * S::TILE, &maps.dout, n0, h, p.dout.sl == 0 ? 0 : l, d_full(st));
            }
            wait.drain(held_full, 0);
            for (int i = max(0, n_items - ST); i < n_items; ++i) {
                wait.drain(q_full(i % ST), (i / ST) & 1);
                wait.drain(d_full(i % ST), (i / ST) & 1);
            }
        }
        __syncwarp();
    } else if (warp == S::STATS_WARP) {
        // ------------------------------------------------------------------ lse and delta of the query tiles
        const float by = find_this_factor() * per_weight<T>;
        for (int i = 0; i < n_items; ++i) {
            const int st = i % ST, item = from + i, lg = item / q_tiles, l = l_first + lg / p.G, h = hk * p.G + lg % p.G;
            const int n0 = item % q_tiles * TC_ROWS;
            const float* const lse   = p.lse + l * p.lse_sl + h * p.lse_sh;
            const float* const delta = p.delta + (static_cast<long long>(l) * p.H + h) * p.N;
            float a[4], d[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int n = n0 + e * 32 + lane;
                a[e] = n < p.N ? weight_log2<T> - lse[n] * (1.0f / LN2) : -INFINITY;
                d[e] = n < p.N && !p.own_delta ? -delta[n] * by : 0.0f;
            }
            if (i >= ST) wait(t_empty(st), (i / ST - 1) & 1);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                stats[st * 2 * TC_ROWS + e * 32 + lane]           = a[e];
                stats[st * 2 * TC_ROWS + TC_ROWS + e * 32 + lane] = d[e];
            }
            __threadfence_block();
            __syncwarp();
            if (lane == 0) mbar_arrive(t_full(st));
        }
    } else if (warp == S::MMA_WARP && n_items > 0) {
        // ------------------------------------------------------------------ products
        wait(held_full, 0);
        wait(q_full(0), 0);
        tc::fence_after_sync();
        issue_channels<T, DP>(p.D, s_col, desc_channels(held_k), desc_channels(ring_q), s_full);
        wait(d_full(0), 0);
        tc::fence_after_sync();
        issue_channels<T, DP>(p.D, dp_col, desc_channels(held_v), desc_channels(ring_d), dp_full);
        for (int i = 0; i < n_items; ++i) {
            const int st = i % ST, next = (i + 1) % ST;
            wait(p_ready, i & 1);
            tc::fence_after_sync();
            issue_rows<T, DP>(p.D, dv_col, s_col, desc_rows(ring_d + st * S::TILE), i > 0);
            issue_commit(d_empty(st));
            if (i + 1 < n_items) {
                wait(q_full(next), ((i + 1) / ST) & 1);
                tc::fence_after_sync();
                issue_channels<T, DP>(p.D, s_col, desc_channels(held_k), desc_channels(ring_q + next * S::TILE), s_full);
            }
            wait(ds_ready, i & 1);
            tc::fence_after_sync();
            issue_rows<T, DP>(p.D, dk_col, dp_col, desc_rows(ring_q + st * S::TILE), i > 0);
            issue_commit(q_empty(st));
            if (i + 1 < n_items) {
                wait(d_full(next), ((i + 1) / ST) & 1);
                tc::fence_after_sync();
                issue_channels<T, DP>(p.D, dp_col, desc_channels(held_v), desc_channels(ring_d + next * S::TILE), dp_full);
            }
        }
        issue_commit(done);
        wait.drain(done, 0);
    }
    tc::fence_before_sync();
    __syncthreads();
    tc::fence_after_sync();
    if (warp == S::MMA_WARP) tc::tmem_dealloc(tmem, 512);
    if (threadIdx.x == 0 && s_expired) g_attention_grad_wait_expired = 1;
}

// dq of 128 queries of a head.
template <typename T, int DP>
__device__ __forceinline__ void gradient_of_queries(const AttentionGradParams& p, const GradMaps& maps, int block) {
    typedef GradTensorShape<DP> S;
    constexpr int KS = S::K_STAGES, VS = S::V_STAGES;
    extern __shared__ unsigned char smem_raw[];
    __shared__ __align__(8) unsigned long long s_bars[2 * KS + 2 * VS + 6];
    __shared__ float s_part[2][TC_ROWS];
    __shared__ uint32_t s_tmem;
    __shared__ int s_expired;
    const uint32_t raw = smem_addr(smem_raw), base = (raw + 1023u) & ~1023u, bars = smem_addr(s_bars);
    const int      warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    auto k_full  = [&](int st) { return bars + 8u * st; };
    auto k_empty = [&](int st) { return bars + 8u * (KS + st); };
    auto v_full  = [&](int st) { return bars + 8u * (2 * KS + st); };
    auto v_empty = [&](int st) { return bars + 8u * (2 * KS + VS + st); };
    const uint32_t held_full = bars + 8u * (2 * KS + 2 * VS), dp_full = held_full + 8, ds_ready = held_full + 16, done = held_full + 24;
    auto s_full  = [&](int buf) { return held_full + 32 + 8u * buf; };
    if (threadIdx.x == 0) {
        for (int st = 0; st < KS; ++st) mbar_init(k_full(st), 1), mbar_init(k_empty(st), 1);
        for (int st = 0; st < VS; ++st) mbar_init(v_full(st), 1), mbar_init(v_empty(st), 1);
        mbar_init(held_full, 1), mbar_init(dp_full, 1), mbar_init(done, 1), mbar_init(s_full(0), 1), mbar_init(s_full(1), 1);
        mbar_init(ds_ready, S::WARPS_ON_WEIGHTS);
        s_expired = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        tc::fence_smem_to_async();
    }
    if (warp == S::MMA_WARP) tc::tmem_alloc(smem_addr(&s_tmem), 512);

    const int tiles = (p.N + TC_ROWS - 1) / TC_ROWS;
    const int n0 = block % tiles * TC_ROWS; block /= tiles;
    const int split = block % p.q_splits;   block /= p.q_splits;
    const int h = block % p.H, l = block / p.H, hk = h / p.G;
    const int kl = p.kv_batch == 1 ? 0 : l;
    // this block's piece of the keys: tiles [first, first + n_items)
    const int count = key_count(p.lengths, p.lengths_stride, l, p.M), key_tiles = (count + TC_ROWS - 1) / TC_ROWS;
    const int first = key_tiles * split / p.q_splits, n_items = key_tiles * (split + 1) / p.q_splits - first;      // at most 2^23 tiles, 64 pieces

    tc::fence_before_sync();
    __syncthreads();
    tc::fence_after_sync();
    // two sets of scores: the next one is ready when the warps come to it
    const uint32_t tmem = s_tmem, dp_col = tmem + 256, dq_col = tmem + 384;
    const uint32_t held_q = base, held_d = base + S::TILE, ring_k = base + 2 * S::TILE, ring_v = ring_k + KS * S::TILE;
    Waits wait{&s_expired};

    if (warp < S::WARPS_ON_WEIGHTS) {
        // ------------------------------------------------------------------ weights: lane = query, 64 keys of a tile
        const int      half = warp >> 2, n = n0 + (threadIdx.x & 127);
        const float    factor = n_items > 0 ? row_factor<T>(p, l, h, n, find_v_peak<T>(p, kl, hk, count)) : 1.0f;
        const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16, at = lanes + half * 64;
        const float    shift = n < p.N ? -p.lse[l * p.lse_sl + h * p.lse_sh + n] * (1.0f / LN2) : -INFINITY;
        const float    delta = n < p.N && !p.own_delta ? -p.delta[(static_cast<long long>(l) * p.H + h) * p.N + n] * factor : 0.0f;
        const u64      c2 = pack2(p.scale_log2, p.scale_log2), by2 = pack2(factor, factor), shift2 = pack2(shift, shift);
        u64            delta2 = pack2(delta, delta);
        for (int i = 0; i < n_items; ++i) {
            uint32_t w[64];
            wait(s_full(i & 1), (i >> 1) & 1);
            tc::fence_after_sync();
            tmem_load32(tmem + (i & 1) * 128 + at, w);
            tmem_load32(tmem + (i & 1) * 128 + at + 32, w + 32);
            tmem_wait_load();
            tmem_loaded32(w);
            tmem_loaded32(w + 32);
#pragma unroll
            for (int j = 0; j < 64; j += 2) {
                float x, y;
                unpack2(fma2(pack2(__uint_as_float(w[j]), __uint_as_float(w[j + 1])), c2, shift2), x, y);
                w[j] = __float_as_uint(ex2_approx(x)), w[j + 1] = __float_as_uint(ex2_approx(y));
            }
            const int  there = count - (first + i) * TC_ROWS;          // keys of this tile
            const bool tail  = there < TC_ROWS;
            if (tail && count < p.M) {
                // rows of k behind the length hold whatever the memory holds, and 0 * NaN is NaN
                const int st = i % KS;
                wait(k_full(st), (i / KS) & 1);
                char* const tile = reinterpret_cast<char*>(smem_raw) + (ring_k - raw) + st * S::TILE;
                for (int e = there * 8 + static_cast<int>(threadIdx.x); e < TC_ROWS * 8; e += 32 * S::WARPS_ON_WEIGHTS)
#pragma unroll
                    for (int d = 0; d < DP / 64; ++d) *reinterpret_cast<uint4*>(tile + d * TC_SLAB + e * 16) = make_uint4(0, 0, 0, 0);
                tc::fence_smem_to_async();
            }
            wait(dp_full, i & 1);
            tc::fence_after_sync();
            if (count <= TC_ROWS) {
                // every key of the entry is here: delta = sum_m p (dout v^T)
                float part = 0.0f;
#pragma unroll
                for (int j = 0; j < 64; j += 32) {
                    uint32_t g[32];
                    tmem_load32(dp_col + at + j, g);
                    tmem_wait_load();
                    tmem_loaded32(g);
#pragma unroll
                    for (int e = 0; e < 32; ++e)
                        if (half * 64 + j + e < there) part = fmaf(__uint_as_float(w[j + e]), __uint_as_float(g[e]), part);
                }
                s_part[half][threadIdx.x & 127] = part;
                asm volatile("barrier.cta.sync 1, 256;" ::: "memory");
                const float all = s_part[0][threadIdx.x & 127] + s_part[1][threadIdx.x & 127];
                delta2 = pack2(-all * factor, -all * factor);
            }
            uint32_t y[32];
#pragma unroll
            for (int j = 0; j < 64; j += 32) {
                uint32_t g[32];
                tmem_load32(dp_col + at + j, g);
                tmem_wait_load();
                tmem_loaded32(g);
#pragma unroll
                for (int e = 0; e < 32; e += 2) {
                    float x0, x1;
                    unpack2(mul2(pack2(__uint_as_float(w[j + e]), __uint_as_float(w[j + e + 1])),
                                 fma2(pack2(__uint_as_float(g[e]), __uint_as_float(g[e + 1])), by2, delta2)), x0, x1);
                    if (tail) {
                        x0 = half * 64 + j + e < there ? x0 : 0.0f;
                        x1 = half * 64 + j + e + 1 < there ? x1 : 0.0f;
                    }
                    y[(j + e) / 2] = Type<T>::pair(x0, x1);
                }
            }
            tmem_store32(dp_col + at, y);
            tc::wait_st();
            tc::fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive(ds_ready);
        }
        if (n_items > 0) {
            wait(done, 0);
            tc::fence_after_sync();
        }
        const bool   good = n < p.N && *reinterpret_cast<volatile int*>(&s_expired) == 0;
        // partial sums [slice][entry of q][n][h][D]: a broadcast q has one entry and a slice for each l and piece
        const bool   one_q = p.q_slices > p.q_splits;
        float* const part = p.q_slices > 1 ? p.dq_part + static_cast<long long>(one_q ? l * p.q_splits + split : split * p.L) * p.N * p.H * p.D : nullptr;
        if (n_items > 0) {
            if (half == 0) {                 // the warps of the first half write whole rows, where q was held
                char* const stage = reinterpret_cast<char*>(smem_raw) + (held_q - raw) + warp * 4096;
                put_sums<T, DP>(dq_col + lanes, stage, p.dq, part, p.vec_grad, good, one_q ? 0 : l, n, h, p.N, p.H, p.D, p.scale / factor);
            }
        } else if (half == 0) {
            put_zeros<T>(p.dq, part, p.vec_grad, good, one_q ? 0 : l, n, h, p.N, p.H, p.D);
        }
    } else if (warp == S::LOAD_WARP) {
        // ------------------------------------------------------------------ copies
        if (tc::elect_one() && n_items > 0) {
            mbar_expect_tx(held_full, 2 * S::TILE);
            load_tile<DP>(held_q, &maps.q, n0, h, p.q.sl == 0 ? 0 : l, held_full);
            load_tile<DP>(held_d, &maps.dout, n0, h, p.dout.sl == 0 ? 0 : l, held_full);
            for (int i = 0; i < n_items; ++i) {
                const int ks = i % KS, vs = i % VS;
                if (i >= KS) wait(k_empty(ks), (i / KS - 1) & 1);
                mbar_expect_tx(k_full(ks), S::TILE);
                load_tile<DP>(ring_k + ks * S::TILE, &maps.k, (first + i) * TC_ROWS, hk, p.k.sl == 0 ? 0 : kl, k_full(ks));
                if (i >= VS) wait(v_empty(vs), (i / VS - 1) & 1);
                mbar_expect_tx(v_full(vs), S::TILE);
                load_tile<DP>(ring_v + vs * S::TILE, &maps.v, (first + i) * TC_ROWS, hk, p.v.sl == 0 ? 0 : kl, v_full(vs));
            }
            wait.drain(held_full, 0);
            for (int i = max(0, n_items - KS); i < n_items; ++i) wait.drain(k_full(i % KS), (i / KS) & 1);
            for (int i = max(0, n_items - VS); i < n_items; ++i) wait.drain(v_full(i % VS), (i / VS) & 1);
        }
        __syncwarp();
    } else if (warp == S::MMA_WARP && n_items > 0) {
        // ------------------------------------------------------------------ products
        auto scores = [&](int i) {
            wait(k_full(i % KS), (i / KS) & 1);
            tc::fence_after_sync();
            issue_channels<T, DP>(p.D, tmem + (i & 1) * 128, desc_channels(held_q), desc_channels(ring_k + i % KS * S::TILE), s_full(i & 1));
        };
        auto gradients = [&](int i) {
            wait(v_full(i % VS), (i / VS) & 1);
            tc::fence_after_sync();
            issue_channels<T, DP>(p.D, dp_col, desc_channels(held_d), desc_channels(ring_v + i % VS * S::TILE), dp_full);
            issue_commit(v_empty(i % VS));
        };
        wait(held_full, 0);
        scores(0);
        gradients(0);
        if (n_items > 1) scores(1);
        for (int i = 0; i < n_items; ++i) {
            wait(ds_ready, i & 1);
            tc::fence_after_sync();
            issue_rows<T, DP>(p.D, dq_col, dp_col, desc_rows(ring_k + i % KS * S::TILE), i > 0);
            issue_commit(k_empty(i % KS));
            if (i + 1 < n_items) gradients(i + 1);
            if (i + 2 < n_items) scores(i + 2);       // over the scores that ds(i) was the last to need
        }
        issue_commit(done);
        wait.drain(done, 0);
    }
    tc::fence_before_sync();
    __syncthreads();
    tc::fence_after_sync();
    if (warp == S::MMA_WARP) tc::tmem_dealloc(tmem, 512);
    if (threadIdx.x == 0 && s_expired) g_attention_grad_wait_expired = 1;
}

template <typename T, int DP>
__global__ void __launch_bounds__(GradTensorShape<DP>::BLOCK, 1)
attention_grad_tensor_kernel(const __grid_constant__ AttentionGradParams p, const __grid_constant__ GradMaps maps, const int first_blocks,
                             const int keys_first) {
    after_previous_grid();
    const bool first = static_cast<int>(blockIdx.x) < first_blocks;
    const int  block = first ? blockIdx.x : blockIdx.x - first_blocks;
    if (first == (keys_first != 0))
        gradient_of_keys<T, DP>(p, maps, block);
    else
        gradient_of_queries<T, DP>(p, maps, block);
}

template <typename T, int DP>
int launch_grad_tensor(const AttentionGradParams& p, const GradMaps& maps, cudaStream_t st) {
    typedef GradTensorShape<DP> S;
    constexpr int smem = S::at_least_half(S::KEYS_SMEM > S::QUERIES_SMEM ? S::KEYS_SMEM : S::QUERIES_SMEM);
    static_assert(smem <= 227 * 1024, "more shared memory than a block has");
    auto* const kernel = &attention_grad_tensor_kernel<T, DP>;
    if (int rc = cuda_status(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem), "cudaFuncSetAttribute")) return rc;
    const long long kb = ceil_div_ll(p.M, TC_ROWS) * p.kv_slices * p.Hk * p.kv_batch, qb = ceil_div_ll(p.N, TC_ROWS) * p.q_splits * p.H * p.L;
    if (kb + qb > 0x7fffffffLL) return fail(KM_ERR_TOO_LARGE, "attention: more than 2^31 - 1 blocks");
    auto launch = [&](long long first, long long then, bool keys_first) {
        return cuda_status(launch_overlapped(kernel, dim3(static_cast<unsigned>(first + then)), S::BLOCK, smem, st, p, maps, static_cast<int>(first),
                                             static_cast<int>(keys_first)),
                           "attention_grad_tensor_kernel");
    };
    return p.keys_first ? launch(kb, qb, true) : launch(qb, kb, false);
}

}  // namespace
}  // namespace att

int attention_grad_tensor_launch(const AttentionGradParams& p, int type, cudaStream_t st) {
    using namespace att;
    GradMaps maps = {};
    int rc = encode_rows(&maps.q, p.q, p.N, p.H, p.L, p.D, type);
    if (!rc) rc = encode_rows(&maps.dout, p.dout, p.N, p.H, p.L, p.D, type);
    if (!rc) rc = encode_rows(&maps.k, p.k, p.M, p.Hk, p.kv_batch, p.D, type);
    if (!rc) rc = encode_rows(&maps.v, p.v, p.M, p.Hk, p.kv_batch, p.D, type);
    if (rc) return rc;
    if (type == ATT_BF16)
        return p.D <= 64 ? launch_grad_tensor<__nv_bfloat16, 64>(p, maps, st) : launch_grad_tensor<__nv_bfloat16, 128>(p, maps, st);
    return p.D <= 64 ? launch_grad_tensor<__half, 64>(p, maps, st) : launch_grad_tensor<__half, 128>(p, maps, st);
}

int attention_grad_tensor_take_wait_flag() { return att::take_wait_flag(att::g_attention_grad_wait_expired); }

}  // namespace km
