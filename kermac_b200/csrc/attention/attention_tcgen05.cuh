// Pieces that the tensor-core attention kernels share: operand descriptors, 16-bit tcgen05.mma, tensor-memory reads and writes,
// and the shared-memory layout of a tile.
//
// A tile of 128 rows is held as slabs of 64 channels: row r of a slab is 128 bytes, its 16-byte chunk c at position c ^ (r % 8),
// which is what a TMA copy with the 128-byte swizzle writes.  One copy of a tile serves both kinds of product: as a K-major operand
// (contraction over channels) and, through the transpose bit of the instruction, as an MN-major one (contraction over rows).
#pragma once

#include "../km_mbar.cuh"
#include "../km_tcgen05.cuh"
#include "attention_work.cuh"

namespace km {
namespace att {

constexpr int TC_ROWS = 128, TC_SLAB = TC_ROWS * 128;

// Instruction descriptor: fp32 sums (1 in bits [4,6)), both operands float16 (0) or bfloat16 (1) in [7,10) and [10,13), B MN-major
// in bit 16, N / 8 in [17,23), M / 16 in [24,29).
template <typename T>
__device__ __forceinline__ constexpr uint32_t instr_desc(int n, bool b_rows) {
    const uint32_t f = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
    return (1u << 4) | (f << 7) | (f << 10) | (b_rows ? 1u << 16 : 0u) | (static_cast<uint32_t>(n >> 3) << 17) | (8u << 24);
}
// A tile as a K-major operand (contraction over channels).
__device__ __forceinline__ uint64_t desc_channels(uint32_t tile) { return tc::smem_desc_k_major_sw128(tile); }
// A tile as an MN-major operand (contraction over rows): 64-channel blocks TC_SLAB apart (leading offset), groups of eight rows
// 1024 bytes apart (stride offset).
__device__ __forceinline__ uint64_t desc_rows(uint32_t tile) {
    return static_cast<uint64_t>((tile & 0x3FFFFu) >> 4) | (static_cast<uint64_t>(TC_SLAB >> 4) << 16) | (64ull << 32) | (1ull << 46) | (2ull << 61);
}

// D (+)= A B, A and B in shared memory.
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(static_cast<uint32_t>(accumulate))
        : "memory");
}
// The same with A in tensor memory, two of its columns in one of 32 bits.
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool accumulate) {
    tc::mma_bf16_a_tmem(d, a, b, idesc, accumulate);
}

// The products of two tiles, issued by one lane: called by a converged warp.  Descriptors are formed by the whole warp and the guard
// is elect_one() itself, so that they stay in uniform registers.
//
// d (128 x 128) = A B^T over the D channels (those up to the next multiple of 16 are zeros in both).  The full width has code of its
// own: with the test at every instruction train steps of 128 channels took 3 % longer.
template <typename T, int DP>
__device__ __forceinline__ void issue_channels(int D, uint32_t d, uint64_t a, uint64_t b, uint32_t done) {
    if (D > DP - 16) {
        if (tc::elect_one()) {
#pragma unroll
            for (int k = 0; k < DP / 16; ++k) {
                const uint64_t at = (k >> 2) * (TC_SLAB >> 4) + (k & 3) * 2;
                mma_ss(d, a + at, b + at, instr_desc<T>(128, false), k > 0);
            }
            tc::commit(done);
        }
    } else {
        if (tc::elect_one()) {
#pragma unroll
            for (int k = 0; k < DP / 16 - 1; ++k) {
                const uint64_t at = (k >> 2) * (TC_SLAB >> 4) + (k & 3) * 2;
                if (k * 16 < D) mma_ss(d, a + at, b + at, instr_desc<T>(128, false), k > 0);
            }
            tc::commit(done);
        }
    }
    __syncwarp();
}
// d (128 x D, rounded up to 16) (+)= A B over the 128 rows of B; A in tensor memory, 32 columns from `a` on and 32 from a + 64
template <typename T, int DP>
__device__ __forceinline__ void issue_rows(int D, uint32_t d, uint32_t a, uint64_t b, bool accumulate) {
    if (D > DP - 16) {
        if (tc::elect_one()) {
#pragma unroll
            for (int k = 0; k < 8; ++k)
                mma_ts(d, a + (k >> 2) * 64 + (k & 3) * 8, b + k * 128, instr_desc<T>(DP, true), accumulate || k > 0);
        }
    } else {
        const uint32_t idesc = instr_desc<T>((D + 15) & ~15, true);
        if (tc::elect_one()) {
#pragma unroll
            for (int k = 0; k < 8; ++k) mma_ts(d, a + (k >> 2) * 64 + (k & 3) * 8, b + k * 128, idesc, accumulate || k > 0);
        }
    }
    __syncwarp();
}
__device__ __forceinline__ void issue_commit(uint32_t bar) {
    if (tc::elect_one()) tc::commit(bar);
    __syncwarp();
}

// Host: 1 if a wait of the kernel has run out since the last call (the flag is then taken back), 0 if not, -1 if the device did not tell.
inline int take_wait_flag(const int& flag_on_device) {
    int flag = 0;
    if (cudaMemcpyFromSymbol(&flag, flag_on_device, sizeof(flag)) != cudaSuccess) return -1;
    const int zero = 0;
    if (flag && cudaMemcpyToSymbol(flag_on_device, &zero, sizeof(zero)) != cudaSuccess) return -1;
    return flag ? 1 : 0;
}

// One row (lane) of 32 columns.  The values may be used behind wait_loaded() of the same registers.
__device__ __forceinline__ void tmem_load32(uint32_t addr, uint32_t* r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, "
        "%19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
          "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),
          "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
          "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(addr)
        : "memory");
}
__device__ __forceinline__ void tmem_wait_load() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
// Ties 32 registers to the wait before it, so that no use of them moves in front.
__device__ __forceinline__ void tmem_loaded32(uint32_t* r) {
    asm volatile("" : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]),
                 "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]), "+r"(r[17]),
                 "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]),
                 "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31]));
}
__device__ __forceinline__ void tmem_store8(uint32_t addr, const uint32_t* r) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]),
                 "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
                 : "memory");
}
__device__ __forceinline__ void tmem_store32(uint32_t addr, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, "
        "%19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};"
        ::"r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
          "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]),
          "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]),
          "r"(r[30]), "r"(r[31])
        : "memory");
}

// Host: a 16-bit tensor [l][row][head][channel] for copies of boxes of 64 channels; what a box has beyond `rows` or D
// is filled with zeros.  Needs tma_rows_ok().
int encode_rows(CUtensorMap* map, const Heads& t, int rows, int heads, int L, int D, int type, int box_rows = TC_ROWS);
// The keys and values of a forward pass, those that it has.
struct TensorMaps { CUtensorMap k, v, kp, vp; };
int encode_forward(TensorMaps* maps, const AttentionParams& p, int type, int box_rows);
// The queries as the rows of a forward pass: boxes of 64 channels x G heads x 128 / G queries.  Tells for which of the two sets of
// rows (own, prefix) there is such a box: G divides 128, and the queries of a prefix's rows are evenly apart over the whole batch.
struct QueryMaps { CUtensorMap own, prefix; };
enum { QUERIES_OWN = 1, QUERIES_PREFIX = 2 };
int encode_queries(QueryMaps* maps, int* which, const AttentionParams& p, int type);

// One box of a rank-4 tensor of 16-bit values; x is 0 or 64 (a multiple of 128 bytes).  The second form: of a [l][head][row][channel] one.
__device__ __forceinline__ void tma_load_box(uint32_t dst, const CUtensorMap* map, int x, int y, int z, int w, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
        ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(bar)
        : "memory");
}
__device__ __forceinline__ void tma_load_rows(uint32_t dst, const CUtensorMap* map, int x, int row, int head, int l, uint32_t bar) {
    tma_load_box(dst, map, x, row, head, l, bar);
}

// A row of 16-bit channels into a tile by the thread that owns the row; nullptr: zeros.  D is a multiple of 8.
template <int DP>
__device__ __forceinline__ void fill_row(char* tile, int r, const char* row, int D) {
#pragma unroll
    for (int c = 0; c < DP / 8; ++c) {
        uint4 x = make_uint4(0, 0, 0, 0);
        if (row != nullptr && c * 8 < D) x = *reinterpret_cast<const uint4*>(row + c * 16);
        *reinterpret_cast<uint4*>(tile + (c >> 3) * TC_SLAB + r * 128 + ((c & 7) ^ (r & 7)) * 16) = x;
    }
}

// Rows of eight 16-byte chunks that the lanes of a warp hold one each, written to global memory so that neighbouring lanes write
// neighbouring chunks: through 4 KB of shared memory.  `to` is where the lane's row goes (nullptr: nowhere), `many` how many chunks of
// it there are.  (Each lane writing its own row: 2.0 us a block for 128 16-bit channels, 3.9 for 32-bit ones.)
__device__ __forceinline__ void store_rows(char* stage, const uint32_t* x, char* to, int many) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int c = 0; c < 8; ++c)
        *reinterpret_cast<uint4*>(stage + lane * 128 + ((c ^ lane) & 7) * 16) = make_uint4(x[4 * c], x[4 * c + 1], x[4 * c + 2], x[4 * c + 3]);
    __syncwarp();
    const u64 mine = reinterpret_cast<u64>(to);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int   row = i * 4 + (lane >> 3), c = lane & 7;
        char* const at  = reinterpret_cast<char*>(__shfl_sync(0xffffffffu, mine, row));
        const uint4 v   = *reinterpret_cast<const uint4*>(stage + row * 128 + ((c ^ row) & 7) * 16);
        if (at != nullptr && c < many) *reinterpret_cast<uint4*>(at + c * 16) = v;
    }
    __syncwarp();
}
// Columns [0, DP) of 32 rows (a warp's lanes) from tensor memory, times `by`, into rows of 16-bit channels at `to` or of 32-bit ones at
// `part`; one of the two is null for every lane, both where the row is nobody's.
template <typename T, int DP>
__device__ __forceinline__ void store_sums(uint32_t columns, char* stage, char* to, char* part, bool parts, int D, float by) {
#pragma unroll
    for (int j = 0; j < DP; j += 64) {
        uint32_t o[64];
        tmem_load32(columns + j, o);
        tmem_load32(columns + j + 32, o + 32);
        tmem_wait_load();
        tmem_loaded32(o);
        tmem_loaded32(o + 32);
#pragma unroll
        for (int e = 0; e < 64; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * by);
        if (parts) {
            store_rows(stage, o, part ? part + j * 4 : nullptr, (D - j) / 4);
            store_rows(stage, o + 32, part ? part + (j + 32) * 4 : nullptr, (D - j - 32) / 4);
        } else {
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = Type<T>::pair(__uint_as_float(o[2 * e]), __uint_as_float(o[2 * e + 1]));
            store_rows(stage, o, to ? to + j * 2 : nullptr, (D - j) / 8);
        }
    }
}

}  // namespace att
}  // namespace km
