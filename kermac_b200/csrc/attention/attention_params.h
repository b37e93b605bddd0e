// Parameter blocks and launchers of the attention kernels, shared by their translation units.
#pragma once

#include "../../../include/kermac_b200_attention.h"
#include "../km_host.h"

namespace km {

// One argument of heads [l][row][head][channel], channels contiguous; strides in elements, stride_l 0 broadcasts.
struct Heads {
    char*     ptr;
    long long sl, sr, sh;
};

// Forward pass.  For one batch entry and key head the G = H / Hk query heads of N queries are N * G rows (row = n * G + g)
// against the entry's own keys; against a shared prefix the rows of all batch entries are one matrix (row =
// (l * N + n) * G + g), so its keys are read once for the whole batch.  Each of the two sets of keys may be split among
// blocks; every piece leaves a normalised sum with its maximum and weight (a "part"), which join_kernel adds up.
struct AttentionParams {
    int L, N, H, Hk, G, D, M, P;
    Heads q, k, v, kp, vp, out;
    const int* lengths; long long lengths_stride;
    float* lse; long long lse_sl, lse_sh;
    float scale_log2;                    // scale * log2(e)
    int   causal;                        // own key j is seen by query n when j <= length - N + n
    int   own_tiles, own_splits;         // row tiles of one (l, key head), pieces of its keys; 0 pieces: no own keys
    int   prefix_tiles, prefix_splits;
    int   parts;                         // pieces of one row: own_splits + prefix_splits; 1: results are written directly
    int   cluster;                       // FEW: blocks of a cluster that share a row's keys and join its pieces themselves; else 1
    float* part_o;                       // [part][l][n][h][D]
    float* part_top;                     // [2][part][l][n][h]: maximum (log2 domain), sum of exp2 of what lies below it
    int   vec;                           // every row of k, v, kp, vp and q can be read 16 bytes at a time
    int   vec_out;                       // rows of out can be written 16 bytes at a time
};

// Backward pass: dq, dk and dv from the forward pass's output and lse.
struct AttentionGradParams {
    int L, N, H, Hk, G, D, M;
    Heads q, k, v, out, dout;
    const int* lengths; long long lengths_stride;
    const float* lse; long long lse_sl, lse_sh;
    float scale, scale_log2;
    float* delta;                        // [l][h][n]: sum over channels of dout * out, unused where few 16-bit keys share a query (attention_grad_tensor.cu)
    // float16 only, else null: from these find_factor() (attention_grad.cuh) takes the power of two that keeps the weights' gradients in
    // float16's range.
    float* peaks; int peak_count;        // [l][h][peaks]: the largest |dout| of ATT_PEAK_ROWS queries
    float* v_peaks; int v_peak_count;    // [entry of v][key head][peaks]: the largest |v| of ATT_PEAK_ROWS keys that a query sees
    // Destinations.  slices 1: the gradients in the inputs' type.  More: 32-bit partial sums [slice][...] that
    // grad_reduce adds up, where a broadcast input's gradient is a sum over the batch or the sum is split.
    Heads dq, dk, dv;
    float *dq_part, *dk_part, *dv_part;
    int   q_slices;                      // partial sums of dq: q_splits, times L for a broadcast q
    int   q_splits;                      // pieces of the sum over keys
    int   kv_batch;                      // batch entries of k and v: 1 or L
    int   kv_slices;                     // pieces of the sum over (l of a broadcast k, head of the group, query tile)
    int   keys_first;                    // tensor cores: blocks of dk and dv are the longer ones
    int   own_delta;                     // 16 bits and no more keys than a block holds: every block forms delta itself, nothing does beforehand
    int   vec;                           // rows of q, k, v and dout can be read 16 bytes at a time
    int   vec_out;                       // rows of out and dout can
    int   vec_grad;                      // rows of dq, dk and dv can be written so
};

enum { ATT_F32 = KM_TYPE_FLOAT32, ATT_BF16 = KM_TYPE_BFLOAT16, ATT_F16 = KM_TYPE_FLOAT16 };

// attention_rows.cu (mma.sync): any layout and type.  ATT_TILE_ROWS rows a block; `few`: the form whose warps share ATT_FEW_ROWS.
int  attention_rows_launch(const AttentionParams& p, int type, bool few, cudaStream_t st);
constexpr int ATT_FEW_ROWS = 16, ATT_TILE_ROWS = 64;
int  attention_join_launch(const AttentionParams& p, int type, cudaStream_t st);
// attention_few.cu: 16-bit types, D a multiple of 8 up to 128, rows that TMA can copy; 8 or 16 rows a block.
// Keys of a tile, from the channels and the keys of the launch's two sets (0: none): see attention_few.cu.
inline int attention_few_tile(int d, int keys, int prefix) { return d > 64 && keys <= 2048 && prefix <= 2048 ? 16 : 32; }
int  attention_few_launch(const AttentionParams& p, int type, int rows, cudaStream_t st);
int  attention_few_take_wait_flag();
// Blocks of a forward launch: every (key head, row tile, piece) of both sets of keys.
int  count_blocks(const AttentionParams& p, unsigned* blocks);
// attention_tensor.cu (tcgen05): 16-bit types, D a multiple of 8 up to 128, rows that TMA can copy.
constexpr int ATT_TENSOR_ROWS = 256;
int  attention_tensor_launch(const AttentionParams& p, int type, cudaStream_t st);
int  attention_tensor_take_wait_flag();
// attention_tensor32.cu (tcgen05): float32, up to 64 channels, any layout, with attention_planes_bytes() of scratch (16-byte aligned).
constexpr int ATT_TENSOR32_CHANNELS = 64;
long long attention_planes_bytes(const AttentionParams& p);
int  attention_tensor32_launch(const AttentionParams& p, void* planes, cudaStream_t st);
int  attention_tensor32_take_wait_flag();
// attention_grad_rows.cu
constexpr int ATT_GRAD_ROWS = 64, ATT_PEAK_ROWS = 64;
int  attention_delta_launch(const AttentionGradParams& p, int type, cudaStream_t st);
int  attention_grad_rows_launch(const AttentionGradParams& p, int type, cudaStream_t st);
// attention_grad_tensor.cu (tcgen05): as attention_tensor_launch
constexpr int ATT_GRAD_TENSOR_ROWS = 128;
int  attention_grad_tensor_launch(const AttentionGradParams& p, int type, cudaStream_t st);
int  attention_grad_tensor_take_wait_flag();
// dst[l][row][head][c] = sum over the slices of src[slice][l][row][head][c], in their order; no slices: zeros.  Up to three in a launch.
struct SliceSum {
    const float* src;
    Heads        dst;
    int          slices, L, rows, heads, D;
};
struct SliceSums {
    SliceSum  job[3];
    long long first[4];                  // elements in front of each
    int       count;
    void add(const float* src, int slices, const Heads& dst, int L, int rows, int heads, int D) {
        job[count]       = {src, dst, slices, L, rows, heads, D};
        first[count + 1] = first[count] + static_cast<long long>(L) * rows * heads * D;
        ++count;
    }
};
// vec: rows of every dst can be written 16 bytes at a time.
int attention_reduce_launch(const SliceSums& sums, int type, bool vec, cudaStream_t st);

inline int padded_channels(int d) { return d <= 64 ? 64 : d <= 128 ? 128 : 256; }
inline int type_bytes(int type) { return type == ATT_F32 ? 4 : 2; }

}  // namespace km
