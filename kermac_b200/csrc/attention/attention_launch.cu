// Attention behind the C-ABI: checks of arguments, the plan of a call (which kernel, how many pieces) and its launches.
#include <algorithm>
#include <cmath>

#include "../km_build_tma.cuh"
#include "attention_tcgen05.cuh"

namespace km {
namespace att {
int encode_rows(CUtensorMap* map, const Heads& t, int rows, int heads, int L, int D, int type, int box_rows) {
    // an extent of one may come with any stride; a broadcast batch is one entry
    const long long dense = (D + 7) & ~7;
    const cuuint64_t dims[4]    = {static_cast<cuuint64_t>(D), static_cast<cuuint64_t>(rows), static_cast<cuuint64_t>(heads),
                                   static_cast<cuuint64_t>(t.sl == 0 ? 1 : L)};
    const cuuint64_t strides[3] = {static_cast<cuuint64_t>(rows > 1 ? t.sr : dense) * 2, static_cast<cuuint64_t>(heads > 1 ? t.sh : dense) * 2,
                                   static_cast<cuuint64_t>(dims[3] > 1 ? t.sl : dense) * 2};
    const cuuint32_t box[4] = {64, static_cast<cuuint32_t>(box_rows), 1, 1};
    return encode_tma_16bit(map, t.ptr, type == ATT_BF16, dims, strides, box);
}

int encode_forward(TensorMaps* maps, const AttentionParams& p, int type, int box_rows) {
    int rc = 0;
    if (p.own_tiles > 0 && p.M > 0) {
        rc = encode_rows(&maps->k, p.k, p.M, p.Hk, p.L, p.D, type, box_rows);
        if (!rc) rc = encode_rows(&maps->v, p.v, p.M, p.Hk, p.L, p.D, type, box_rows);
    }
    if (!rc && p.prefix_tiles > 0) {
        rc = encode_rows(&maps->kp, p.kp, p.P, p.Hk, 1, p.D, type, box_rows);
        if (!rc) rc = encode_rows(&maps->vp, p.vp, p.P, p.Hk, 1, p.D, type, box_rows);
    }
    return rc;
}

int encode_queries(QueryMaps* maps, int* which, const AttentionParams& p, int type) {
    *which = 0;
    const long long most = 1LL << 38;
    if (128 % p.G != 0 || p.q.sh >= most || p.q.sr >= most || p.q.sl >= most || (p.H > 1 && p.q.sh == 0)) return 0;
    const cuuint32_t box[4] = {64, static_cast<cuuint32_t>(p.G), static_cast<cuuint32_t>(128 / p.G), 1};
    const long long  dense = (p.D + 7) & ~7;
    auto encode = [&](CUtensorMap* map, long long rows, long long sr, int batch, long long sl) {
        const cuuint64_t dims[4]    = {static_cast<cuuint64_t>(p.D), static_cast<cuuint64_t>(p.H), static_cast<cuuint64_t>(rows),
                                       static_cast<cuuint64_t>(batch)};
        const cuuint64_t strides[3] = {static_cast<cuuint64_t>(p.H > 1 ? p.q.sh : dense) * 2, static_cast<cuuint64_t>(rows > 1 ? sr : dense) * 2,
                                       static_cast<cuuint64_t>(batch > 1 ? sl : dense) * 2};
        return encode_tma_16bit(map, p.q.ptr, type == ATT_BF16, dims, strides, box);
    };
    if (p.own_tiles > 0 && (p.N == 1 || p.q.sr > 0)) {
        if (int rc = encode(&maps->own, p.N, p.q.sr, p.q.sl == 0 ? 1 : p.L, p.q.sl)) return rc;
        *which |= QUERIES_OWN;
    }
    // one distance between all the queries of the batch
    const bool even = p.L == 1 || p.N == 1 || p.q.sl == p.N * p.q.sr;
    const long long apart = p.N == 1 ? p.q.sl : p.q.sr;
    if (p.prefix_tiles > 0 && even && (static_cast<long long>(p.L) * p.N == 1 || apart > 0)) {
        if (int rc = encode(&maps->prefix, static_cast<long long>(p.L) * p.N, apart, 1, 0)) return rc;
        *which |= QUERIES_PREFIX;
    }
    return 0;
}
}  // namespace att

int count_blocks(const AttentionParams& p, unsigned* blocks) {
    const long long n = static_cast<long long>(p.Hk) * p.prefix_tiles * p.prefix_splits +
                        static_cast<long long>(p.L) * p.Hk * p.own_tiles * p.own_splits;
    if (n > 0x7fffffffLL) return fail(KM_ERR_TOO_LARGE, "attention: more than 2^31 - 1 blocks");
    *blocks = static_cast<unsigned>(n);
    return 0;
}

namespace {

enum Kind { CROSS = 0, PREFIX = 1, GRAD = 2 };

constexpr long long MAX_STRIDE = 1LL << 40;
constexpr float     LOG2E = 1.4426950408889634f;

int check_heads(const char* name, const KmHeads& t, long long rows, long long heads, long long batch) {
    if (batch * rows * heads > 0 && !t.ptr) return fail(KM_ERR_NULL_POINTER, "%s must not be NULL", name);
    if (t.stride_l < 0 || t.stride_row < 0 || t.stride_head < 0)
        return fail(KM_ERR_BAD_STRIDE, "%s must not have a negative stride", name);
    if (t.stride_l >= MAX_STRIDE || t.stride_row >= MAX_STRIDE || t.stride_head >= MAX_STRIDE)
        return fail(KM_ERR_BAD_STRIDE, "%s has a stride of 2^40 elements or more", name);
    return 0;
}
// A written tensor must not hold two elements in one place: sorted by stride, each dimension spans the ones before it.
int check_written(const char* name, const KmHeads& t, long long rows, long long heads, long long batch, int d) {
    if (int rc = check_heads(name, t, rows, heads, batch)) return rc;
    std::pair<long long, long long> dims[3] = {{t.stride_l, batch}, {t.stride_row, rows}, {t.stride_head, heads}};
    std::sort(dims, dims + 3);
    long long span = d;
    for (const auto& dim : dims) {
        if (dim.second <= 1) continue;
        if (dim.first < span) return fail(KM_ERR_BAD_STRIDE, "%s has strides that put two elements in one place", name);
        span = dim.first * (dim.second - 1) + span;
    }
    return 0;
}

int check(const KmAttentionArgs* a, Kind kind) {
    if (!a) return fail(KM_ERR_NULL_POINTER, "args must not be NULL");
    if (a->l < 0 || a->n < 0 || a->m < 0 || a->prefix < 0) return fail(KM_ERR_BAD_SHAPE, "extents must not be negative");
    if (a->heads < 0 || a->key_heads < 1 || a->heads % a->key_heads != 0)
        return fail(KM_ERR_BAD_SHAPE, "heads (%d) must be a multiple of key_heads (%d)", a->heads, a->key_heads);
    if (a->d < 1 || a->d > 256) return fail(KM_ERR_BAD_SHAPE, "the number of channels must be in [1, 256], got %d", a->d);
    if (a->type < ATT_F32 || a->type > ATT_F16) return fail(KM_ERR_BAD_ENUM, "type must be a KM_TYPE_*");
    if (!(a->scale >= 0.0f) || std::isinf(a->scale * LOG2E)) return fail(KM_ERR_BAD_HYPERPARAM, "scale must be finite and not negative (and below 2^127)");
    if (kind != PREFIX && a->prefix != 0) return fail(KM_ERR_BAD_SHAPE, "only prefix_attention has a prefix");
    if (a->m > (1 << 30) || a->prefix > (1 << 30)) return fail(KM_ERR_TOO_LARGE, "more than 2^30 keys");
    const long long rows = static_cast<long long>(a->l) * a->n * a->heads;
    const long long most_rows = (1LL << 31) - 1024;           // row numbers of the last tile stay below 2^31
    if (static_cast<long long>(a->l) * a->n > most_rows || rows > most_rows) return fail(KM_ERR_TOO_LARGE, "batch * queries * heads must be below 2^31");
    if ((a->k.stride_l == 0) != (a->v.stride_l == 0) && a->l > 1 && a->m > 0)
        return fail(KM_ERR_BAD_STRIDE, "k and v must both be broadcast over the batch, or neither");
    const bool any = rows > 0;
    int rc = check_heads("q", a->q, a->n, a->heads, a->l);
    if (!rc && any) rc = check_heads("k", a->k, a->m, a->key_heads, a->l);
    if (!rc && any) rc = check_heads("v", a->v, a->m, a->key_heads, a->l);
    if (!rc && any && kind == PREFIX) rc = check_heads("k_prefix", a->k_prefix, a->prefix, a->key_heads, 1);
    if (!rc && any && kind == PREFIX) rc = check_heads("v_prefix", a->v_prefix, a->prefix, a->key_heads, 1);
    if (rc) return rc;
    if (a->lengths && a->lengths_stride < 0) return fail(KM_ERR_BAD_STRIDE, "lengths must not have a negative stride");
    if (a->lse && (a->lse_stride_l < 0 || a->lse_stride_head < 0)) return fail(KM_ERR_BAD_STRIDE, "lse must not have a negative stride");
    if (kind != GRAD) {
        if (a->lse && any) {
            const KmHeads lse = {a->lse, a->lse_stride_l, a->lse_stride_head, 1};       // [l][head][n]
            if (int bad = check_written("lse", lse, a->heads, a->n, a->l, 1)) return bad;
        }
        return check_written("out", a->out, a->n, a->heads, a->l, a->d);
    }
    if (any && !a->lse) return fail(KM_ERR_NULL_POINTER, "lse must not be NULL");
    if ((a->q_batch != a->l && a->q_batch != 1) || (a->kv_batch != a->l && a->kv_batch != 1))
        return fail(KM_ERR_BAD_SHAPE, "q_batch and kv_batch must be 1 or l");
    if (a->l > 1 && ((a->q_batch == 1 && a->q.stride_l != 0) || (a->kv_batch == 1 && a->k.stride_l != 0)))
        return fail(KM_ERR_BAD_STRIDE, "a batch of 1 must have a batch stride of 0");
    rc = check_heads("out", a->out, a->n, a->heads, a->l);
    if (!rc) rc = check_heads("grad_out", a->grad_out, a->n, a->heads, a->l);
    if (!rc) rc = check_written("grad_q", a->grad_q, a->n, a->heads, a->q_batch, a->d);
    if (!rc) rc = check_written("grad_k", a->grad_k, a->m, a->key_heads, a->kv_batch, a->d);
    if (!rc) rc = check_written("grad_v", a->grad_v, a->m, a->key_heads, a->kv_batch, a->d);
    return rc;
}

Heads heads(const KmHeads& t) { return {static_cast<char*>(t.ptr), t.stride_l, t.stride_row, t.stride_head}; }

// Every row of every head starts on a 16-byte boundary and is a whole number of 16-byte units.
bool rows_aligned(const KmHeads& t, int type, int d) {
    const long long unit = 16 / type_bytes(type);
    return aligned16(t.ptr) && t.stride_l % unit == 0 && t.stride_row % unit == 0 && t.stride_head % unit == 0 && d % unit == 0;
}

// What a TMA copy of 64 x 128 boxes needs beyond that: no stride of zero but the batch's, none beyond its 40 bits.
bool tma_rows_ok(const KmHeads& t, int rows, int n_heads, int type, int d) {
    const long long most = 1LL << 38;
    return type != ATT_F32 && rows_aligned(t, type, d) && (rows <= 1 || (t.stride_row > 0 && t.stride_row < most)) &&
           (n_heads <= 1 || (t.stride_head > 0 && t.stride_head < most)) && t.stride_l < most;
}

// The kernels of the forward pass.  TENSOR: 256 rows on tcgen05.  FEW: 8 or 16 rows whose keys a few warps share out, fed by TMA.
// TENSOR32: 256 rows of float32 on tcgen05, from copies in three bf16 planes.  For what these do not take: SCALAR_FEW, 16 rows in the manner of FEW, and ROWS, 64 rows that share key tiles.
enum Kernel { TENSOR, FEW, TENSOR32, SCALAR_FEW, ROWS };
struct Form {
    Kernel kernel;
    int    rows;            // of a block
    int    per_sm, least;   // blocks that an SM holds; keys below which a piece does not pay
    bool operator!=(const Form& f) const { return kernel != f.kernel || rows != f.rows; }
    const char* name() const { return kernel == TENSOR ? "tensor" : kernel == FEW ? "few" : kernel == TENSOR32 ? "tensor32" : kernel == ROWS ? "rows" : "scalar few"; }
};

struct Plan {
    Form own, prefix;
    AttentionParams p;
    long long parts;         // bytes of partial sums, and of the planes behind them
    long long planes;
    long long bytes() const { return parts + planes; }
};

// keys: of both sets.
Form choose_form(long long rows, bool tma_ok, int type, int d, long long keys, bool planes) {
    // 16 rows: two tiles of FEW for 17 to 32 rows against one block of TENSOR, us: 64 channels 85 and 114 (64 x 2000 keys, 8 key heads), 28 and 35
    // (32 x 1000); 128 channels 131 and 132, 45 and 41, 88 and 64 (16 x 4000, 32 rows).  Pieces of 256 keys, two tiles, against 128 and 512: 100 rows
    // of 2000 keys, 8 heads, 15.6, 15.3 and 19.5; 100 of 500, 11.0, 11.7 and 11.0; 256 of 4000, 4 heads, 19.0, 17.7 and 21.2.
    if (tma_ok && rows > 16) return {TENSOR, ATT_TENSOR_ROWS, 1, 256};
    // Pieces of 128 keys, a tile for each warp, against 64 and 256: a token of 8 heads of 128 and 1000 keys 8.4, 10.2 and 9.3; of 500 7.1, 7.8 and 8.6; of 8 heads
    // of 64 and 1000 keys 7.6, 9.6 and 6.9; 2 tokens of 2000 keys, 2 key heads, 11.5, 9.5 and 10.8.
    if (tma_ok) return {FEW, rows <= 8 ? 8 : 16, 0, 128};             // plan_forward() knows how many blocks an SM holds
    // These two take long for a key, and their pieces are short: 64 keys against 256, a token of 500 (8 heads of 128) in float32 42.0 -> 17.5 us;
    // 32 against 256, 2 x 300 x 500 (4 heads of 128) 120 -> 42, and against 64, 300 x 300 (4 heads of 256) 54 -> 42.  As many blocks as the shared
    // memory of an SM holds; with twice as many 2 x 2000 x 200 (4 heads of 128) 71.8 -> 100.8.
    if (rows <= ATT_FEW_ROWS) return {SCALAR_FEW, ATT_FEW_ROWS, d <= 64 ? 2 : 1, 64};
    // Above 32 keys: see attention_tensor32.cu.  Pieces of 192 keys: a tile of 128 is 5 us, the join 4 to 6 (2 x 300 x 500, 4 heads: one piece
    // 27.5 us, two 21.2; but 2 x 2000 x 260, which 128 would split, 23.7 and 28.5).
    if (planes && keys > 32) return {TENSOR32, ATT_TENSOR_ROWS, 1, 192};
    // (float32 of up to 64 channels, which has more than 32 keys here where planes cannot be had: 64; 1024 queries of 64 keys, 8 heads, 12.8, with 32 16.6)
    if (type == ATT_F32 && d <= 64) return {ROWS, ATT_TILE_ROWS, 4, 64};
    return {ROWS, ATT_TILE_ROWS, type != ATT_F32 || d <= 128 ? 2 : 1, 32};
}

// How many pieces the keys of `blocks` blocks are split into: as many as the SMs hold at once, no piece shorter than `least` keys.
int pieces(long long blocks, long long keys, int per_sm, int least) {
    if (blocks <= 0 || keys <= 0) return 1;
    const long long fit = static_cast<long long>(sm_count()) * per_sm / blocks;
    return static_cast<int>(std::max(1LL, std::min({fit, keys / least, 256LL})));
}

// `split`: keys may be divided; `planes`: copies of the inputs may be made.
Plan plan_forward(const KmAttentionArgs& a, Kind kind, bool split, bool planes) {
    Plan plan = {};
    AttentionParams& p = plan.p;
    p.L = a.l, p.N = a.n, p.H = a.heads, p.Hk = a.key_heads, p.G = a.heads / a.key_heads, p.D = a.d, p.M = a.m, p.P = a.prefix;
    p.q = heads(a.q), p.k = heads(a.k), p.v = heads(a.v), p.out = heads(a.out), p.kp = heads(a.k_prefix), p.vp = heads(a.v_prefix);
    p.lengths = a.lengths, p.lengths_stride = a.lengths_stride;
    p.lse = a.lse, p.lse_sl = a.lse_stride_l, p.lse_sh = a.lse_stride_head;
    // a scale of 0 becomes 2^-149: the -inf of a masked score stays -inf, and no finite score, below 2^128, moves a weight by more than 2^-21
    p.scale_log2 = std::max(a.scale * LOG2E, 0x1p-149f);
    p.causal = kind == PREFIX;
    // Keys that a whole batch shares are a prefix without own keys.
    if (kind == CROSS && a.l > 1 && a.k.stride_l == 0 && !a.lengths && a.m > 0) {
        p.P = a.m, p.M = 0, p.kp = p.k, p.vp = p.v;
    }
    p.vec = rows_aligned(a.q, a.type, a.d) && (p.M == 0 || (rows_aligned(a.k, a.type, a.d) && rows_aligned(a.v, a.type, a.d)));
    if (p.P > 0) {
        const KmHeads &k = kind == PREFIX ? a.k_prefix : a.k, &v = kind == PREFIX ? a.v_prefix : a.v;
        p.vec = p.vec && rows_aligned(k, a.type, a.d) && rows_aligned(v, a.type, a.d);
    }
    const bool narrow = a.type != ATT_F32 && a.d <= 128 && p.vec;
    const bool own_ok = narrow && tma_rows_ok(a.k, a.m, a.key_heads, a.type, a.d) && tma_rows_ok(a.v, a.m, a.key_heads, a.type, a.d);
    const bool prefix_ok = kind == PREFIX ? narrow && tma_rows_ok(a.k_prefix, a.prefix, a.key_heads, a.type, a.d) &&
                                                tma_rows_ok(a.v_prefix, a.prefix, a.key_heads, a.type, a.d)
                                          : own_ok;
    p.vec_out = rows_aligned(a.out, a.type, a.d);
    const long long own_rows = static_cast<long long>(p.N) * p.G, prefix_rows = own_rows * p.L;
    const long long keys = static_cast<long long>(p.M) + p.P;
    plan.own    = choose_form(own_rows, own_ok, a.type, p.D, keys, planes);
    plan.prefix = choose_form(prefix_rows, prefix_ok, a.type, p.D, keys, planes);
    // A short prefix goes along with few own rows: its keys are read again, from L2, for every 8 or 16 rows, which costs less than a launch
    // of its own up to some 8 MB (72 sequences with 64 keys before 40 own ones, 2 key heads of 128: 19.2 -> 11.9 us; 1024 keys, 24 MB: 23.4
    // and 22.2; 4096: 23.6 and 39.0).
    const double again = plan.own.kernel == FEW ? static_cast<double>(ceil_div_ll(prefix_rows, plan.own.rows)) * p.Hk * p.P * p.D * 4 : 0.0;
    if (p.M > 0 && p.P > 0 && plan.own.kernel == FEW && plan.prefix.kernel == TENSOR && again <= 8e6) plan.prefix = plan.own;
    // one launch for both sets where the same kernel takes them
    if (p.M > 0 && p.P > 0 && plan.own.kernel == FEW && plan.prefix.kernel == FEW)
        plan.own.rows = plan.prefix.rows = std::max(plan.own.rows, plan.prefix.rows);
    // the tiles of the launch, which may have both sets, and so the blocks that an SM holds
    const int few_tile   = attention_few_tile(p.D, plan.own.kernel == FEW ? p.M : 0, plan.prefix.kernel == FEW ? p.P : 0);
    const int few_per_sm = p.D <= 64 || few_tile == 16 ? 2 : 1;
    for (Form* form : {&plan.own, &plan.prefix})
        if (form->kernel == FEW) form->per_sm = few_per_sm;
    if (p.M > 0 || p.P == 0) {
        p.own_tiles  = static_cast<int>(ceil_div_ll(own_rows, plan.own.rows));
        p.own_splits = split ? pieces(static_cast<long long>(p.own_tiles) * p.L * p.Hk, p.M, plan.own.per_sm, plan.own.least) : 1;
    }
    if (p.P > 0) {
        p.prefix_tiles  = static_cast<int>(ceil_div_ll(prefix_rows, plan.prefix.rows));
        p.prefix_splits = split ? pieces(static_cast<long long>(p.prefix_tiles) * p.Hk, p.P, plan.prefix.per_sm, plan.prefix.least) : 1;
    }
    p.parts = p.own_splits + p.prefix_splits, p.cluster = 1;
    if (p.parts > 1 && p.parts <= 8 && (p.own_splits == 0 || p.prefix_splits == 0) && (p.own_splits ? plan.own : plan.prefix).kernel == FEW)
        p.cluster = p.parts, p.parts = 1;              // 8 blocks: the largest cluster that every GPU of this kind takes
    auto round16 = [](long long n) { return (n + 15) & ~15LL; };
    if (p.parts > 1) plan.parts = round16(static_cast<long long>(p.parts) * p.L * p.N * p.H * (p.D + 2) * 4);
    if ((p.own_splits > 0 && plan.own.kernel == TENSOR32) || (p.prefix_splits > 0 && plan.prefix.kernel == TENSOR32))
        plan.planes = round16(attention_planes_bytes(p));
    return plan;
}

bool empty(const KmAttentionArgs& a) { return a.l == 0 || a.n == 0 || a.heads == 0; }

// The most scratch that a call asks for beyond the two parts of a row that both sets of keys need: partial sums, and planes of float32 inputs.
constexpr long long MOST_SCRATCH = 512LL << 20, MOST_PLANES = 1LL << 30;

// The plan that a scratch of `most` bytes allows: first without planes, then with a single piece for each set of keys, whatever these two take.
Plan plan_within(const KmAttentionArgs& a, Kind kind, long long most) {
    Plan plan = {};
    const bool one_set = a.l > 1 && a.k.stride_l == 0 && a.lengths;      // see attention_tensor32_launch
    if (a.type == ATT_F32 && a.d <= ATT_TENSOR32_CHANNELS && !one_set) {
        plan = plan_forward(a, kind, true, true);
        if (plan.parts > MOST_SCRATCH) plan = plan_forward(a, kind, false, true);
        if (plan.planes <= MOST_PLANES && plan.bytes() <= most) return plan;
    }
    plan = plan_forward(a, kind, true, false);
    if (plan.parts > std::min(most, MOST_SCRATCH)) plan = plan_forward(a, kind, false, false);
    return plan;
}

int64_t forward_scratch(const KmAttentionArgs* a, Kind kind) {
    if (check(a, kind) || empty(*a)) return 0;
    return plan_within(*a, kind, MOST_SCRATCH + MOST_PLANES).bytes();
}

int forward(const KmAttentionArgs* a, Kind kind, void* stream) {
    int rc = check(a, kind);
    if (rc) return rc;
    if (empty(*a)) return 0;
    rc = require_sm100();
    if (rc) return rc;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    Plan plan = plan_within(*a, kind, a->scratch && aligned16(a->scratch) ? a->scratch_bytes : 0);
    if (plan.bytes() > 0) {
        if (!a->scratch || a->scratch_bytes < plan.bytes() || !aligned16(a->scratch))
            return fail(KM_ERR_NULL_POINTER, "attention: %lld bytes of 16-byte aligned scratch are needed", plan.bytes());
        plan.p.part_o   = static_cast<float*>(a->scratch);
        plan.p.part_top = plan.p.part_o + static_cast<long long>(plan.p.parts) * plan.p.L * plan.p.N * plan.p.H * plan.p.D;
    }
    auto launch = [&](const AttentionParams& p, const Form& form) {
        if (form.kernel == TENSOR) return attention_tensor_launch(p, a->type, st);
        if (form.kernel == TENSOR32) return attention_tensor32_launch(p, static_cast<char*>(a->scratch) + plan.parts, st);
        if (form.kernel == FEW) return attention_few_launch(p, a->type, form.rows, st);
        return attention_rows_launch(p, a->type, form.kernel == SCALAR_FEW, st);
    };
    const bool own = plan.p.own_splits > 0, prefix = plan.p.prefix_splits > 0;
    if (own && prefix && plan.own != plan.prefix) {
        AttentionParams p = plan.p;
        p.own_tiles = 0;                                   // the blocks of the prefix alone
        rc = launch(p, plan.prefix);
        p = plan.p, p.prefix_tiles = 0;
        if (!rc) rc = launch(p, plan.own);
    } else {
        rc = launch(plan.p, own ? plan.own : plan.prefix);
    }
    if (!rc && plan.p.parts > 1) rc = attention_join_launch(plan.p, a->type, st);
    return rc;
}

struct GradPlan {
    AttentionGradParams p;
    bool tensor;
    long long delta, peaks, v_peaks, dq, dkv;     // floats of scratch, each a multiple of 4
    long long bytes() const { return 4 * (delta + peaks + v_peaks + dq + 2 * dkv); }
};
long long round4(long long n) { return (n + 3) & ~3LL; }

GradPlan plan_grad(const KmAttentionArgs& a) {
    GradPlan plan = {};
    AttentionGradParams& p = plan.p;
    p.L = a.l, p.N = a.n, p.H = a.heads, p.Hk = a.key_heads, p.G = a.heads / a.key_heads, p.D = a.d, p.M = a.m;
    p.q = heads(a.q), p.k = heads(a.k), p.v = heads(a.v), p.out = heads(a.out), p.dout = heads(a.grad_out);
    p.dq = heads(a.grad_q), p.dk = heads(a.grad_k), p.dv = heads(a.grad_v);
    p.lengths = a.lengths, p.lengths_stride = a.lengths_stride;
    p.lse = a.lse, p.lse_sl = a.lse_stride_l, p.lse_sh = a.lse_stride_head;
    p.scale = a.scale, p.scale_log2 = a.scale * LOG2E;
    p.vec = rows_aligned(a.q, a.type, a.d) && rows_aligned(a.k, a.type, a.d) && rows_aligned(a.v, a.type, a.d) &&
            rows_aligned(a.grad_out, a.type, a.d);
    p.vec_out  = rows_aligned(a.out, a.type, a.d) && rows_aligned(a.grad_out, a.type, a.d);
    p.vec_grad = rows_aligned(a.grad_q, a.type, a.d) && rows_aligned(a.grad_k, a.type, a.d) && rows_aligned(a.grad_v, a.type, a.d);
    plan.tensor = a.d <= 128 && tma_rows_ok(a.q, a.n, a.heads, a.type, a.d) && tma_rows_ok(a.grad_out, a.n, a.heads, a.type, a.d) &&
                  tma_rows_ok(a.k, a.m, a.key_heads, a.type, a.d) && tma_rows_ok(a.v, a.m, a.key_heads, a.type, a.d);
    p.own_delta = a.type != ATT_F32 && a.m <= (plan.tensor ? ATT_GRAD_TENSOR_ROWS : ATT_GRAD_ROWS);
    p.kv_batch = a.kv_batch;
    const long long key_sums = static_cast<long long>(a.kv_batch == 1 ? a.l : 1) * p.G;       // heads and entries whose queries a key meets
    if (plan.tensor) {
        // Both sums are split to fill the SMs, in pieces of at least four tiles of 128, and so that no block runs on for long when all the others
        // have ended (us: 1.9 and 1.4 a tile, 5 to start and end; a split that is not there anyway costs a launch that adds up, so it has to
        // save some 25).  Training steps: 13 queries of 4 x 4064 keys (one head of 112) 83 -> 52 us, 9 of 4396 (32 heads of 40) 92 -> 72; but
        // split to 12 us, one of 15 queries of 1244 keys (40 heads), whose blocks then start in two rounds, 43 -> 52.
        const long long key_tiles = ceil_div_ll(a.m, ATT_GRAD_TENSOR_ROWS), query_tiles = ceil_div_ll(a.n, ATT_GRAD_TENSOR_ROWS);
        const long long key_blocks = key_tiles * a.key_heads * a.kv_batch, query_blocks = query_tiles * a.heads * a.l, sms = sm_count();
        const double    of_keys = 1.9 * key_sums * query_tiles, of_queries = 1.4 * key_tiles;
        const double    busy = (key_blocks * (of_keys + 5.0) + query_blocks * (of_queries + 5.0)) / sms, target = std::max(1.5 * busy, 25.0);
        auto split = [&](long long blocks, long long others, long long tiles, double time) {
            if (blocks <= 0) return 1;                       // nothing to sum
            const long long fill = std::min((sms - others) / blocks, tiles / 4), even = static_cast<long long>(std::ceil(time / target));
            return static_cast<int>(std::min(std::max({1LL, fill, even}), 64LL));
        };
        p.kv_slices = split(key_blocks, query_blocks, key_sums * query_tiles, of_keys);
        p.q_splits  = split(query_blocks, key_blocks * p.kv_slices, key_tiles, of_queries);
        p.keys_first = of_keys / p.kv_slices >= of_queries / p.q_splits;
    } else {
        // pieces of both sums where their tiles alone do not fill the SMs (of 64 against 128: 2 x 2000 x 40, 4 heads, 56 -> 50 us)
        p.kv_slices = pieces(ceil_div_ll(a.m, ATT_GRAD_ROWS) * a.key_heads * a.kv_batch, key_sums * a.n, 2, 64);
        p.q_splits  = pieces(ceil_div_ll(a.n, ATT_GRAD_ROWS) * a.heads * a.l, a.m, 2, 64);
    }
    if (static_cast<long long>(p.q_splits) * a.l * a.n * a.heads * a.d > (MOST_SCRATCH >> 3)) p.q_splits = 1;
    if (static_cast<long long>(p.kv_slices) * a.kv_batch * a.m * a.key_heads * a.d > (MOST_SCRATCH >> 3)) p.kv_slices = 1;
    p.q_slices = (a.q_batch == 1 && a.l > 1 ? a.l : 1) * p.q_splits;
    plan.delta = round4(static_cast<long long>(a.l) * a.heads * a.n);
    if (a.type == ATT_F16) {
        p.peak_count = static_cast<int>(ceil_div_ll(a.n, ATT_PEAK_ROWS));
        plan.peaks   = round4(static_cast<long long>(a.l) * a.heads * p.peak_count);
        p.v_peak_count = static_cast<int>(ceil_div_ll(a.m, ATT_PEAK_ROWS));
        plan.v_peaks   = round4(static_cast<long long>(a.kv_batch) * a.key_heads * p.v_peak_count);
    }
    if (p.q_slices > 1) plan.dq = round4(static_cast<long long>(p.q_slices) * a.q_batch * a.n * a.heads * a.d);
    if (p.kv_slices > 1) plan.dkv = round4(static_cast<long long>(p.kv_slices) * a.kv_batch * a.m * a.key_heads * a.d);
    return plan;
}

int gradient(const KmAttentionArgs* a, void* stream) {
    int rc = check(a, GRAD);
    if (rc) return rc;
    const bool no_queries = a->q_batch == 0 || a->n == 0 || a->heads == 0, no_keys = a->kv_batch == 0 || a->m == 0;
    if (no_queries && no_keys) return 0;                   // no gradient has a row
    rc = require_sm100();
    if (rc) return rc;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    GradPlan plan = plan_grad(*a);
    AttentionGradParams& p = plan.p;
    if (empty(*a) || a->m == 0) {
        // zeros: no pair of query and key reaches them
        SliceSums none = {};
        none.add(nullptr, 0, p.dq, a->q_batch, p.N, p.H, p.D);
        none.add(nullptr, 0, p.dk, p.kv_batch, p.M, p.Hk, p.D);
        none.add(nullptr, 0, p.dv, p.kv_batch, p.M, p.Hk, p.D);
        return attention_reduce_launch(none, a->type, p.vec_grad, st);
    }
    if (!a->scratch || a->scratch_bytes < plan.bytes() || !aligned16(a->scratch))
        return fail(KM_ERR_NULL_POINTER, "attention gradient: %lld bytes of 16-byte aligned scratch are needed", plan.bytes());
    float* at = static_cast<float*>(a->scratch);
    p.delta = at, at += plan.delta;
    if (plan.peaks) {
        p.peaks = at, at += plan.peaks;
        p.v_peaks = at, at += plan.v_peaks;
    }
    if (plan.dq) p.dq_part = at, at += plan.dq;
    if (plan.dkv) p.dk_part = at, p.dv_part = at + plan.dkv;
    if (!p.own_delta || p.peaks) rc = attention_delta_launch(p, a->type, st);
    if (!rc) rc = plan.tensor ? attention_grad_tensor_launch(p, a->type, st) : attention_grad_rows_launch(p, a->type, st);
    SliceSums sums = {};
    if (p.q_slices > 1) sums.add(p.dq_part, p.q_slices, p.dq, a->q_batch, p.N, p.H, p.D);
    if (p.kv_slices > 1) {
        sums.add(p.dk_part, p.kv_slices, p.dk, p.kv_batch, p.M, p.Hk, p.D);
        sums.add(p.dv_part, p.kv_slices, p.dv, p.kv_batch, p.M, p.Hk, p.D);
    }
    return rc ? rc : attention_reduce_launch(sums, a->type, p.vec_grad, st);
}

}  // namespace
}  // namespace km

extern "C" {

int kermac_b200_cross_attention(const KmAttentionArgs* args, void* stream) { return km::forward(args, km::CROSS, stream); }
int kermac_b200_prefix_attention(const KmAttentionArgs* args, void* stream) { return km::forward(args, km::PREFIX, stream); }
int kermac_b200_cross_attention_grad(const KmAttentionArgs* args, void* stream) { return km::gradient(args, stream); }
int64_t kermac_b200_cross_attention_scratch_bytes(const KmAttentionArgs* args) { return km::forward_scratch(args, km::CROSS); }
int64_t kermac_b200_prefix_attention_scratch_bytes(const KmAttentionArgs* args) { return km::forward_scratch(args, km::PREFIX); }
int64_t kermac_b200_cross_attention_grad_scratch_bytes(const KmAttentionArgs* args) {
    if (km::check(args, km::GRAD) || km::empty(*args) || args->m == 0) return 0;
    return km::plan_grad(*args).bytes();
}

int kermac_b200_describe_attention(const KmAttentionArgs* args, int32_t kind, char* buf, int32_t buf_len) {
    using namespace km;
    if (kind < CROSS || kind > GRAD) return fail(KM_ERR_BAD_ENUM, "kind must be 0 (cross), 1 (prefix) or 2 (gradient)");
    if (int rc = check(args, static_cast<Kind>(kind))) return rc;
    if (!buf || buf_len <= 0) return fail(KM_ERR_NULL_POINTER, "buf must not be NULL");
    if (kind == GRAD) {
        const GradPlan plan = plan_grad(*args);
        snprintf(buf, buf_len, "grad=%s q_slices=%d kv_slices=%d scratch=%lld", plan.tensor ? "tensor" : "rows", plan.p.q_slices, plan.p.kv_slices, plan.bytes());
    } else {
        const Plan plan = plan_within(*args, static_cast<Kind>(kind), MOST_SCRATCH + MOST_PLANES);
        snprintf(buf, buf_len, "own=%s rows=%d tiles=%d splits=%d prefix=%s rows=%d tiles=%d splits=%d scratch=%lld", plan.own.name(),
                 plan.own.rows, plan.p.own_tiles, plan.p.own_splits, plan.prefix.name(), plan.prefix.rows, plan.p.prefix_tiles, plan.p.prefix_splits,
                 plan.bytes());
    }
    return 0;
}

}  // extern "C"
