// C ABI of the feed-forward operators in 8-bit floating point (include/accera_mi355x_f8.h): argument checks and the choice of kernel.
#include "../../include/accera_mi355x_f8.h"
#include "f8.h"
#include <cstdio>
#include <utility>

using namespace acc950;

namespace {

int refuse(const char* text) { return set_last_error(ACC950_INVALID_ARGUMENT, text); }

int ended(hipError_t e, const char* what)
{
    if (e == hipSuccess) return ACC950_OK;
    if (e == hipErrorInvalidConfiguration) return set_last_error(ACC950_UNSUPPORTED, "more workgroups than one launch takes");
    char text[160];
    snprintf(text, sizeof text, "%s: %s", what, hipGetErrorString(e));
    return set_last_error(ACC950_HIP_ERROR, text);
}

bool float_type(int64_t t) { return t == ACC950_F32 || t == ACC950_F16 || t == ACC950_BF16; }
bool size_ok(int64_t n) { return n >= 0 && n <= 0x7fffffffll - 1023; } // (so that rounding a size up to a tile stays in 32 bits)
bool misaligned(const void* p, size_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) != 0; }
size_t type_bytes(int64_t t) { return t == ACC950_F32 ? 4 : 2; }
int64_t blocks_of(int64_t n) { return (n + F8_BLOCK - 1) / F8_BLOCK; }

// Whether bytes lie within 32-bit offsets from the first of `rows` rows: these and `more` of the last one (which may be more than the rows are apart).
bool offsets_in_32_bits(int64_t rows, int64_t stride, int64_t more) { return more < 1ll << 32 && stride <= ((1ll << 32) - 1 - more) / rows; }

// Whether the kernels that fetch 16 bytes at a time take the problem: A and B contiguous along K with rows on 16-byte boundaries (the
// rows' own padding is read where K ends inside 16 bytes, never used), C's columns contiguous, and 32-bit offsets from the row a tile
// starts at (it has 256 at most) -- from A's first row where a plan picks the rows (one for every top_k pairs).
bool vectors_can_take(const F8GemmArgs& g)
{
    if (g.K == 0 || g.a_cs != 1 || g.b_rs != 1 || (g.c_cs != 1 && g.N > 1)) return false;
    if ((g.a_rs | g.b_cs | g.b_es) % 16 || misaligned(g.A, 16) || misaligned(g.B, 16)) return false;
    const int64_t a_rows = g.offsets && g.gather ? (g.M + g.top_k - 1) / g.top_k : g.M < 256 ? g.M : 256, b_cols = g.N < 256 ? g.N : 256;
    return offsets_in_32_bits(a_rows, g.a_rs, g.K) && offsets_in_32_bits(a_rows * 4, g.as_rs, 4) && offsets_in_32_bits(b_cols, g.b_cs, g.K) && offsets_in_32_bits(b_cols * 4, g.bs_cs, 4);
}

// Operands that those kernels do not take as they lie can be laid out anew in scratch memory, where nothing but their strides and alignment is in the way.
struct Packed {
    int64_t a_pitch, a_bytes, b_bytes; // (0 bytes: taken as it is)
    bool possible;
};
Packed packed(const F8GemmArgs& g)
{
    Packed p{};
    if (vectors_can_take(g) || g.K == 0) return p;
    p.a_pitch = (g.K + 15) / 16 * 16;
    F8GemmArgs t = g;
    if (g.a_cs != 1 || g.a_rs % 16 || misaligned(g.A, 16)) {
        p.a_bytes = (g.M * p.a_pitch + 255) / 256 * 256;
        t.A = nullptr; t.a_rs = p.a_pitch; t.a_cs = 1;
    }
    if (g.b_rs != 1 || g.b_cs % 16 || misaligned(g.B, 16)) {
        p.b_bytes = (g.N * p.a_pitch + 255) / 256 * 256;
        t.B = nullptr; t.b_cs = p.a_pitch; t.b_rs = 1;
    }
    p.possible = vectors_can_take(t);
    return p;
}

constexpr int FEW_ROWS = 16;

// Rows that stand behind one matrix: all, or those of an expert were they spread evenly.
int64_t rows_of_matrix(const F8GemmArgs& g) { return g.offsets ? (g.M + g.experts - 1) / g.experts : g.M; }

// Kernel of few rows: 128 columns to a workgroup where that makes nearly one for every CU, 16 columns and K over four waves where it does
// not.  (us, 128 / 16 columns: 16x28672x8192 47.9 / 64.1, 48 rows of 64 experts' 2048x1024 13.7 / 27.3; 8x11008x4096 21.6 / 12.0, 8x4096x11008
// 53.9 / 11.8.)
int few_form(const F8GemmArgs& g)
{
    const int64_t matrices = g.offsets ? (g.experts < g.M ? g.experts : g.M) : 1;
    return matrices * ((g.N + 127) / 128) >= 200 ? 1 : 0;
}

struct TileChoice {
    int tile, slices;
    bool few; // neither: the kernel of few rows, 16 columns to a workgroup
};

// Tile and number of K slices by an estimate of the time: rounds of workgroups over the CUs times what a block of K takes in them.
TileChoice choose_tile(const F8GemmArgs& g, bool wide, int64_t workspace_bytes)
{
    // us to a block of K, with one workgroup on a CU and with as many as fit (measured on 4096- to 8192-sized products and on single rounds), to a tile's
    // start and write-back, and how many fit
    struct Rate { double one, full, ends; int fit; };
    static const Rate native[F8_TILES] = {{1.60, 1.60, 10.0, 1}, {0.80, 1.13, 3.8, 2}, {0.40, 0.55, 3.0, 2}, {0.45, 0.95, 3.0, 4}};
    static const Rate widened[F8_TILES] = {{0, 0, 0, 1}, {1.45, 2.0, 3.8, 2}, {0.75, 1.0, 3.0, 2}, {0.75, 1.6, 3.0, 4}};
    const int blocks = (int)blocks_of(g.K);
    const int64_t rows = rows_of_matrix(g), matrices = g.offsets ? (g.experts < g.M ? g.experts : g.M) : 1;
    const int64_t slice_bytes = 4 * (int64_t)g.M * ((g.N + 3) / 4 * 4);
    TileChoice best{F8_TILES - 1, 1, false};
    double best_us = 1e30;
    for (int t = 0; t < F8_TILES; ++t) {
        if (!f8_tile_can_take(g, t, wide)) continue;
        const Rate& r = (wide ? widened : native)[t];
        const double tiles = (double)matrices * ((rows + F8_TILE_SIZE[t] - 1) / F8_TILE_SIZE[t]) * ((g.N + F8_TILE_SIZE[t] - 1) / F8_TILE_SIZE[t]);
        for (int want = 1; want <= 16; ++want) {
            const int per = (blocks + want - 1) / want, slices = (blocks + per - 1) / per;
            if (slices != want) continue;
            if (want > 1 && (g.offsets || per < 4 || want * slice_bytes > workspace_bytes)) break;
            const double n = tiles * want, rounds = n / (kComputeUnits * r.fit);
            // (rounds that all workgroups start together are whole ones; later on they drift apart)
            const double whole = rounds <= 4 ? (double)(int64_t)(rounds + 0.999) : rounds;
            const double us = (n <= kComputeUnits ? r.one : r.full * (rounds < 1 ? 0.5 + 0.5 * rounds : whole)) * per + r.ends * whole +
                              (want > 1 ? 5.0 + want * slice_bytes * 2 / 4.5e6 : 0.0);
            if (us < best_us) { best_us = us; best = TileChoice{t, want, false}; }
        }
    }
    // Small results: 16 x 16 of them to a workgroup, K over its four waves.  A first one on every CU takes what its blocks take one after another, more of
    // them what their fetches do.  (us, so / by tiles: 40x300x5000 6.5 / 11.7, 96x500x3000 5.1 / 10.2, 17x2048x2048 4.1 / 8.4, 24x4096x4096 9.4 / 12.4;
    // 300x1000x700 8.1 / 6.2, 64x4096x1024 9.5 / 5.7, 24x11008x4096 23.2 / 15.9.)
    if (!g.offsets) {
        const double first = 2.4 + 0.11 * blocks, more = (double)((rows + 15) / 16) * ((g.N + 15) / 16) / kComputeUnits - 1.0;
        best.few = first + (more > 0 ? more * (1.3 + 0.075 * blocks) : 0.0) < 0.95 * best_us;
    }
    return best;
}

// Kernel of a product; the problem is not empty.  wide: sums in fp32 throughout (see F8Fragment), what fp32 results get.
int run_gemm(F8GemmArgs g, int64_t variant, bool wide, int64_t k_slices, void* workspace, int64_t workspace_bytes, hipStream_t stream)
{
    const char* what = "block-scaled product";
    if (variant != ACC950_VARIANT_AUTO && (variant < 0 || variant >= ACC950_F8_VARIANT_FEW + 2 * F8_FEW_FORMS ||
                                           (variant >= ACC950_F8_VARIANT_TILE + 2 * F8_TILES && variant < ACC950_F8_VARIANT_FEW)))
        return refuse("unknown kernel variant");
    bool vectors = vectors_can_take(g);
    if (variant == ACC950_VARIANT_AUTO && !vectors && !g.offsets && workspace) {
        const Packed p = packed(g);
        if (p.possible && p.a_bytes + p.b_bytes <= workspace_bytes) {
            uint8_t* at = (uint8_t*)workspace;
            if (p.a_bytes) {
                if (int rc = ended(launch_f8_pack(F8PackArgs{g.A, g.a_rs, g.a_cs, g.M, g.K, at, p.a_pitch}, stream), what)) return rc;
                g.A = at; g.a_rs = p.a_pitch; g.a_cs = 1;
                at += p.a_bytes;
            }
            if (p.b_bytes) {
                if (int rc = ended(launch_f8_pack(F8PackArgs{g.B, g.b_cs, g.b_rs, g.N, g.K, at, p.a_pitch}, stream), what)) return rc;
                g.B = at; g.b_cs = p.a_pitch; g.b_rs = 1;
                at += p.b_bytes;
            }
            workspace = at;
            workspace_bytes -= p.a_bytes + p.b_bytes;
            vectors = true;
        }
    }
    if (variant == ACC950_F8_VARIANT_ANY || (variant == ACC950_VARIANT_AUTO && !vectors)) return ended(launch_f8_gemm_any(g, stream), what);
    if (!vectors) return set_last_error(ACC950_UNSUPPORTED, "this kernel takes operands that are contiguous along K, with rows on 16-byte boundaries");
    if (!workspace) workspace_bytes = 0;
    TileChoice choice;
    if (variant == ACC950_VARIANT_AUTO) {
        if (rows_of_matrix(g) <= FEW_ROWS) return ended(launch_f8_gemm_few(g, few_form(g), wide, stream), what);
        choice = choose_tile(g, wide, workspace_bytes);
        if (choice.few) return ended(launch_f8_gemm_few(g, 0, wide, stream), what);
    } else if (variant >= ACC950_F8_VARIANT_FEW) {
        const int n = (int)variant - ACC950_F8_VARIANT_FEW;
        return ended(launch_f8_gemm_few(g, n % F8_FEW_FORMS, n >= F8_FEW_FORMS, stream), what);
    } else {
        const int n = (int)variant - ACC950_F8_VARIANT_TILE;
        wide = n >= F8_TILES;
        choice = TileChoice{n % F8_TILES, k_slices > 1 && !g.offsets ? (int)(k_slices < blocks_of(g.K) ? k_slices : blocks_of(g.K)) : 1, false};
    }
    if (!f8_tile_can_take(g, choice.tile, wide)) return set_last_error(ACC950_UNSUPPORTED, "the 256x256 tiles take factors for 128 columns and the e4m3 instruction's sums");
    g.parts_rs = (g.N + 3) / 4 * 4;
    if (choice.slices > 1) {
        if ((int64_t)choice.slices * 4 * g.M * g.parts_rs > workspace_bytes) return refuse("the workspace does not hold the slices' sums");
        if (choice.slices > 65535) return refuse("at most 65535 slices of K");
        g.slice_blocks = (int)((blocks_of(g.K) + choice.slices - 1) / choice.slices);
        g.slices = (int)((blocks_of(g.K) + g.slice_blocks - 1) / g.slice_blocks);
        g.parts = (float*)workspace;
    }
    if (int rc = ended(launch_f8_gemm_tile(g, choice.tile, wide, stream), what)) return rc;
    return g.slices > 1 ? ended(launch_f8_add_slices(g, stream), what) : ACC950_OK;
}

} // namespace

extern "C" int acc950_f8_quantize(const acc950_f8_quantize_call* c)
{
    if (!c) return refuse("null call");
    if (!float_type(c->in_type)) return refuse("quantising takes fp32, fp16 and bf16");
    if (!size_ok(c->rows) || !size_ok(c->cols)) return refuse("matrix sizes must lie between 0 and 2^31 - 1024");
    if (c->x_row_stride < 0 || c->x_col_stride < 0 || c->q_row_stride < 0 || c->s_row_stride < 0 || c->s_block_stride < 0)
        return refuse("negative strides are not supported");
    if (c->activation != ACC950_ACT_NONE && c->activation != ACC950_ACT_RELU && c->activation != ACC950_ACT_SILU_MUL) return refuse("unknown activation");
    if (c->transpose && c->activation != ACC950_ACT_NONE) return set_last_error(ACC950_UNSUPPORTED, "an activation goes with rows quantised as they lie, not transposed");
    if (c->group_rows != 1 && c->group_rows != F8_BLOCK) return refuse("group_rows must be 1 or 128");
    if (c->rows == 0 || c->cols == 0) return ACC950_OK;
    if (!c->x || !c->q || !c->scale) return refuse("null matrix pointer");
    if (misaligned(c->x, type_bytes(c->in_type)) || misaligned(c->scale, 4)) return refuse("a pointer is not aligned to its element type");
    F8QuantizeArgs a{};
    a.x = c->x; a.x_rs = c->x_row_stride; a.x_cs = c->x_col_stride;
    a.in_type = (int)c->in_type; a.rows = (int)c->rows; a.cols = (int)c->cols;
    a.act = (int)c->activation; a.transpose = c->transpose != 0; a.group_rows = (int)c->group_rows; a.pow2 = c->power_of_two != 0;
    if (a.act == ACC950_ACT_NONE && a.x_cs != 1 && a.x_rs == 1) { // a matrix that lies transposed (bf16 4096x4096 column by column 73 us, so 11)
        std::swap(a.rows, a.cols);
        std::swap(a.x_rs, a.x_cs);
        a.transpose = !a.transpose;
    }
    a.q = (uint8_t*)c->q; a.q_rs = c->q_row_stride;
    a.scale = (float*)c->scale; a.s_rs = c->s_row_stride; a.s_bs = c->s_block_stride;
    return ended(launch_f8_quantize(a, (hipStream_t)c->stream), "quantising");
}

namespace {

F8GemmArgs args_of(const acc950_f8_gemm_call* c)
{
    F8GemmArgs g{};
    g.A = (const uint8_t*)c->A; g.a_rs = c->a_row_stride; g.a_cs = c->a_col_stride;
    g.a_scale = (const float*)c->a_scale; g.as_rs = c->as_row_stride; g.as_ks = c->as_block_stride;
    g.B = (const uint8_t*)c->B; g.b_rs = c->b_row_stride; g.b_cs = c->b_col_stride;
    g.b_scale = (const float*)c->b_scale; g.bs_ks = c->bs_block_stride; g.bs_cs = c->bs_col_stride;
    g.group_shift = c->group_cols == 1 ? 0 : 7;
    g.C = c->C; g.c_rs = c->c_row_stride; g.c_cs = c->c_col_stride;
    g.M = (int)c->M; g.N = (int)c->N; g.K = (int)c->K;
    g.out_type = (int)c->out_type; g.epilogue = (int)c->epilogue;
    return g;
}

} // namespace

extern "C" int acc950_f8_gemm(const acc950_f8_gemm_call* c)
{
    if (!c) return refuse("null call");
    if (!float_type(c->out_type)) return refuse("the product's result is fp32, fp16 or bf16");
    if (!size_ok(c->M) || !size_ok(c->N) || !size_ok(c->K)) return refuse("matrix sizes must lie between 0 and 2^31 - 1024");
    if (c->a_row_stride < 0 || c->a_col_stride < 0 || c->as_row_stride < 0 || c->as_block_stride < 0 || c->b_row_stride < 0 || c->b_col_stride < 0 ||
        c->bs_block_stride < 0 || c->bs_col_stride < 0 || c->c_row_stride < 0 || c->c_col_stride < 0)
        return refuse("negative strides are not supported");
    if (c->group_cols != 1 && c->group_cols != F8_BLOCK) return refuse("group_cols must be 1 or 128");
    if (c->epilogue != ACC950_EPILOGUE_NONE && c->epilogue != ACC950_EPILOGUE_RELU) return refuse("the epilogue of a block-scaled product is none or ReLU");
    if (c->M == 0 || c->N == 0) return ACC950_OK;
    if (!c->C || (c->K > 0 && (!c->A || !c->B || !c->a_scale || !c->b_scale))) return refuse("null matrix pointer");
    if (misaligned(c->C, type_bytes(c->out_type)) || misaligned(c->a_scale, 4) || misaligned(c->b_scale, 4))
        return refuse("a pointer is not aligned to its element type");
    if (c->k_slices < 0 || c->workspace_bytes < 0) return refuse("negative number of slices or bytes");
    if (misaligned(c->workspace, 16)) return refuse("the workspace must be 16-byte aligned");
    return run_gemm(args_of(c), c->variant, c->out_type == ACC950_F32, c->k_slices, c->workspace, c->workspace_bytes, (hipStream_t)c->stream);
}

extern "C" int64_t acc950_f8_gemm_workspace(const acc950_f8_gemm_call* c)
{
    if (!c || !float_type(c->out_type) || !size_ok(c->M) || !size_ok(c->N) || !size_ok(c->K)) return -1;
    if (c->M == 0 || c->N == 0 || c->K == 0) return 0;
    if (c->variant != ACC950_VARIANT_AUTO) return c->k_slices > 1 && c->k_slices <= 65535 ? c->k_slices * 4 * c->M * ((c->N + 3) / 4 * 4) : 0;
    const F8GemmArgs g = args_of(c);
    int64_t bytes = 0;
    if (!vectors_can_take(g)) {
        const Packed p = packed(g);
        if (!p.possible) return 0;
        bytes = p.a_bytes + p.b_bytes;
    }
    if (g.M <= FEW_ROWS) return bytes;
    const TileChoice t = choose_tile(g, c->out_type == ACC950_F32, INT64_MAX);
    return bytes + (t.slices > 1 && !t.few ? t.slices * 4 * c->M * ((c->N + 3) / 4 * 4) : 0);
}

extern "C" int acc950_route(const acc950_route_call* c)
{
    if (!c) return refuse("null call");
    if (!float_type(c->in_type)) return refuse("routing takes fp32, fp16 and bf16 logits");
    if (!size_ok(c->tokens) || c->experts < 1 || c->experts > 1024) return refuse("routing takes 1 to 1024 experts and a number of tokens below 2^31 - 1024");
    if (c->top_k < 1 || c->top_k > 64 || c->top_k > c->experts) return refuse("top_k must lie between 1 and the number of experts, 64 at most");
    if (c->l_row_stride < 0) return refuse("negative strides are not supported");
    if (c->score != ACC950_SCORE_SOFTMAX && c->score != ACC950_SCORE_SIGMOID) return refuse("unknown score");
    if (c->group_score != ACC950_GROUP_BEST && c->group_score != ACC950_GROUP_BEST_TWO) return refuse("unknown score of a group");
    if (c->groups < 1 || c->groups > 64 || c->experts % c->groups) return refuse("the number of groups must divide the number of experts, 64 at most");
    if (c->top_groups < 1 || c->top_groups > c->groups) return refuse("top_groups must lie between 1 and the number of groups");
    if (c->route_scale != c->route_scale) return refuse("NaN op argument");
    if (c->tokens == 0) return ACC950_OK;
    if (!c->logits || !c->ids || !c->weights) return refuse("null pointer");
    if (misaligned(c->logits, type_bytes(c->in_type)) || misaligned(c->bias, 4) || misaligned(c->ids, 4) || misaligned(c->weights, 4))
        return refuse("a pointer is not aligned to its element type");
    RouteArgs a{};
    a.logits = c->logits; a.l_rs = c->l_row_stride; a.bias = (const float*)c->bias;
    a.in_type = (int)c->in_type; a.tokens = (int)c->tokens; a.experts = (int)c->experts; a.top_k = (int)c->top_k;
    a.score = (int)c->score; a.groups = (int)c->groups; a.top_groups = (int)c->top_groups; a.group_score = (int)c->group_score;
    a.renormalise = c->renormalise != 0; a.scale = (float)c->route_scale;
    a.ids = (int*)c->ids; a.weights = (float*)c->weights;
    return ended(launch_route(a, (hipStream_t)c->stream), "routing");
}

extern "C" int acc950_route_backward(const acc950_route_backward_call* c)
{
    if (!c) return refuse("null call");
    if (!float_type(c->in_type)) return refuse("routing takes fp32, fp16 and bf16 logits");
    if (!size_ok(c->tokens) || c->experts < 1 || c->experts > 1024) return refuse("routing takes 1 to 1024 experts and a number of tokens below 2^31 - 1024");
    if (c->top_k < 1 || c->top_k > 64 || c->top_k > c->experts) return refuse("top_k must lie between 1 and the number of experts, 64 at most");
    if (c->l_row_stride < 0 || c->grad_row_stride < 0) return refuse("negative strides are not supported");
    if (c->score != ACC950_SCORE_SOFTMAX && c->score != ACC950_SCORE_SIGMOID) return refuse("unknown score");
    if (c->route_scale != c->route_scale) return refuse("NaN op argument");
    if (c->tokens == 0) return ACC950_OK;
    if (!c->logits || !c->ids || !c->dweights || !c->dlogits) return refuse("null pointer");
    if (misaligned(c->logits, type_bytes(c->in_type)) || misaligned(c->dlogits, type_bytes(c->in_type)) || misaligned(c->ids, 4) || misaligned(c->dweights, 4))
        return refuse("a pointer is not aligned to its element type");
    RouteArgs a{};
    a.logits = c->logits; a.l_rs = c->l_row_stride;
    a.in_type = (int)c->in_type; a.tokens = (int)c->tokens; a.experts = (int)c->experts; a.top_k = (int)c->top_k;
    a.score = (int)c->score; a.renormalise = c->renormalise != 0; a.scale = (float)c->route_scale;
    a.ids = (int*)c->ids; a.dweights = (const float*)c->dweights; a.dlogits = c->dlogits; a.g_rs = c->grad_row_stride;
    return ended(launch_route_backward(a, (hipStream_t)c->stream), "routing's gradient");
}

extern "C" int64_t acc950_expert_plan_workspace(int64_t tokens, int64_t top_k, int64_t experts)
{
    if (!size_ok(tokens) || top_k < 1 || top_k > 64 || !size_ok(tokens * top_k) || experts < 1 || experts > 1024) return -1;
    return expert_plan_workspace(tokens * top_k, experts);
}

extern "C" int acc950_expert_plan(const acc950_expert_plan_call* c) { return acc950_expert_plan_within(c, INT64_MAX); }

extern "C" int acc950_expert_plan_within(const acc950_expert_plan_call* c, int64_t workspace_bytes)
{
    if (!c) return refuse("null call");
    const int64_t need = acc950_expert_plan_workspace(c->tokens, c->top_k, c->experts);
    if (need < 0) return refuse("a plan takes 1 to 1024 experts, top_k of 1 to 64, and a number of pairs below 2^31 - 1024");
    if (workspace_bytes < need) return refuse("the workspace is smaller than the plan's");
    if (!c->offsets || (c->tokens > 0 && (!c->ids || !c->order || !c->position)) || (need > 0 && !c->workspace)) return refuse("null pointer");
    if (misaligned(c->ids, 4) || misaligned(c->order, 4) || misaligned(c->position, 4) || misaligned(c->offsets, 4) || misaligned(c->workspace, 4))
        return refuse("a pointer is not aligned to its element type");
    PlanArgs a{};
    a.ids = (const int*)c->ids; a.pairs = (int)(c->tokens * c->top_k); a.experts = (int)c->experts;
    a.order = (int*)c->order; a.position = (int*)c->position; a.offsets = (int*)c->offsets; a.counts = (int*)c->workspace;
    return ended(launch_expert_plan(a, (hipStream_t)c->stream), "the plan of the experts' rows");
}

extern "C" int acc950_f8_expert_gemm(const acc950_f8_expert_gemm_call* c)
{
    if (!c) return refuse("null call");
    if (!float_type(c->out_type)) return refuse("the product's result is fp32, fp16 or bf16");
    if (!size_ok(c->rows) || !size_ok(c->N) || !size_ok(c->K)) return refuse("matrix sizes must lie between 0 and 2^31 - 1024");
    if (c->experts < 1 || c->experts > 1024 || c->top_k < 1 || c->top_k > 64) return refuse("experts' products take 1 to 1024 experts and top_k of 1 to 64");
    if (c->a_row_stride < 0 || c->as_row_stride < 0 || c->as_block_stride < 0 || c->b_expert_stride < 0 || c->b_col_stride < 0 || c->bs_expert_stride < 0 ||
        c->bs_block_stride < 0 || c->bs_col_stride < 0 || c->c_row_stride < 0)
        return refuse("negative strides are not supported");
    if (c->rows == 0 || c->N == 0) return ACC950_OK;
    if (!c->C || !c->order || !c->offsets || (c->K > 0 && (!c->A || !c->B || !c->a_scale || !c->b_scale))) return refuse("null pointer");
    if (misaligned(c->C, type_bytes(c->out_type)) || misaligned(c->a_scale, 4) || misaligned(c->b_scale, 4) || misaligned(c->order, 4) ||
        misaligned(c->offsets, 4) || misaligned(c->row_weights, 4))
        return refuse("a pointer is not aligned to its element type");
    F8GemmArgs g{};
    g.A = (const uint8_t*)c->A; g.a_rs = c->a_row_stride; g.a_cs = 1;
    g.a_scale = (const float*)c->a_scale; g.as_rs = c->as_row_stride; g.as_ks = c->as_block_stride;
    g.B = (const uint8_t*)c->B; g.b_rs = 1; g.b_cs = c->b_col_stride; g.b_es = c->b_expert_stride;
    g.b_scale = (const float*)c->b_scale; g.bs_ks = c->bs_block_stride; g.bs_cs = c->bs_col_stride; g.bs_es = c->bs_expert_stride;
    g.group_shift = 7;
    g.C = c->C; g.c_rs = c->c_row_stride; g.c_cs = 1;
    g.M = (int)c->rows; g.N = (int)c->N; g.K = (int)c->K;
    g.out_type = (int)c->out_type; g.epilogue = EPI_NONE;
    g.offsets = (const int*)c->offsets; g.order = (const int*)c->order;
    g.experts = (int)c->experts; g.gather = c->gather != 0;
    g.top_k = (int)c->top_k; g.by_top_k = F8Over((unsigned)c->top_k);
    g.row_weights = (const float*)c->row_weights;
    return run_gemm(g, c->variant, c->out_type == ACC950_F32, 1, nullptr, 0, (hipStream_t)c->stream);
}

extern "C" int acc950_expert_combine(const acc950_expert_combine_call* c)
{
    if (!c) return refuse("null call");
    if (!float_type(c->type)) return refuse("rows are fp32, fp16 or bf16");
    if (!size_ok(c->tokens) || !size_ok(c->cols) || c->top_k < 1 || c->top_k > 64) return refuse("sizes must lie between 0 and 2^31 - 1024, top_k between 1 and 64");
    if (c->x_row_stride < 0 || c->y_row_stride < 0) return refuse("negative strides are not supported");
    if (c->tokens == 0 || c->cols == 0) return ACC950_OK;
    if (!c->x || !c->position || !c->y) return refuse("null pointer");
    if (misaligned(c->x, type_bytes(c->type)) || misaligned(c->y, type_bytes(c->type)) || misaligned(c->position, 4) || misaligned(c->weights, 4))
        return refuse("a pointer is not aligned to its element type");
    CombineArgs a{};
    a.x = c->x; a.x_rs = c->x_row_stride; a.position = (const int*)c->position; a.weights = (const float*)c->weights;
    a.y = c->y; a.y_rs = c->y_row_stride; a.in_type = a.type = (int)c->type; a.tokens = (int)c->tokens; a.top_k = (int)c->top_k; a.cols = (int)c->cols;
    return ended(launch_expert_combine(a, (hipStream_t)c->stream), "the sum of the experts' rows");
}

namespace {

// Whether the gate and up product of a routed layer goes through the kernels that end in codes: whole 16-byte pieces of K, 32-bit offsets
// from x's first row, from a tile's first column in the weights, and from the gate's scales to the up matrix's.
bool ends_in_codes(int64_t tokens, int64_t hidden, int64_t inner)
{
    const int64_t most = 1ll << 32;
    return hidden % 16 == 0 && tokens * hidden < most && tokens * 4 < most && 256 * hidden < most && blocks_of(inner + 256) * blocks_of(hidden) * 4 < most;
}

// Where the steps of a routed layer keep their results in its workspace (bytes from its start).
struct FfnLayout {
    int64_t order, position, offsets, counts, xq, x_scale, h, hq, h_scale, rows, row_scale, tickets, bytes;
    int64_t x_pitch, h_pitch;
};

FfnLayout ffn_layout(int64_t tokens, int64_t hidden, int64_t inner, int64_t experts, int64_t top_k)
{
    FfnLayout l{};
    const int64_t pairs = tokens * top_k;
    auto place = [&](int64_t bytes) {
        const int64_t at = l.bytes;
        l.bytes += (bytes + 255) / 256 * 256;
        return at;
    };
    l.x_pitch = (hidden + 15) / 16 * 16;
    l.h_pitch = (inner + 15) / 16 * 16;
    l.order = place(pairs * 4);
    l.position = place(pairs * 4);
    l.offsets = place((experts + 1) * 4);
    l.counts = place(expert_plan_workspace(pairs, experts));
    l.xq = place(tokens * l.x_pitch);
    l.x_scale = place(tokens * blocks_of(hidden) * 4);
    l.h = place(ends_in_codes(tokens, hidden, inner) ? 0 : pairs * 2 * inner * 4);
    l.hq = place(pairs * l.h_pitch);
    l.h_scale = place(pairs * blocks_of(inner) * 4);
    l.rows = place(pairs * hidden * 4);
    l.tickets = place(16 * 4);
    l.row_scale = place(pairs * ((hidden + 63) / 64 * 2) * 4);
    return l;
}

bool ffn_sizes_ok(int64_t tokens, int64_t hidden, int64_t inner, int64_t experts, int64_t top_k)
{
    return size_ok(tokens) && size_ok(hidden) && size_ok(inner) && inner <= 0x3fffffff && experts >= 1 && experts <= 1024 && top_k >= 1 && top_k <= 64 &&
           size_ok(tokens * top_k);
}

} // namespace

extern "C" int64_t acc950_f8_expert_ffn_workspace(int64_t tokens, int64_t hidden, int64_t inner, int64_t experts, int64_t top_k)
{
    if (!ffn_sizes_ok(tokens, hidden, inner, experts, top_k)) return -1;
    return ffn_layout(tokens, hidden, inner, experts, top_k).bytes;
}

extern "C" int acc950_f8_expert_ffn(const acc950_f8_expert_ffn_call* c) { return acc950_f8_expert_ffn_within(c, INT64_MAX); }

extern "C" int acc950_f8_expert_ffn_within(const acc950_f8_expert_ffn_call* c, int64_t workspace_bytes)
{
    if (!c) return refuse("null call");
    if (c->type != ACC950_F16 && c->type != ACC950_BF16) return refuse("a routed layer takes fp16 and bf16");
    if (!ffn_sizes_ok(c->tokens, c->hidden, c->inner, c->experts, c->top_k))
        return refuse("a routed layer takes 1 to 1024 experts, top_k of 1 to 64, inner below 2^30, and sizes and a number of pairs below 2^31 - 1024");
    if (c->x_row_stride < 0 || c->y_row_stride < 0) return refuse("negative strides are not supported");
    if (c->tokens == 0 || c->hidden == 0) return ACC950_OK;
    if (!c->x || !c->ids || !c->weights || !c->y || !c->workspace || (c->inner > 0 && (!c->w13 || !c->w13_scale || !c->w2 || !c->w2_scale)))
        return refuse("null pointer");
    if (misaligned(c->x, 2) || misaligned(c->y, 2) || misaligned(c->ids, 4) || misaligned(c->weights, 4) || misaligned(c->w13_scale, 4) || misaligned(c->w2_scale, 4))
        return refuse("a pointer is not aligned to its element type");
    if (misaligned(c->workspace, 256)) return refuse("the workspace must be 256-byte aligned");
    if (misaligned(c->w13, 16) || misaligned(c->w2, 16)) return refuse("the experts' matrices must start on 16-byte boundaries");
    const int64_t pairs = c->tokens * c->top_k, hb = blocks_of(c->hidden), ib = blocks_of(c->inner);
    const FfnLayout l = ffn_layout(c->tokens, c->hidden, c->inner, c->experts, c->top_k);
    if (workspace_bytes < l.bytes) return refuse("the workspace is smaller than the layer's");
    char* ws = (char*)c->workspace;
    const hipStream_t stream = (hipStream_t)c->stream;

    PlanArgs plan{};
    plan.ids = (const int*)c->ids; plan.pairs = (int)pairs; plan.experts = (int)c->experts;
    plan.order = (int*)(ws + l.order); plan.position = (int*)(ws + l.position); plan.offsets = (int*)(ws + l.offsets); plan.counts = (int*)(ws + l.counts);
    plan.zeros = (int*)(ws + l.tickets);
    F8QuantizeArgs q{};
    q.x = c->x; q.x_rs = c->x_row_stride; q.x_cs = 1; q.in_type = (int)c->type; q.rows = (int)c->tokens; q.cols = (int)c->hidden;
    q.group_rows = 1; q.pow2 = 1;
    q.q = (uint8_t*)(ws + l.xq); q.q_rs = l.x_pitch;
    q.scale = (float*)(ws + l.x_scale); q.s_rs = 1; q.s_bs = c->tokens;
    if (int rc = ended(launch_expert_plan_and_quantize(plan, q, stream), "the plan of the experts' rows")) return rc;

    // The inner values are not rounded before they become codes: half a unit of fp16 already moves 1 in 500 of them across a boundary between
    // two codes.  The e4m3 instruction's sums (2^-16) move 1 in 5000, and 1 in 30000 of a row's scales.  With few rows to an expert, where the weights' bytes are what takes the
    // time, both products have fp32 sums (us with / without, 64 experts of 2048x1024: 8 tokens 47.0 / 47.0, 120 115.4 / 114.6; 20 of 1040x720: 8 tokens 23.2 / 21.8).  With
    // more, the gate and up product of a fp16 layer has, and that of a bf16 layer has not: it would cost 100 of 304 us (4096 tokens), 16 of 156 (1024), for an
    // error against the same layer in 64 bits of 1.7e-3, which is bf16's own rounding, and not 2.0e-3.
    const bool wide = c->type == ACC950_F16;
    F8GemmArgs g{};
    g.A = q.q; g.a_rs = q.q_rs; g.a_cs = 1; g.a_scale = q.scale; g.as_rs = q.s_rs; g.as_ks = q.s_bs;
    g.B = (const uint8_t*)c->w13; g.b_rs = 1; g.b_cs = c->hidden; g.b_es = 2 * c->inner * c->hidden; g.b_up = c->inner * c->hidden;
    g.b_scale = (const float*)c->w13_scale; g.bs_ks = 1; g.bs_cs = hb; g.bs_es = 2 * ib * hb; g.bs_up = ib * hb; g.group_shift = 7;
    g.C = ws + l.hq; g.c_rs = l.h_pitch; g.c_cs = 1; g.M = (int)pairs; g.N = (int)c->inner; g.K = (int)c->hidden; g.epilogue = EPI_NONE;
    g.offsets = plan.offsets; g.order = plan.order; g.experts = (int)c->experts; g.gather = 1;
    g.top_k = (int)c->top_k; g.by_top_k = F8Over((unsigned)c->top_k);
    g.out_scale = (float*)(ws + l.h_scale); g.os_rs = 1; g.os_bs = pairs;
    g.tickets = plan.zeros;
    if (c->inner > 0 && ends_in_codes(c->tokens, c->hidden, c->inner)) {
        if (int rc = ended(rows_of_matrix(g) <= FEW_ROWS ? launch_f8_gated_few(g, stream) : launch_f8_gated_tile(g, wide, stream), "gate and up product")) return rc;
    } else if (c->inner > 0) {
        // gate | up in fp32, then the activation
        F8GemmArgs half = g;
        half.c_rs = 2 * c->inner; half.out_type = T_F32;
        for (int up = 0; up < 2; ++up) {
            half.B = g.B + up * g.b_up; half.b_scale = g.b_scale + up * g.bs_up;
            half.C = (float*)(ws + l.h) + up * c->inner;
            if (int rc = run_gemm(half, ACC950_VARIANT_AUTO, true, 1, nullptr, 0, stream)) return rc;
        }
        q.x = ws + l.h; q.x_rs = 2 * c->inner; q.in_type = T_F32; q.rows = (int)pairs; q.cols = (int)c->inner; q.act = ACC950_ACT_SILU_MUL;
        q.q = (uint8_t*)(ws + l.hq); q.q_rs = l.h_pitch; q.scale = g.out_scale; q.s_rs = 1; q.s_bs = pairs;
        if (int rc = ended(launch_f8_quantize(q, stream), "quantising")) return rc;
    }

    // A token's rows are terms of its sum and are not rounded to the result's type (the layer's error against 64 bits would be 1.4 times that of one
    // rounding).  They stay in fp32; or, where there are many for a bf16 result, in fp16 with a power of two for each 32 or 64 columns: 2^-12 of a value
    // beside the result's 2^-9, and half the bytes of the largest thing the layer writes and reads.
    g.A = (const uint8_t*)(ws + l.hq); g.a_rs = l.h_pitch; g.a_scale = g.out_scale; g.as_rs = 1; g.as_ks = pairs;
    g.B = (const uint8_t*)c->w2; g.b_cs = c->inner; g.b_es = c->hidden * c->inner;
    g.b_scale = (const float*)c->w2_scale; g.bs_cs = ib; g.bs_es = hb * ib;
    g.C = ws + l.rows; g.c_rs = c->hidden; g.N = (int)c->hidden; g.K = (int)c->inner;
    const bool halves = c->type == ACC950_BF16 && rows_of_matrix(g) > FEW_ROWS && vectors_can_take(g);
    g.out_type = halves ? T_F16 : T_F32;
    g.out_scale = halves ? (float*)(ws + l.row_scale) : nullptr; g.os_rs = (c->hidden + 63) / 64 * 2;
    g.gather = 0; g.tickets = plan.zeros + 8;
    const bool few = rows_of_matrix(g) <= FEW_ROWS; // (else the e4m3 instruction: 2^-16 of a row beside 2^-12 or 2^-9 of the result)
    if (int rc = run_gemm(g, ACC950_VARIANT_AUTO, few, 1, nullptr, 0, stream)) return rc;

    CombineArgs y{};
    y.x = ws + l.rows; y.x_rs = c->hidden; y.position = plan.position; y.y = c->y; y.y_rs = c->y_row_stride;
    y.weights = (const float*)c->weights; y.in_type = g.out_type; y.scale = g.out_scale; y.s_rs = g.os_rs; y.type = (int)c->type; y.tokens = (int)c->tokens; y.top_k = (int)c->top_k; y.cols = (int)c->hidden;
    return ended(launch_expert_combine(y, stream), "the sum of the experts' rows");
}
