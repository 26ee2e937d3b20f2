// Feed-forward operators in 8-bit floating point: what the kernels' translation units and capi_f8.hip share.
#pragma once
#include "common.h"

namespace acc950 {

constexpr int T_F8 = 6;
constexpr int F8_BLOCK = 128;

// Quotients of numbers below 2^31 by one divisor d > 0: with 2^(l - 1) < d <= 2^l, floor(2^(31 + l) / d) + 1 fits 32 bits, and the high half of its product
// shifted right by l - 1 is exact.  (A division takes twenty instructions, one of 64 bits a hundred.)
struct F8Over {
    unsigned mul; // 0: d is 1
    int shift;
    F8Over() = default;
    explicit F8Over(unsigned d) : mul(0), shift(0)
    {
        int l = 0;
        while ((1ull << l) < d) ++l;
        if (d > 1) mul = (unsigned)((1ull << (31 + l)) / d + 1), shift = l - 1;
    }
    __device__ __forceinline__ unsigned operator()(unsigned n) const { return mul ? __umulhi(n, mul) >> shift : n; }
};

// One block-scaled product, or one per expert of a plan.  Strides are in elements.
struct F8GemmArgs {
    const uint8_t* A;
    int64_t a_rs, a_cs;
    const float* a_scale;
    int64_t as_rs, as_ks; // per row, per block of K
    const uint8_t* B;
    int64_t b_rs, b_cs;   // per k, per column
    const float* b_scale;
    int64_t bs_ks, bs_cs; // per block of K, per group of columns
    int group_shift;      // columns of a group: 1 << group_shift (0 or 7)
    void* C;
    int64_t c_rs, c_cs;
    int M, N, K;
    int out_type, epilogue;
    // experts: rows [offsets[e], offsets[e + 1]) of C take the matrix of expert e (offsets null: a plain product)
    const int* offsets;
    const int* order;     // pair of a sorted row
    int experts, top_k, gather;
    F8Over by_top_k; // a pair's token
    int64_t b_es, bs_es;
    const float* row_weights; // by pair, or null
    int rows_log2;        // rows of an expert's tile, set at the launch: what the kernel's tiles hold, or half of it
    int* tickets;         // 8 counters, zero at the launch (f8_tile_by_ticket), or null
    // gated: B's second matrix (up) lies b_up elements behind the first (gate), its scales bs_up; C takes codes, out_scale their scales.
    // Not gated, tiles of experts' rows, out_type fp16: with out_scale C takes fp16 values, whose row has a power of two for each 32 columns at
    // out_scale + row * os_rs (even); such rows have no weights.
    int64_t b_up, bs_up;
    float* out_scale;
    int64_t os_rs, os_bs;
    // K in slices of slice_blocks blocks, one per blockIdx.z: fp32 sums of slice z at parts + z * M * parts_rs
    int slices, slice_blocks;
    float* parts;
    int64_t parts_rs;
};

struct F8PackArgs {
    const uint8_t* x;
    int64_t rs, cs;
    int rows, cols;
    uint8_t* q;
    int64_t pitch; // a multiple of 16
};

struct F8QuantizeArgs {
    const void* x;
    int64_t x_rs, x_cs;
    int in_type, rows, cols, act, transpose, group_rows, pow2;
    F8Over by_quads; // set at the launch: a unit's row
    uint8_t* q;
    int64_t q_rs;
    float* scale;
    int64_t s_rs, s_bs;
};

struct RouteArgs {
    const void* logits;
    int64_t l_rs;
    const float* bias;
    int in_type, tokens, experts, top_k, score, groups, top_groups, group_score, renormalise;
    float scale;
    int* ids;
    float* weights;
    const float* dweights; // backward
    void* dlogits;
    int64_t g_rs;
};

struct PlanArgs {
    const int* ids;
    int pairs, experts;
    int *order, *position, *offsets;
    int* counts; // workspace: [chunks][experts + 1]
    int* zeros;  // 16 counters to be set to 0, or null
};

struct CombineArgs {
    const void* x;
    int64_t x_rs;
    const int* position;
    const float* weights;
    void* y;
    int64_t y_rs;
    const float* scale; // of x in fp16, for each 32 columns of a row; or null
    int64_t s_rs;
    F8Over by_pieces; // set at the launch: a piece's token, where there are few enough (below 2^31) of them
    int few;
    int in_type, type, tokens, top_k, cols; // x's type: y's, or fp32, or with `scale` fp16
};

hipError_t launch_f8_quantize(const F8QuantizeArgs& a, hipStream_t s);
hipError_t launch_f8_pack(const F8PackArgs& a, hipStream_t s);
hipError_t launch_f8_gemm_any(const F8GemmArgs& a, hipStream_t s);
// tiles 0 to 3: 256x256 (waves that take turns), 128x128, 64x64 (four blocks of K in LDS), 64x64 (two); wide: the fp16 instruction on widened codes
constexpr int F8_TILES = 4;
constexpr int F8_TILE_SIZE[F8_TILES] = {256, 128, 64, 64};
bool f8_tile_can_take(const F8GemmArgs& a, int tile, bool wide);
hipError_t launch_f8_gemm_tile(const F8GemmArgs& a, int tile, bool wide, hipStream_t s);
hipError_t launch_f8_add_slices(const F8GemmArgs& a, hipStream_t s);
constexpr int F8_FEW_FORMS = 2;
hipError_t launch_f8_gemm_few(const F8GemmArgs& a, int form, bool wide, hipStream_t s);
hipError_t launch_f8_gated_few(const F8GemmArgs& a, hipStream_t s);
hipError_t launch_f8_gated_tile(const F8GemmArgs& a, bool wide, hipStream_t s);
hipError_t launch_route(const RouteArgs& a, hipStream_t s);
hipError_t launch_route_backward(const RouteArgs& a, hipStream_t s);
hipError_t launch_expert_plan(const PlanArgs& a, hipStream_t s);
hipError_t launch_expert_plan_and_quantize(const PlanArgs& a, const F8QuantizeArgs& q, hipStream_t s); // (q: 16-bit rows in groups of 1 x 128)
int64_t expert_plan_workspace(int64_t pairs, int64_t experts);
hipError_t launch_expert_combine(const CombineArgs& a, hipStream_t s);

// Sets the calling thread's error text and hands back its status (capi.hip).
int set_last_error(int code, const char* text) noexcept;

// ---- device helpers ------------------------------------------------------------------------------

typedef int i32x8 __attribute__((ext_vector_type(8)));

// One block of 128 of a 16 x 16 product, d = cols x rows^T from zero.  A lane holds 32 values of one row on either side (which 32 is
// the same on both); of d lane l has row l % 16 of `rows` and columns (l / 16) * 4 .. + 3 of `cols`.
//
// NATIVE: the e4m3 instruction.  It adds its products in groups of eight lined up with the largest of them and keeps 13 bits below
// that (2^16 + 2^2 is 2^16, 2^16 + 2^3 is not): a result of random terms is off by 2^-16 of itself, which 16-bit results (2^-9 and
// 2^-12 rounded) do not show and fp32 ones do.
// WIDE: the values as fp16, which holds all of e4m3, on the fp16 instruction: sums in fp32 throughout, at half the rate.
template <bool WIDE> struct F8Fragment;
template <> struct F8Fragment<false> {
    i32x8 v;
    __device__ __forceinline__ void set(const i32x4& lo, const i32x4& hi) { v = i32x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]}; }
};
template <> struct F8Fragment<true> {
    f16x8 v[4];
    __device__ __forceinline__ void set_step(int s, const i32x4& lo, const i32x4& hi) // a quarter
    {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int at = s * 2 + h, x = at < 4 ? lo[at] : hi[at - 4];
            const auto a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x, 1.f, false), b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x, 1.f, true);
            v[s][h * 4] = a[0]; v[s][h * 4 + 1] = a[1]; v[s][h * 4 + 2] = b[0]; v[s][h * 4 + 3] = b[1];
        }
    }
    __device__ __forceinline__ void set(const i32x4& lo, const i32x4& hi)
    {
#pragma unroll
        for (int s = 0; s < 4; ++s) set_step(s, lo, hi);
    }
};
// one step (of 4) of a block of the wide form
__device__ __forceinline__ f32x4 mfma_f8_step(const F8Fragment<true>& cols, const F8Fragment<true>& rows, int s, const f32x4& d)
{
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(cols.v[s], rows.v[s], d, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma_f8_block(const F8Fragment<false>& cols, const F8Fragment<false>& rows)
{
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(cols.v, rows.v, f32x4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma_f8_block(const F8Fragment<true>& cols, const F8Fragment<true>& rows)
{
    f32x4 d{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int s = 0; s < 4; ++s) d = mfma_f8_step(cols, rows, s, d);
    return d;
}

// the larger of a lane's value and that of the lane d (1, 2, 4, 8: of the 16 in its row, turned; 16 or 32) away, without a trip through the LDS unit
__device__ __forceinline__ unsigned f8_max_over(unsigned m, int d)
{
    if (d == 1) return max(m, (unsigned)__builtin_amdgcn_mov_dpp((int)m, 0x121, 0xf, 0xf, true)); // row_ror
    if (d == 2) return max(m, (unsigned)__builtin_amdgcn_mov_dpp((int)m, 0x122, 0xf, 0xf, true));
    if (d == 4) return max(m, (unsigned)__builtin_amdgcn_mov_dpp((int)m, 0x124, 0xf, 0xf, true));
    if (d == 8) return max(m, (unsigned)__builtin_amdgcn_mov_dpp((int)m, 0x128, 0xf, 0xf, true));
    const auto v = d == 16 ? __builtin_amdgcn_permlane16_swap(m, m, false, false) : __builtin_amdgcn_permlane32_swap(m, m, false, false);
    return max(v[0], v[1]);
}

// a pair's token
__device__ __forceinline__ int f8_token(const F8GemmArgs& p, int pair) { return (int)p.by_top_k((unsigned)pair); }

// A scale from the largest magnitude of its group, and its inverse.  The power of two not below amax / 448 = amax / (1.75 * 2^8): exponent - 8, one more where
// the mantissa is over 1.75 (the quotient's own rounding changes none).  (NaN stays NaN; with powers of two it becomes infinity, whose group
// stands for NaN just the same.)
__device__ __forceinline__ float f8_scale_of(float amax, bool pow2)
{
    if (pow2) {
        const int bits = (int)__float_as_uint(amax), up = max(bits - (8 << 23) + 0x1fffff, 0x00800000) & 0x7f800000;
        return __int_as_float(bits >= 0x7f800000 ? 0x7f800000 : up);
    }
    // amax / 448, correctly rounded: the product with the reciprocal, and its remainder's share
    constexpr float over = 1.f / 448.f;
    const float q = amax * over, s = q < INFINITY ? fmaf(fmaf(-448.f, q, amax), over, q) : q;
    return s < 1.17549435e-38f ? 1.17549435e-38f : s;
}
__device__ __forceinline__ float f8_inverse_of(float s, bool pow2) { return pow2 ? __int_as_float(max(0x7f000000 - (int)__float_as_uint(s), 0)) : 1.f / s; }

// four values as e4m3, nearest even
__device__ __forceinline__ unsigned f8_pack4(float a, float b, float c, float d)
{
    int v = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, v, true);
}

// gate / (1 + exp(-gate)) * up, within 8 * 2^-24: exp(-gate) = 2^t * (1 + rest ln 2), t + rest = -gate log2(e) (the product's own rounding goes
// into `rest`), and the hardware's reciprocal, within one unit.  (With expf and a division the quantiser was bound by its arithmetic:
// 8192 x 11008 in 148 us.)  Where 2^t is infinite the quotient is 0, and below 2^-128 it adds nothing to 1; `rest` is left out of both, for where t itself is
// infinite (gates past 2.4e38) so is `rest`.
__device__ __forceinline__ float silu_mul(float gate, float up)
{
    const float t = gate * -1.44269502f;
    const float rest = fmaf(gate, -1.44269502f, -t) + gate * -1.92596303e-8f;
    const float e = __builtin_amdgcn_exp2f(t);
    return gate * __builtin_amdgcn_rcpf(1.f + (fabsf(t) < 128.f ? fmaf(e, rest * 0.693147182f, e) : e)) * up;
}

// The same for values that become codes at once behind sums of the e4m3 instruction, half the instructions: the exponent's own rounding moves exp(-gate) by |gate| * 2^-24 of itself, no more than
// what the sums of the e4m3 instruction bring along, and 1 in 10^5 of the codes across a boundary.
__device__ __forceinline__ float silu_mul_to_code(float gate, float up)
{
    return gate * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(gate * -1.44269502f)) * up;
}

// four neighbouring values of a row from column c on, in one store (vec: the row allows it) where none lies behind column n
__device__ __forceinline__ void f8_store4(char* row, int out_type, int64_t c, int64_t n, const f32x4& v, bool vec)
{
    if (vec && c + 4 <= n) {
        if (out_type == T_F32) *(f32x4*)(row + c * 4) = v;
        else {
            unsigned h[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) h[e] = out_type == T_F16 ? float_to_f16_bits(v[e]) : float_to_bf16_bits(v[e]);
            *(i32x2*)(row + c * 2) = i32x2{(int)(h[0] | h[1] << 16), (int)(h[2] | h[3] << 16)};
        }
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (c + e < n) store_out(row, out_type, c + e, v[e]);
    }
}

// the sum of a lane's value and all before it, by shifts within rows of 16 lanes and then of rows' last lanes into the rows behind
template <int CTRL, int ROWS>
__device__ __forceinline__ int shifted(int v) { return __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xf, false); }
__device__ __forceinline__ int sum_to_here(int v)
{
    v += shifted<0x111, 0xf>(v); // row_shr:1, 2, 4, 8
    v += shifted<0x112, 0xf>(v);
    v += shifted<0x114, 0xf>(v);
    v += shifted<0x118, 0xf>(v);
    v += shifted<0x142, 0xa>(v); // row_bcast:15 into rows 1 and 3
    v += shifted<0x143, 0xc>(v); // row_bcast:31 into rows 2 and 3
    return v;
}

// How many tiles of 2^rows_log2 rows the experts have; every lane of a wave calls it.
__device__ __forceinline__ int count_expert_tiles(const int* offsets, int experts, int rows_log2, int lane)
{
    int n = 0;
    for (int e0 = 0; e0 < experts; e0 += 64) {
        const int e = e0 + lane, lo = e < experts ? offsets[e] : 0, hi = e < experts ? offsets[e + 1] : 0;
        n += (hi - lo + (1 << rows_log2) - 1) >> rows_log2;
    }
    return __builtin_amdgcn_readlane(sum_to_here(n), 63);
}

// The experts' tiles of 2^rows_log2 rows: which expert has tile `t`, and its first row and rows' end.  Every lane of a wave calls it with
// the same t; false: there are fewer tiles.  `width` tiles of columns stand beside each tile of rows; on return t is the index
// among the expert's own tiles.
__device__ __forceinline__ bool find_expert_tile(const int* offsets, int experts, int rows_log2, int width, int lane, int& t, int& expert, int& row0, int& row_end)
{
    int base = 0;
    for (int e0 = 0; e0 < experts; e0 += 64) {
        const int e = e0 + lane;
        const int lo = e < experts ? offsets[e] : 0, hi = e < experts ? offsets[e + 1] : 0;
        const int n = ((hi - lo + (1 << rows_log2) - 1) >> rows_log2) * width;
        const int sum = sum_to_here(n);
        const unsigned long long past = __ballot(base + sum > t);
        if (past) {
            const int at = __builtin_amdgcn_readfirstlane(__ffsll((long long)past) - 1);
            expert = e0 + at;
            row0 = __builtin_amdgcn_readlane(lo, at);
            row_end = __builtin_amdgcn_readlane(hi, at);
            t -= base + __builtin_amdgcn_readlane(sum - n, at);
            return true;
        }
        base += __builtin_amdgcn_readlane(sum, 63);
    }
    return false;
}

} // namespace acc950
