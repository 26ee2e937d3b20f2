// Block-scaled e4m3 product of few rows: B streams from memory straight into registers, once; bound by its bytes.  8x11008x4096 (45 MB) 11.6 us, of which
// 2.5 are the launch; gate and up of 48 rows of 64 experts (143 MB) 26.5 us, 5.4 TB/s; down (71 MB) 14.2 us.
//
// A wave has TN blocks of 16 columns and every KW-th block of K (the KW waves of a column block read neighbouring pieces of B's rows at
// a time and add their sums up in LDS at the end); DEPTH blocks are on the way while one is multiplied.  A's rows come from the caches:
// 16 * TM rows of the block, again for every wave.
#pragma once
#include "f8_gemm_tile.h"

namespace acc950 {

// CW column units of a workgroup, KW slices of K.  GATED: a unit's first block of 16 columns is of the gate matrix, its second of
// the up matrix, eight units make a group of 128 inner values, and the result is silu(gate) * up as codes and scales.
template <int TM_, int TN_, int CW_, int KW_, int DEPTH_, bool WIDE_, bool COLUMNS_, bool EXPERTS_, bool GATED_>
struct F8FewConfig {
    static constexpr int TM = TM_, TN = TN_, CW = CW_, KW = KW_, DEPTH = DEPTH_;
    static constexpr bool WIDE = WIDE_, COLUMNS = COLUMNS_, EXPERTS = EXPERTS_, GATED = GATED_;
    static constexpr int NW = CW * KW, NT = NW * 64, BM = TM * 16, BN = GATED ? 128 : CW * TN * 16;
    static_assert(!GATED || (TN == 2 && CW == 8 && EXPERTS && !COLUMNS), "eight waves of 16 gate and 16 up columns");
};

template <typename Cfg>
__global__ void __launch_bounds__(Cfg::NT) f8_gemm_few_kernel(F8GemmArgs p)
{
    constexpr int TM = Cfg::TM, TN = Cfg::TN, KW = Cfg::KW, DEPTH = Cfg::DEPTH, BM = Cfg::BM, BN = Cfg::BN;
    using Fragment = F8Fragment<Cfg::WIDE>;
    __shared__ f32x4 parts[KW > 1 ? Cfg::CW * (KW - 1) * TM * TN : 1][64];
    __shared__ unsigned tops[Cfg::GATED ? 8 : 1][BM];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int unit = wave % Cfg::CW, slice = wave / Cfg::CW;
    const int frow = lane & 15, fg = lane >> 4;
    const int tiles_n = (p.N + BN - 1) / BN;
    int m0, row_end, n0, expert = 0;
    {
        int t = blockIdx.x;
        if constexpr (Cfg::EXPERTS) {
            int row0;
            if (!find_expert_tile(p.offsets, p.experts, __builtin_ctz(BM), tiles_n, lane, t, expert, row0, row_end)) return;
            // (tiles of rows that share columns of B stand beside each other)
            const int tiles_m = (row_end - row0 + BM - 1) / BM;
            m0 = row0 + t % tiles_m * BM;
            n0 = t / tiles_m * BN;
        } else {
            m0 = t / tiles_n * BM; row_end = p.M; n0 = t % tiles_n * BN;
        }
    }
    const uint8_t* B = p.B + expert * p.b_es;
    const float* b_scale = p.b_scale + expert * p.bs_es;

    const uint8_t *a_src[TM], *b_src[TN];
    const float* as_src[TM];
    int64_t bs_at[TN];
#pragma unroll
    for (int i = 0; i < TM; ++i) {
        const int r = m0 + i * 16 + frow < row_end ? m0 + i * 16 + frow : row_end - 1;
        int64_t row = r;
        if constexpr (Cfg::EXPERTS)
            if (p.gather) row = f8_token(p, p.order[r]);
        a_src[i] = p.A + row * p.a_rs + fg * 16;
        as_src[i] = p.a_scale + row * p.as_rs;
    }
#pragma unroll
    for (int j = 0; j < TN; ++j) {
        const int first = Cfg::GATED ? n0 + unit * 16 : n0 + (unit * TN + j) * 16;
        const int c = first + frow < p.N ? first + frow : p.N - 1;
        b_src[j] = B + (int64_t)c * p.b_cs + fg * 16 + (Cfg::GATED && j == 1 ? p.b_up : 0);
        // (columns of one block of 16 share a group of 128)
        bs_at[j] = (Cfg::COLUMNS ? 0 : (int64_t)((first < p.N ? first : p.N - 1) >> 7) * p.bs_cs) + (Cfg::GATED && j == 1 ? p.bs_up : 0);
    }
    int64_t bs_col[Cfg::COLUMNS ? TN : 1][4];
    if constexpr (Cfg::COLUMNS) {
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int c = n0 + (unit * TN + j) * 16 + fg * 4 + e;
                bs_col[j][e] = (int64_t)(c < p.N ? c : p.N - 1) * p.bs_cs;
            }
    }

    // (a zero that the compiler takes for the lane's own: factors that are the same in all lanes come by vector loads, like the rest, in
    // the order of the loads; scalar ones come in any order, and waiting for one is waiting for all)
    int lane_zero;
    asm volatile("v_mov_b32 %0, 0" : "=v"(lane_zero));
#pragma unroll
    for (int j = 0; j < TN; ++j) bs_at[j] += lane_zero;

    f32x4 acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

    struct Block { // of K, on its way
        i32x4 a[TM][2], b[TN][2];
        float sa[TM];
        f32x4 sb[TN];
    };
    auto load = [&](Block& x, int kt) {
        const int64_t at = (int64_t)kt * F8_BLOCK;
#pragma unroll
        for (int j = 0; j < TN; ++j) {
            x.b[j][0] = *(const i32x4*)(b_src[j] + at);
            x.b[j][1] = *(const i32x4*)(b_src[j] + at + 64);
        }
#pragma unroll
        for (int i = 0; i < TM; ++i) {
            x.a[i][0] = *(const i32x4*)(a_src[i] + at);
            x.a[i][1] = *(const i32x4*)(a_src[i] + at + 64);
            x.sa[i] = as_src[i][kt * p.as_ks];
        }
#pragma unroll
        for (int j = 0; j < TN; ++j) {
            if constexpr (Cfg::COLUMNS) {
#pragma unroll
                for (int e = 0; e < 4; ++e) x.sb[j][e] = b_scale[bs_col[j][e] + kt * p.bs_ks];
            } else x.sb[j][0] = b_scale[bs_at[j] + kt * p.bs_ks];
        }
    };
    auto multiply = [&](const Block& x) {
        Fragment rows[TM], cols[TN];
#pragma unroll
        for (int i = 0; i < TM; ++i) rows[i].set(x.a[i][0], x.a[i][1]);
#pragma unroll
        for (int j = 0; j < TN; ++j) cols[j].set(x.b[j][0], x.b[j][1]);
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int j = 0; j < TN; ++j) {
                const f32x4 d = mfma_f8_block(cols[j], rows[i]);
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[i][j][e] = fmaf(d[e], x.sa[i] * x.sb[j][Cfg::COLUMNS ? e : 0], acc[i][j][e]);
            }
    };

    // whole blocks of K: slice, slice + KW, ...
    const int whole = p.K / F8_BLOCK, mine = (whole - slice + KW - 1) / KW;
    if (mine > 0) {
        Block ring[DEPTH];
        // workgroups start at different blocks: B's rows often lie a power of two apart, and with all of them at the same k a few memory
        // channels would have all the work
        const int turn = (int)(blockIdx.x % (unsigned)mine);
        auto block_of = [&](int n) {
            n = (n < mine ? n : mine - 1) + turn;
            return slice + (n < mine ? n : n - mine) * KW;
        };
#pragma unroll
        for (int d = 0; d < DEPTH; ++d) {
            load(ring[d], block_of(d));
            __builtin_amdgcn_sched_barrier(0);
        }
        int n = 0;
        for (; n + DEPTH < mine; n += DEPTH) {
#pragma unroll
            for (int d = 0; d < DEPTH; ++d) {
                multiply(ring[d]);
                load(ring[d], block_of(n + DEPTH + d));
                __builtin_amdgcn_sched_barrier(0); // (or all DEPTH are multiplied first, with nothing on the way)
            }
        }
#pragma unroll
        for (int d = 0; d < DEPTH; ++d)
            if (n + d < mine) multiply(ring[d]);
    }
    if (p.K % F8_BLOCK && slice == whole % KW) {
        // what is left of K: 16 bytes at a time where any of them is inside (rows are padded to 16), zeros behind it
        Block x;
        const int64_t at = (int64_t)whole * F8_BLOCK;
        const int left = p.K % F8_BLOCK;
        auto piece = [&](const uint8_t* src, int h) {
            const int inside = left - (fg * 16 + h * 64);
            if (inside <= 0) return i32x4{0, 0, 0, 0};
            const i32x4 v = *(const i32x4*)(src + at + h * 64);
            return inside < 16 ? f8_cut16(v, inside) : v;
        };
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int j = 0; j < TN; ++j) x.b[j][h] = piece(b_src[j], h);
#pragma unroll
            for (int i = 0; i < TM; ++i) x.a[i][h] = piece(a_src[i], h);
        }
#pragma unroll
        for (int i = 0; i < TM; ++i) x.sa[i] = as_src[i][whole * p.as_ks];
#pragma unroll
        for (int j = 0; j < TN; ++j) {
            if constexpr (Cfg::COLUMNS) {
#pragma unroll
                for (int e = 0; e < 4; ++e) x.sb[j][e] = b_scale[bs_col[j][e] + whole * p.bs_ks];
            } else x.sb[j][0] = b_scale[bs_at[j] + whole * p.bs_ks];
        }
        multiply(x);
    }

    if constexpr (KW > 1) {
        if (slice > 0) {
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
                for (int j = 0; j < TN; ++j) parts[((slice - 1) * Cfg::CW + unit) * TM * TN + i * TN + j][lane] = acc[i][j];
        }
        __syncthreads();
        if (slice == 0) {
#pragma unroll
            for (int s = 0; s < KW - 1; ++s)
#pragma unroll
                for (int i = 0; i < TM; ++i)
#pragma unroll
                    for (int j = 0; j < TN; ++j) acc[i][j] += parts[(s * Cfg::CW + unit) * TM * TN + i * TN + j][lane];
        }
    }
    if constexpr (Cfg::GATED) {
        const int c = n0 + unit * 16 + fg * 4;
        f32x4 h[TM];
        if (slice == 0) {
#pragma unroll
            for (int i = 0; i < TM; ++i) {
                unsigned top = 0;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    h[i][e] = c + e < p.N ? silu_mul(acc[i][0][e], acc[i][1][e]) : 0.f;
                    top = max(top, __float_as_uint(h[i][e]) & 0x7fffffffu);
                }
                top = f8_max_over(top, 16);
                top = f8_max_over(top, 32);
                if (fg == 0) tops[unit][i * 16 + frow] = top;
            }
        }
        __syncthreads();
        if (slice == 0) {
#pragma unroll
            for (int i = 0; i < TM; ++i) {
                unsigned top = 0;
#pragma unroll
                for (int u = 0; u < 8; ++u) top = max(top, tops[u][i * 16 + frow]);
                const int r = m0 + i * 16 + frow;
                if (r >= row_end) continue;
                const float s = f8_scale_of(__uint_as_float(top), true), inv = f8_inverse_of(s, true);
                // (rows of codes are padded to 16, so that the four bytes are the row's own)
                if (c < p.N) *(unsigned*)((uint8_t*)p.C + (int64_t)r * p.c_rs + c) = f8_pack4(h[i][0] * inv, h[i][1] * inv, h[i][2] * inv, h[i][3] * inv);
                if (unit == 0 && fg == 0) p.out_scale[(int64_t)r * p.os_rs + (int64_t)(n0 >> 7) * p.os_bs] = s;
            }
        }
        return;
    }
    if (slice > 0) return;
    const bool relu = p.epilogue == EPI_RELU;
    const int os = p.out_type == T_F32 ? 4 : 2;
    const bool vec = (p.c_rs * os) % (4 * os) == 0 && ((size_t)p.C & (4 * os - 1)) == 0;
#pragma unroll
    for (int i = 0; i < TM; ++i) {
        const int r = m0 + i * 16 + frow;
        if (r >= row_end) continue;
        float w = 1.f;
        if constexpr (Cfg::EXPERTS)
            if (p.row_weights) w = p.row_weights[p.order[r]];
        char* row = (char*)p.C + (int64_t)r * p.c_rs * os;
#pragma unroll
        for (int j = 0; j < TN; ++j) {
            const int c = n0 + (unit * TN + j) * 16 + fg * 4;
            f32x4 v = acc[i][j];
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = (relu ? (v[e] > 0.f ? v[e] : 0.f) : v[e]) * w;
            f8_store4(row, p.out_type, c, p.N, v, vec);
        }
    }
}

template <typename Cfg>
hipError_t launch_f8_few(const F8GemmArgs& a, hipStream_t s)
{
    const int64_t tiles_n = (a.N + Cfg::BN - 1) / Cfg::BN;
    const int64_t tiles_m = Cfg::EXPERTS ? a.M / Cfg::BM + (a.experts < a.M ? a.experts : a.M) : (a.M + Cfg::BM - 1) / Cfg::BM;
    if (tiles_m * tiles_n > 0x7fffffffll) return hipErrorInvalidConfiguration;
    f8_gemm_few_kernel<Cfg><<<dim3((unsigned)(tiles_m * tiles_n)), dim3(Cfg::NT), 0, s>>>(a);
    return hipGetLastError();
}

} // namespace acc950
