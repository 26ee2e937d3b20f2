// Block-scaled e4m3 product on LDS tiles: A and B contiguous along K, rows on 16-byte boundaries.
//
//   C[i, j] = sum over blocks b of 128 of a_scale[i, b] * b_scale[b, j] * (A[i, b] . B[b, j])
//
// A K tile is one block: a matrix instruction per 16 x 16 results and block, from zero, and its four results per lane are scaled
// and added to the sums by vector instructions.  That is what shapes the kernels: the sums have to lie where vector instructions reach
// them (not in the accumulator file), so a wave has at most 128 x 64 of them.
//
// Here: tiles of 128x128 (two workgroups to a CU, so that one computes while the other starts or writes back) and 64x64 (four, or two with four stages
// for a short wait at the start); f8_gemm_pp.h has the 256x256 ones.  With 64x64 of a tile to a wave its fragments' way out of LDS (1024 cycles to a
// block of K and CU) takes as long as the matrix instructions: 4096^3 to bf16 75 us, 1.84 PFLOP/s.  The wide form is bound by the instructions that
// a wave can issue (64 matrix ones, 128 to widen, 80 to 128 to scale, to a block): 4096x11008x2048 to fp32 180 us, 1.0 PFLOP/s.
#pragma once
#include "f8.h"

namespace acc950 {

// WIDE: see F8Fragment.  COLUMNS: b_scale has a factor for every column (else one per 128).  EXPERTS: rows come from a plan.
// GATED: half of the tile's columns are of the gate matrix, half the same ones of the up matrix, and the result is silu(gate) * up as
// codes and scales: a tile has 128 of the inner values, one group of every row.
template <int BM_, int BN_, int WAVES_M_, int WAVES_N_, int STAGES_, bool WIDE_, bool COLUMNS_, bool EXPERTS_, bool GATED_ = false>
struct F8TileConfig {
    static constexpr bool GATED = GATED_;
    static constexpr int OUT_N = GATED ? BN_ / 2 : BN_; // columns of the result that a tile makes
    static_assert(!GATED || (BN_ == 256 && EXPERTS_ && !COLUMNS_), "one group of 128 inner values");
    static constexpr int BM = BM_, BN = BN_, WAVES_M = WAVES_M_, WAVES_N = WAVES_N_, STAGES = STAGES_;
    static constexpr bool WIDE = WIDE_, COLUMNS = COLUMNS_, EXPERTS = EXPERTS_;
    static constexpr int NW = WAVES_M * WAVES_N, NT = NW * 64;
    static constexpr int A_BYTES = BM * F8_BLOCK, B_BYTES = BN * F8_BLOCK, S_BYTES = (BM + BN) * 4;
    static constexpr int STAGE_BYTES = A_BYTES + B_BYTES + S_BYTES, LDS_BYTES = STAGES * STAGE_BYTES;
    static constexpr int WGS_PER_CU = 2 * LDS_BYTES <= 160 * 1024 && NW <= 4 ? 2 : 1;
    static_assert(LDS_BYTES <= 160 * 1024 && NW * 2304 <= LDS_BYTES, "LDS of one CU; slabs of the write-back");
    static_assert((BM * 8) % NT == 0 && (BN * 8) % NT == 0, "fills are whole");
};

// 16-byte chunk c of a row of 128 bytes lies at position c ^ (row & 7).  The four lanes of a fragment's row read chunks 0 to 3 and then 4 to 7:
// no two lanes in one bank, 4.1 cycles to a read of 1 KB (neighbouring chunks to a lane, 0 2 4 6 and then 1 3 5 7, took 6.8).
__device__ __forceinline__ int f8_chunk(int row, int c) { return c ^ (row & 7); }

// Straight from memory into LDS: lane l's 16 (4) bytes go to lds + 16 l (4 l); both base addresses are the same in all lanes.
// A memory instruction may read a scalar register five instructions after a vector instruction has written it, no sooner (the compiler brings back spilled
// ones with v_readlane, and does not look into inline assembly): the address is copied by the scalar unit, which waits by itself, and the copy stands where
// m0 needs an instruction behind it anyway.
__device__ __forceinline__ void fill_b128(unsigned lds, unsigned off, const void* base)
{
    const void* at;
    asm volatile("s_mov_b32 m0, %1\n\ts_mov_b64 %0, %3\n\tglobal_load_lds_dwordx4 %2, %0" : "=&s"(at) : "s"(lds), "v"(off), "s"(base) : "memory");
}
__device__ __forceinline__ void fill_b32(unsigned lds, unsigned off, const void* base)
{
    const void* at;
    asm volatile("s_mov_b32 m0, %1\n\ts_mov_b64 %0, %3\n\tglobal_load_lds_dword %2, %0" : "=&s"(at) : "s"(lds), "v"(off), "s"(base) : "memory");
}
// All but the last N of the wave's fills have landed and its reads of LDS are done, in every wave.
template <int N>
__device__ __forceinline__ void f8_tile_barrier() { asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory"); }

// The order of tiles.  Workgroup ids go round the 8 XCDs; an XCD has a run of neighbouring tiles of its own, so that what its workgroups do at a
// time shares A and B through its L2.  The n-th tile of workgroup `id` (-1: there is none) of `total`, with `ids` workgroups that each take
// several:
__device__ __forceinline__ int f8_nth_tile(int id, int ids, int n, int total)
{
    constexpr int XCDS = 8;
    if (ids % XCDS) return id + n * ids < total ? id + n * ids : -1;
    const int xcd = id % XCDS, each = total / XCDS, more = total % XCDS;
    const int size = each + (xcd < more), local = id / XCDS + n * (ids / XCDS);
    return local < size ? xcd * each + (xcd < more ? xcd : more) + local : -1;
}
// The same by tickets, for tiles that cost more and less: the first tiles as above, the others of an XCD's run to whoever is free first, and
// when its own run is done a workgroup takes from the other XCDs'.  One thread calls it; `tickets`: 8 counters, zero at the launch.  (Which
// workgroup computes a tile has no part in its result.)
__device__ __forceinline__ int f8_tile_by_ticket(int id, int ids, int total, int* tickets)
{
    constexpr int XCDS = 8;
    const int each = total / XCDS, more = total % XCDS;
    for (int s = 0; s < XCDS; ++s) {
        const int xcd = (id + s) % XCDS, size = each + (xcd < more);
        if (size <= ids / XCDS) continue; // (all of them first tiles)
        const int local = ids / XCDS + atomicAdd(tickets + xcd, 1);
        if (local < size) return xcd * each + (xcd < more ? xcd : more) + local;
    }
    return -1;
}
// Tiles of a plain product are walked in bands of 4 rows of them: a run is a compact rectangle.
__device__ __forceinline__ void f8_tile_coords(int t, int tiles_m, int tiles_n, int& tm, int& tn)
{
    constexpr int BAND = 4;
    const int per_band = BAND * tiles_n, band = t / per_band, first = band * BAND, rows = tiles_m - first < BAND ? tiles_m - first : BAND;
    tm = first + t % per_band % rows;
    tn = t % per_band / rows;
}

// the first `inside` (1 to 15) bytes of 16, zeros behind them
__device__ __forceinline__ i32x4 f8_cut16(i32x4 v, int inside)
{
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        const int bytes = inside - w * 4;
        v[w] = bytes >= 4 ? v[w] : bytes <= 0 ? 0 : v[w] & ((1 << bytes * 8) - 1);
    }
    return v;
}

// the low half of a product, and no more: with the addition behind it the compiler makes it a multiply-add of 64 bits, and keeps both halves
// of the result in registers for as long as the one that is used.  (b goes through the scalar unit first, as in fill_b128: a vector instruction needs two between)
__device__ __forceinline__ unsigned f8_mul32(unsigned a, unsigned b)
{
    unsigned d, copy;
    asm("s_mov_b32 %1, %3\n\tv_mul_lo_u32 %0, %2, %1" : "=v"(d), "=&s"(copy) : "v"(a), "s"(b));
    return d;
}

// A workgroup's tile of the result and how its operands are filled into LDS: wave w's f-th fill of an operand covers rows (f * NW + w) * 8 .. + 7
// of its tile, a lane one chunk.
template <typename Cfg>
struct F8Tile {
    static constexpr int BM = Cfg::BM, BN = Cfg::BN, NW = Cfg::NW, FA = BM * 8 / Cfg::NT, FB = BN * 8 / Cfg::NT;
    int m0, row_end, n0, KT, tail, total;
    const uint8_t *A, *B;
    const char* s_base;
    int64_t s_step, b_up;
    unsigned a_off[FA], b_off, b_step, s_off, s_lds; // (B's: of the first fill, and from one to the next)
    unsigned a_last, b_last; // offset of the last piece of the last row that the tile may read, of its last column

    __device__ __forceinline__ void count(const F8GemmArgs& p, int lane)
    {
        const int tiles_n = (p.N + Cfg::OUT_N - 1) / Cfg::OUT_N;
        total = tiles_n * (Cfg::EXPERTS ? count_expert_tiles(p.offsets, p.experts, p.rows_log2, lane) : (p.M + BM - 1) / BM);
    }
    // tile t of all (counted before); false: there is none
    __device__ __forceinline__ bool place(const F8GemmArgs& p, int lane, int wave, int t)
    {
        if (t < 0) return false;
        const int tiles_n = (p.N + Cfg::OUT_N - 1) / Cfg::OUT_N;
        int expert = 0;
        if constexpr (Cfg::EXPERTS) {
            int row0;
            if (!find_expert_tile(p.offsets, p.experts, p.rows_log2, tiles_n, lane, t, expert, row0, row_end)) return false;
            const int rows = 1 << p.rows_log2, tiles_m = (row_end - row0 + rows - 1) >> p.rows_log2;
            m0 = row0 + t % tiles_m * rows;
            row_end = min(row_end, m0 + rows);
            n0 = t / tiles_m * Cfg::OUT_N;
        } else {
            int tm, tn;
            f8_tile_coords(t, (p.M + BM - 1) / BM, tiles_n, tm, tn);
            m0 = tm * BM; row_end = p.M; n0 = tn * BN;
        }
        KT = (p.K + F8_BLOCK - 1) / F8_BLOCK;
        tail = p.K % F8_BLOCK;
        int first_block = 0;
        if (p.slices > 1) {
            first_block = blockIdx.z * p.slice_blocks;
            if ((int)blockIdx.z < p.slices - 1) { KT = p.slice_blocks; tail = 0; }
            else KT -= first_block;
        }
        const int first_k = first_block * F8_BLOCK;
        b_up = p.b_up;
        B = p.B + expert * p.b_es + (int64_t)n0 * p.b_cs + first_k;
        const float* b_scale = p.b_scale + expert * p.bs_es + (int64_t)(n0 >> p.group_shift) * p.bs_cs + first_block * p.bs_ks;
        // (of gathered rows offsets count from A's first, otherwise from the tile's)
        const bool gather = Cfg::EXPERTS && p.gather;
        A = p.A + (gather ? 0 : (int64_t)m0 * p.a_rs) + first_k;
        const float* a_scale = p.a_scale + (gather ? 0 : (int64_t)m0 * p.as_rs) + first_block * p.as_ks;
        auto a_row = [&](int r) { // row of the tile -> row of A from there on; rows behind the end are the last one again
            r = m0 + r < row_end ? r : row_end - 1 - m0;
            return (unsigned)(gather ? f8_token(p, p.order[m0 + r]) : r);
        };
        auto b_col = [&](int c) { // column of the tile -> column of B from n0 on (of the half that it is in)
            if constexpr (Cfg::GATED) c %= Cfg::OUT_N;
            return (unsigned)(n0 + c < p.N ? c : p.N - 1 - n0);
        };
        auto in_up = [&](int c) { return Cfg::GATED && c >= Cfg::OUT_N; };
        const int chunk = f8_chunk(lane >> 3, lane & 7); // (of 8 rows from a multiple of 8 on)
        const unsigned row_end_piece = (unsigned)(((p.K - 1) & ~15) - first_k);
        a_last = (unsigned)(gather ? f8_token(p, p.M - 1) : min(row_end - m0, BM) - 1) * (unsigned)p.a_rs + row_end_piece;
        b_last = (unsigned)(min(p.N - n0, Cfg::OUT_N) - 1) * (unsigned)p.b_cs + row_end_piece;
#pragma unroll
        for (int f = 0; f < FA; ++f) {
            a_off[f] = f8_mul32(a_row((f * NW + wave) * 8 + (lane >> 3)), (unsigned)p.a_rs) + chunk * 16;
        }
        b_off = f8_mul32(wave * 8 + (lane >> 3), (unsigned)p.b_cs) + chunk * 16;
        b_step = NW * 8 * (unsigned)p.b_cs;
        // factors: BM of A's rows, then BN of B's columns, 64 to a wave (waves with none of their own fetch others' again)
        const int first = wave * 64 % (BM + BN);
        const bool of_a = first < BM;
        s_lds = Cfg::A_BYTES + Cfg::B_BYTES + first * 4;
        s_off = of_a ? f8_mul32(a_row(first + lane), (unsigned)p.as_rs * 4)
                     : f8_mul32((unsigned)(((n0 + (int)b_col(first - BM + lane)) >> p.group_shift) - (n0 >> p.group_shift)), (unsigned)p.bs_cs * 4) +
                           (in_up(first - BM) ? (unsigned)p.bs_up * 4 : 0u);
        s_base = (const char*)(of_a ? a_scale : b_scale);
        s_step = 4 * (of_a ? p.as_ks : p.bs_ks);
        return true;
    }
    // Offset of B's f-th fill; columns behind the result's read some of its last one's, and what comes of them is not written.  (gated: the second
    // half of the columns is the up matrix's)
    static __device__ __forceinline__ bool up(int f) { return Cfg::GATED && f >= FB / 2; }
    __device__ __forceinline__ unsigned b_at(int f, unsigned last) const { return min(b_off + (up(f) ? f - FB / 2 : f) * b_step, last); }
    // (In the last block of K chunks behind its end are other rows', or the last piece there is: fetched, never used.)
    template <int F0, int F1>
    __device__ __forceinline__ void fill_a(int kt, unsigned at, int wave) const
    {
        const uint8_t* a = A + (int64_t)kt * F8_BLOCK;
        const unsigned last = a_last - kt * F8_BLOCK;
#pragma unroll
        for (int f = F0; f < F1; ++f) fill_b128(at + (f * NW + wave) * 1024, min(a_off[f], last), a);
    }
    __device__ __forceinline__ void fill_b(int kt, unsigned at, int wave) const
    {
        const uint8_t* b = B + (int64_t)kt * F8_BLOCK;
        const unsigned last = b_last - kt * F8_BLOCK;
#pragma unroll
        for (int f = 0; f < FB; ++f) fill_b128(at + Cfg::A_BYTES + (f * NW + wave) * 1024, b_at(f, last), up(f) ? b + b_up : b);
    }
    __device__ __forceinline__ void fill_s(int kt, unsigned at) const { fill_b32((unsigned)__builtin_amdgcn_readfirstlane((int)(at + s_lds)), s_off, s_base + kt * s_step); }
};

// Write-back of a wave's tile: lane l holds row l % 16 and columns (l / 16) * 4 .. + 3 of every block of 16 x 16.  The rows of a block are put
// together in the wave's own slab of LDS (F8_SLAB bytes), 16 rows of 16-bit values or twice 8 of fp32, and leave as 16-byte pieces of
// whole rows, or one value by one.  row0(i): first row, in the tile, of the wave's i-th blocks.
constexpr int F8_SLAB = 16 * (64 * 2 + 16);
template <typename Cfg, int TM, int TN, typename Row0>
__device__ __forceinline__ void f8_write_tile(const F8GemmArgs& p, f32x4 (&acc)[TM][TN], int m0, int row_end, int n0, Row0&& row0, int wc0, int lane, char* slab)
{
    constexpr int WTN = TN * 16;
    static_assert(WTN <= 64, "a slab's rows");
    const int frow = lane & 15, fg = lane >> 4;
    const bool part = p.slices > 1, relu = !part && p.epilogue == EPI_RELU, f32 = part || p.out_type == T_F32;
    const bool scaled = Cfg::EXPERTS && p.out_scale; // (fp16, see F8GemmArgs)
    const bool whole = n0 + Cfg::OUT_N <= p.N;
    const int os = f32 ? 4 : 2, type = f32 ? T_F32 : p.out_type;
    char* const C = part ? (char*)(p.parts + (int64_t)blockIdx.z * p.M * p.parts_rs) : (char*)p.C;
    const int64_t c_rs = part ? p.parts_rs : p.c_rs;
    const bool vec = (c_rs * os) % 16 == 0 && ((size_t)C & 15) == 0;
    float weight[Cfg::EXPERTS ? TM : 1]; // (all asked for at once: two trips to memory, not two for every 16 rows)
    if constexpr (Cfg::EXPERTS) {
#pragma unroll
        for (int i = 0; i < TM; ++i) weight[i] = 1.f;
        if (p.row_weights) {
            int pair[TM];
#pragma unroll
            for (int i = 0; i < TM; ++i) pair[i] = m0 + row0(i) + frow < row_end ? p.order[m0 + row0(i) + frow] : -1;
#pragma unroll
            for (int i = 0; i < TM; ++i) weight[i] = pair[i] >= 0 ? p.row_weights[pair[i]] : 1.f;
        }
    }
#pragma unroll
    for (int i = 0; i < TM; ++i) {
        if (Cfg::EXPERTS && m0 + row0(i) >= row_end) continue;
        const int r = m0 + row0(i) + frow;
        float w = 1.f;
        if constexpr (Cfg::EXPERTS) w = weight[i];
        auto ended = [&](int j) {
            f32x4 v = acc[i][j];
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = Cfg::EXPERTS ? v[e] * w : relu ? (v[e] > 0.f ? v[e] : 0.f) : v[e];
            return v;
        };
        if constexpr (Cfg::EXPERTS) {
            if (scaled) {
                // the wave's columns of a row: their largest magnitude to 2^14 .. 2^15
                float top = 0.f; // (NaN aside: it stays what it is)
#pragma unroll
                for (int j = 0; j < TN; ++j) {
                    if (!whole) {
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (n0 + wc0 + j * 16 + fg * 4 + e >= p.N) acc[i][j][e] = 0.f;
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e) top = fmaxf(top, fabsf(acc[i][j][e]));
                }
                const unsigned bits = f8_max_over(f8_max_over(__float_as_uint(top), 16), 32);
                // (an exponent's power of two and its inverse, both normal; infinities and NaN stay what they are)
                const int e = min(max((int)(bits >> 23), 16), 254);
                w = __uint_as_float((unsigned)(268 - e) << 23);
                if (fg == 0 && r < row_end && n0 + wc0 < p.N) {
                    float* const at = p.out_scale + (int64_t)r * p.os_rs + ((n0 + wc0) >> 5);
                    const float down = __uint_as_float((unsigned)(e - 14) << 23);
                    if constexpr (TN == 4) *(float2*)at = float2{down, down}; // (rows of factors are padded to pairs)
                    else *at = down;
                }
            }
        }
        auto out = [&](auto os_tag) {
            constexpr int OS = decltype(os_tag)::value, AT_ONCE = 32 / OS, PITCH = WTN * OS + 16, LANES = WTN * OS / 16, ROWS = 64 / LANES, PER = 16 / OS; // lanes to a row
            static_assert(AT_ONCE * PITCH <= F8_SLAB, "fits the slab");
#pragma unroll
            for (int h = 0; h < 16 / AT_ONCE; ++h) {
                if (frow / AT_ONCE == h) {
#pragma unroll
                    for (int j = 0; j < TN; ++j) f8_store4(slab + frow % AT_ONCE * PITCH, type, j * 16 + fg * 4, WTN, ended(j), true);
                }
                // (a wave's accesses to LDS stay in order by themselves; the compiler has to be told that what a lane reads others have written)
                asm volatile("" ::: "memory");
                // rows that do not start on 16 bytes: value by value, a row's side by side (4096x4095 from K = 1024 to bf16 34 us; a lane's own
                // four of 16 rows 49)
                if (!vec) {
                    using Value = std::conditional_t<OS == 4, float, uint16_t>;
                    constexpr int BESIDE = 64 / WTN;
#pragma unroll
                    for (int q = 0; q < AT_ONCE / BESIDE; ++q) {
                        const int row = q * BESIDE + lane / WTN, at = m0 + row0(i) + h * AT_ONCE + row, c = n0 + wc0 + lane % WTN;
                        const Value v = *(const Value*)(slab + row * PITCH + lane % WTN * OS);
                        if (at < row_end && c < p.N) ((Value*)C)[(int64_t)at * c_rs + c] = v;
                    }
                    asm volatile("" ::: "memory");
                    continue;
                }
#pragma unroll
                for (int q = 0; q < AT_ONCE / ROWS; ++q) {
                    const int row = q * ROWS + lane / LANES, piece = lane % LANES, at = m0 + row0(i) + h * AT_ONCE + row, c = n0 + wc0 + piece * PER;
                    const i32x4 v = *(const i32x4*)(slab + row * PITCH + piece * 16);
                    if (at >= row_end || c >= p.N) continue;
                    char* dst = C + ((int64_t)at * c_rs + c) * OS;
                    if (c + PER <= p.N) {
                        // (past the caches, whose lines are the operands': fp16 4096^2 from K = 1024 28 -> 25.5 us; experts' rows are read back at once)
                        if constexpr (Cfg::EXPERTS) *(i32x4*)dst = v;
                        else __builtin_nontemporal_store(v, (i32x4*)dst);
                    } else
                        for (int e = 0; e < p.N - c; ++e) {
                            if constexpr (OS == 4) ((int*)dst)[e] = v[e];
                            else ((uint16_t*)dst)[e] = (uint16_t)((unsigned)v[e / 2] >> (e % 2 * 16));
                        }
                }
                asm volatile("" ::: "memory");
            }
        };
        if (f32) out(std::integral_constant<int, 4>{});
        else out(std::integral_constant<int, 2>{});
    }
}

// Ending of a gate and up product: inner values, their rows' largest magnitude over the tile's 128, codes and scales.  `place`: F8_GATED_LDS bytes.
template <typename Cfg> constexpr int F8_GATED_LDS = Cfg::WAVES_N * Cfg::BM * 4 + 128 * (128 + 16);
template <typename Cfg, int TM, int TN, typename Row0>
__device__ __forceinline__ void f8_finish_gated(const F8GemmArgs& p, f32x4 (&acc)[TM][TN], int m0, int row_end, int n0, Row0&& row0, int wc0, int wave_n, int frow, int fg, int thread, char* place)
{
    constexpr int BM = Cfg::BM, WN = Cfg::WAVES_N, PITCH = 128 + 16, PASSES = BM / 128, TP = TM / PASSES; // 128 rows of codes at a time
    const bool whole = n0 + Cfg::OUT_N <= p.N;
    unsigned* tops = (unsigned*)place; // [WN][BM]; the codes behind
    char* codes = place + WN * BM * 4;
#pragma unroll
    for (int i = 0; i < TM; ++i) {
        if (m0 + row0(i) >= row_end) continue;
        unsigned top = 0;
#pragma unroll
        for (int j = 0; j < TN / 2; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                float h = silu_mul_to_code(acc[i][j][e], acc[i][j + TN / 2][e]);
                if (!whole && n0 + wc0 + j * 16 + fg * 4 + e >= p.N) h = 0.f;
                acc[i][j][e] = h;
                top = max(top, __float_as_uint(h) & 0x7fffffffu);
            }
        top = f8_max_over(top, 16);
        top = f8_max_over(top, 32);
        if (fg == 0) tops[wave_n * BM + row0(i) + frow] = top;
    }
    __syncthreads();
#pragma unroll
    for (int pass = 0; pass < PASSES; ++pass) {
        if (m0 + pass * 128 >= row_end) break;
#pragma unroll
        for (int i = pass * TP; i < (pass + 1) * TP; ++i) { // (the i-th blocks of the pass lie in rows pass * 128 .. + 127)
            const int row = row0(i) + frow, r = m0 + row;
            unsigned top = 0;
#pragma unroll
            for (int w = 0; w < WN; ++w) top = max(top, tops[w * BM + row]);
            const float s = f8_scale_of(__uint_as_float(top), true), inv = f8_inverse_of(s, true);
#pragma unroll
            for (int j = 0; j < TN / 2; ++j) {
                const f32x4 v = acc[i][j];
                *(unsigned*)(codes + (row - pass * 128) * PITCH + wc0 + j * 16 + fg * 4) = f8_pack4(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv);
            }
            if (wave_n == 0 && fg == 0 && r < row_end) p.out_scale[(int64_t)r * p.os_rs + (int64_t)(n0 >> 7) * p.os_bs] = s;
        }
        __syncthreads();
        // (rows of codes are padded to 16: pieces that begin before N are the row's own)
        for (int u = thread; u < 128 * 8; u += Cfg::NT) {
            const int row = u >> 3, c = (u & 7) * 16, r = m0 + pass * 128 + row;
            if (r < row_end && n0 + c < p.N) *(i32x4*)((uint8_t*)p.C + (int64_t)r * p.c_rs + n0 + c) = *(const i32x4*)(codes + row * PITCH + c);
        }
        if (pass + 1 < PASSES) __syncthreads();
    }
}

template <typename Cfg>
__global__ void __launch_bounds__(Cfg::NT, Cfg::WGS_PER_CU * Cfg::NW / 4) f8_gemm_tile_kernel(F8GemmArgs p)
{
    constexpr int BM = Cfg::BM, BN = Cfg::BN, NW = Cfg::NW, NT = Cfg::NT, STAGES = Cfg::STAGES;
    constexpr int WTM = BM / Cfg::WAVES_M, WTN = BN / Cfg::WAVES_N, TM = WTM / 16, TN = WTN / 16;
    constexpr int FILLS = F8Tile<Cfg>::FA + F8Tile<Cfg>::FB + 1;
    using Fragment = F8Fragment<Cfg::WIDE>;
    extern __shared__ __attribute__((aligned(1024))) char smem[];

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    F8Tile<Cfg> tile;
    tile.count(p, lane);
    if (!tile.place(p, lane, wave, f8_nth_tile(blockIdx.x, gridDim.x, 0, tile.total))) return;
    const int m0 = tile.m0, row_end = tile.row_end, n0 = tile.n0, KT = tile.KT, tail = tile.tail;
    const unsigned lds0 = (unsigned)(size_t)(ACC950_LDS char*)smem;
    auto fill = [&](int kt, int stage) {
        const unsigned at = lds0 + stage * Cfg::STAGE_BYTES;
        tile.fill_b(kt, at, wave);
        tile.template fill_a<0, F8Tile<Cfg>::FA>(kt, at, wave);
        tile.fill_s(kt, at);
    };

    // ---- one K tile
    const int wr0 = wave / Cfg::WAVES_N * WTM, wc0 = wave % Cfg::WAVES_N * WTN;
    static_assert(!Cfg::GATED, "the kernel whose waves take turns has that");
    const int frow = lane & 15, fg = lane >> 4;
    f32x4 acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    auto read_fragment = [&](Fragment& f, const char* operand, int row0) {
        const char* row = operand + (row0 + frow) * F8_BLOCK;
        // (rows row0 .. + 15, row0 a multiple of 16: their places depend on the lane alone)
        f.set(*(const i32x4*)(row + f8_chunk(frow, fg) * 16), *(const i32x4*)(row + f8_chunk(frow, fg + 4) * 16));
    };
    auto multiply = [&](int stage) {
        const char *sa = smem + stage * Cfg::STAGE_BYTES, *sb = sa + Cfg::A_BYTES;
        const float* factors = (const float*)(sb + Cfg::B_BYTES);
        Fragment cols[TN];
        f32x4 col_factor[Cfg::COLUMNS ? TN : 1];
        float factor = 0.f;
        if constexpr (Cfg::COLUMNS) {
#pragma unroll
            for (int j = 0; j < TN; ++j) col_factor[j] = *(const f32x4*)(factors + BM + wc0 + j * 16 + fg * 4);
        } else factor = factors[BM + wc0];
#pragma unroll
        for (int j = 0; j < TN; ++j) read_fragment(cols[j], sb, wc0 + j * 16);
        auto add = [&](f32x4& sum, const f32x4& d, float row_factor, int j) {
            if constexpr (Cfg::COLUMNS) {
#pragma unroll
                for (int e = 0; e < 4; ++e) sum[e] = fmaf(d[e] * row_factor, col_factor[j][e], sum[e]);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) sum[e] = fmaf(d[e], row_factor * factor, sum[e]);
            }
        };
        if constexpr (!Cfg::WIDE) {
#pragma unroll
            for (int i = 0; i < TM; ++i) {
                Fragment rows;
                read_fragment(rows, sa, wr0 + i * 16);
                const float row_factor = factors[wr0 + i * 16 + frow];
#pragma unroll
                for (int j = 0; j < TN; ++j) add(acc[i][j], mfma_f8_block(cols[j], rows), row_factor, j);
            }
        } else {
            // Beside a step's matrix instructions stand the additions of the rows before and the widening of the rows behind: the order is held here, for the
            // compiler puts them behind one another.
            Fragment rows[2];
            read_fragment(rows[0], sa, wr0);
            f32x4 d[2][TN];
            float row_factor[2];
#pragma unroll
            for (int i = 0; i <= TM; ++i) {
                i32x4 lo, hi;
                if (i < TM) row_factor[i & 1] = factors[wr0 + i * 16 + frow];
                if (i + 1 < TM) {
                    const char* row = sa + (wr0 + (i + 1) * 16 + frow) * F8_BLOCK;
                    lo = *(const i32x4*)(row + f8_chunk(frow, fg) * 16);
                    hi = *(const i32x4*)(row + f8_chunk(frow, fg + 4) * 16);
                }
#pragma unroll
                for (int s = 0; s < 4; ++s) {
                    if (i < TM)
#pragma unroll
                        for (int j = 0; j < TN; ++j) d[i & 1][j] = mfma_f8_step(cols[j], rows[i & 1], s, s == 0 ? f32x4{0.f, 0.f, 0.f, 0.f} : d[i & 1][j]);
                    if (i > 0)
#pragma unroll
                        for (int j = s * TN / 4; j < (s + 1) * TN / 4; ++j) add(acc[i - 1][j], d[1 - (i & 1)][j], row_factor[1 - (i & 1)], j);
                    if (i + 1 < TM) rows[1 - (i & 1)].set_step(s, lo, hi);
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
        }
    };

    constexpr int AHEAD = STAGES - 1;
#pragma unroll
    for (int s = 0; s < AHEAD; ++s)
        if (s < KT) fill(s, s);
    for (int kt = 0; kt < KT; ++kt) {
        // own fills of this tile have landed (younger ones may be on the way); behind the barrier everyone's have, and everyone is done
        // with the tile whose place the next fill takes
        if (kt + AHEAD <= KT) f8_tile_barrier<(AHEAD - 1) * FILLS>();
        else f8_tile_barrier<0>();
        if (kt + AHEAD < KT) fill(kt + AHEAD, (kt + AHEAD) % STAGES);
        if (tail && kt == KT - 1) {
            char* last = smem + kt % STAGES * Cfg::STAGE_BYTES;
            for (int i = tid; i < (BM + BN) * 8; i += NT) {
                const int row = i >> 3, c = i & 7, left = tail - c * 16; // A's rows, then B's: BM is a multiple of 16
                if (left >= 16) continue;
                i32x4* at = (i32x4*)(last + row * F8_BLOCK + f8_chunk(row, c) * 16);
                *at = left > 0 ? f8_cut16(*at, left) : i32x4{0, 0, 0, 0};
            }
            __syncthreads();
        }
        multiply(kt % STAGES);
    }

    f8_tile_barrier<0>(); // everyone is done with the tiles: their place is the slabs' now
    f8_write_tile<Cfg, TM, TN>(p, acc, m0, row_end, n0, [&](int i) { return wr0 + i * 16; }, wc0, lane, smem + wave * F8_SLAB);
}

// Workgroups of a launch.  (Experts: all their tiles together are at most one more for each expert with rows than the rows alone would make.)
template <typename Cfg>
int64_t f8_tiles(const F8GemmArgs& a)
{
    const int64_t tiles_n = (a.N + Cfg::OUT_N - 1) / Cfg::OUT_N;
    return tiles_n * (Cfg::EXPERTS ? (a.M >> a.rows_log2) + (a.experts < a.M ? a.experts : a.M) : (a.M + Cfg::BM - 1) / Cfg::BM);
}

template <typename Cfg>
hipError_t launch_f8_tile(F8GemmArgs a, hipStream_t s)
{
    a.rows_log2 = __builtin_ctz(Cfg::BM);
    static LdsLimitOnce lds_limit;
    const hipError_t e = lds_limit.ensure((const void*)f8_gemm_tile_kernel<Cfg>, Cfg::LDS_BYTES);
    if (e != hipSuccess) return e;
    const int64_t tiles = f8_tiles<Cfg>(a);
    if (tiles > 0x7fffffffll) return hipErrorInvalidConfiguration;
    f8_gemm_tile_kernel<Cfg><<<dim3((unsigned)tiles, 1, a.slices > 1 ? a.slices : 1), dim3(Cfg::NT), Cfg::LDS_BYTES, s>>>(a);
    return hipGetLastError();
}

} // namespace acc950
