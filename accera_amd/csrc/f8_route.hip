// Routing to experts: scores, choice and weights of a token (a wave or a quarter of one), their gradient, the order of the pairs by expert,
// and the weighted sum of a token's rows.  All of it moves little data; what counts is the number of dependent steps.
#include "f8_quantize.h"

namespace acc950 {
namespace {

constexpr int MAX_EXPERTS = 1024;

__device__ __forceinline__ float load_logit(const void* x, int type, int64_t i) { return load_out(x, type, i); }
__device__ __forceinline__ f32x4 load_logits(const void* x, int type, int64_t i) // four from a multiple of their size on
{
    if (type == T_F32) return *(const f32x4*)((const float*)x + i);
    const uint2 v = *(const uint2*)((const uint16_t*)x + i);
    const unsigned h[4] = {v.x & 0xffff, v.x >> 16, v.y & 0xffff, v.y >> 16};
    f32x4 r;
#pragma unroll
    for (int e = 0; e < 4; ++e) r[e] = type == T_F16 ? f16_bits_to_float((uint16_t)h[e]) : bf16_bits_to_float((uint16_t)h[e]);
    return r;
}

// Reductions over the wave by DPP moves (a shuffle goes through the LDS unit, ten times the latency): shifts within rows of 16 lanes, then lane 15
// and lane 31 into the rows behind; the last lane has the result.
template <int CTRL, int ROWS>
__device__ __forceinline__ unsigned dpp_from(unsigned v) { return (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xf, false); }
template <typename Op>
__device__ __forceinline__ unsigned wave_reduce(unsigned v, Op&& op) // (0 is neutral)
{
    v = op(v, dpp_from<0x111, 0xf>(v)); // row_shr:1, 2, 4, 8
    v = op(v, dpp_from<0x112, 0xf>(v));
    v = op(v, dpp_from<0x114, 0xf>(v));
    v = op(v, dpp_from<0x118, 0xf>(v));
    v = op(v, dpp_from<0x142, 0xa>(v)); // row_bcast:15 into rows 1 and 3
    v = op(v, dpp_from<0x143, 0xc>(v)); // row_bcast:31 into rows 2 and 3
    return (unsigned)__builtin_amdgcn_readlane((int)v, 63);
}
__device__ __forceinline__ unsigned wave_max_u(unsigned v) { return wave_reduce(v, [](unsigned a, unsigned b) { return max(a, b); }); }
__device__ __forceinline__ float wave_sum(float v)
{
    return __uint_as_float(wave_reduce(__float_as_uint(v), [](unsigned a, unsigned b) { return __float_as_uint(__uint_as_float(a) + __uint_as_float(b)); }));
}

// Floats as unsigned integers in the same order, NaN above infinity, -0 like +0; 0 is below all of them (used for "not to be taken").
__device__ __forceinline__ unsigned order_bits(float v)
{
    if (v != v) return 0xffffffffu;
    if (v == 0.f) v = 0.f;
    const unsigned b = __float_as_uint(v);
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float of_order_bits(unsigned u) { return u == 0xffffffffu ? NAN : __uint_as_float((u & 0x80000000u) ? (u & 0x7fffffffu) : ~u); }

// Scores of the token's experts; lane l holds experts l, l + 64, ...  (softmax: exp(x - max) / sum.)  A row without any expert
// left has scores 0.
template <int VPL>
__device__ __forceinline__ void scores_of(float (&x)[VPL], float (&p)[VPL], int experts, int score, int lane)
{
    if (score == ACC950_SCORE_SIGMOID) {
#pragma unroll
        for (int j = 0; j < VPL; ++j) p[j] = 1.f / (1.f + expf(-x[j]));
        return;
    }
    float top = -INFINITY; // (of the numbers: a NaN reaches every score through the sum)
#pragma unroll
    for (int j = 0; j < VPL; ++j) top = fmaxf(top, x[j]);
    top = of_order_bits(wave_max_u(order_bits(top)));
    if (top == -INFINITY) top = 0.f;
    float sum = 0.f;
#pragma unroll
    for (int j = 0; j < VPL; ++j) {
        p[j] = expf(x[j] - top);
        sum += p[j];
    }
    sum = wave_sum(sum);
    if (sum == 0.f) sum = 1.f;
#pragma unroll
    for (int j = 0; j < VPL; ++j) p[j] = p[j] / sum;
}

// Scores taken that are this small altogether, which a bias may lead to, have few or no bits left (fp32 ends at 2^-126); renormalised they are then worked out again beside the
// largest of them: softmax's are exp(x) times something that all share, and so are sigmoid's, to 2^-90 of themselves.
constexpr float SCORES_LOST = 0x1p-90f;

// ---- the choice -----------------------------------------------------------------------------------
// L lanes to a token, VPL experts to a lane.  Bound by the instructions: 16384x256 in groups reads 16.8 MB (3.2 us) and takes 15 us, a third of it the
// sigmoids, exact to the last place (expf, IEEE division), for a choice must not hang on a faster one's rounding.  What is chosen from is kept as doubles: the fp32 value exactly, and in the low bits, which a float leaves
// zero, the expert, so that the lowest of equal values is the largest key and no two keys are the same.  A choice is then one maximum over all keys, and
// its expert's is taken out, with no search for who had it.
constexpr int NO_KEY = (int)0xffefffff, INF_KEY = 0x7fe00000, NAN_KEY = 0x7fe80000; // high words: nothing to choose, infinity, NaN above it (all finite doubles)

__device__ __forceinline__ int high_word(double d) { return __double2hiint(d); }
__device__ __forceinline__ double with_high(double d, int hi) { return __hiloint2double(hi, __double2loint(d)); }
__device__ __forceinline__ double no_key() { return __hiloint2double(NO_KEY, 0); }
__device__ __forceinline__ double key_of(float v, int at)
{
    const bool nan = v != v;
    const double d = (double)((nan ? INFINITY : v) + 0.f); // (-0 like +0)
    const int hi = nan ? NAN_KEY : min(high_word(d), INF_KEY);
    return __hiloint2double(hi, __double2loint(d) | (v < 0.f ? at : MAX_EXPERTS - 1 - at));
}
__device__ __forceinline__ int index_of_key(double d) { return high_word(d) < 0 ? __double2loint(d) & (MAX_EXPERTS - 1) : MAX_EXPERTS - 1 - (__double2loint(d) & (MAX_EXPERTS - 1)); }
__device__ __forceinline__ float value_of_key(double d) { return high_word(d) == NAN_KEY ? NAN : (float)d; } // (what lies below a float's last place rounds away)

// A group's key from its two best: their fp32 sum, or where that passes fp32's range (the type's lowest number as a mask, twice) their sum as a double, its last
// bits cleared for the group's number.  (An infinity below would lie under "nothing to choose", and with the number in its low bits be a NaN.)
__device__ __forceinline__ double key_of_sum(float best, float second, int at)
{
    const float sum = best + second;
    const double wide = (double)best + (double)second;
    if (fabsf(sum) < INFINITY || !(fabs(wide) < (double)INFINITY)) return key_of(sum, at);
    return __hiloint2double(__double2hiint(wide), (__double2loint(wide) & -MAX_EXPERTS) | (wide < 0 ? at : MAX_EXPERTS - 1 - at));
}

// over the L lanes of a token, the result in all of them: turns within rows of 16 lanes, then the four rows' by scalar registers
template <int L, typename T, typename Op>
__device__ __forceinline__ T over_lanes(T v, Op&& op)
{
    auto turned = [](T x, auto ctrl) {
        if constexpr (sizeof(T) == 8) asm volatile("s_nop 1" : "+v"(x)); // (a value that asm wrote: two waits before its lanes are moved)
        auto word = [](int w) { return __builtin_amdgcn_mov_dpp(w, decltype(ctrl)::value, 0xf, 0xf, true); };
        if constexpr (sizeof(T) == 4) return __int_as_float(word(__float_as_int(x)));
        else return __hiloint2double(word(__double2hiint(x)), word(__double2loint(x)));
    };
    v = op(v, turned(v, std::integral_constant<int, 0x128>{})); // row_ror:8, 4, 2, 1
    v = op(v, turned(v, std::integral_constant<int, 0x124>{}));
    v = op(v, turned(v, std::integral_constant<int, 0x122>{}));
    v = op(v, turned(v, std::integral_constant<int, 0x121>{}));
    if constexpr (L == 64) {
        auto row = [&](int lane) {
            if constexpr (sizeof(T) == 4) return __uint_as_float((unsigned)__builtin_amdgcn_readlane((int)__float_as_uint(v), lane));
            else return __hiloint2double(__builtin_amdgcn_readlane(__double2hiint(v), lane), __builtin_amdgcn_readlane(__double2loint(v), lane));
        };
        v = op(op(row(0), row(16)), op(row(32), row(48)));
    }
    return v;
}
// (no key is a NaN, which the compiler cannot know: __builtin_fmax would first turn each of its operands that it did not see computed into a quiet one)
__device__ __forceinline__ double larger(double a, double b)
{
    double r;
    asm("v_max_f64 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
    return r;
}
__device__ __forceinline__ double smaller(double a, double b)
{
    double r;
    asm("v_min_f64 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
    return r;
}

// A lane's experts lie in one group: so many lanes (a power of two) to a group of `per` experts, `each` experts to a lane.  VEC: four logits to a load.
template <int L, int VPL, bool VEC>
__global__ void __launch_bounds__(256) route_kernel(RouteArgs a, int per, int lanes_log2, int each)
{
    const int lane = threadIdx.x & (L - 1);
    const int64_t token = (int64_t)blockIdx.x * (256 / L) + threadIdx.x / L;
    if (token >= a.tokens) return;
    const int lanes = 1 << lanes_log2, group = lane >> lanes_log2, in_group = (lane & (lanes - 1)) * each;
    const int e0 = group * per + in_group, count = group < a.groups ? max(0, min(each, per - in_group)) : 0;
    const int64_t row = token * a.l_rs;
    float x[VPL], p[VPL];
    if constexpr (VEC) {
#pragma unroll
        for (int j = 0; j < VPL; j += 4) {
            f32x4 v = f32x4{-INFINITY, -INFINITY, -INFINITY, -INFINITY};
            if (j < count) v = load_logits(a.logits, a.in_type, row + e0 + j);
#pragma unroll
            for (int i = 0; i < 4; ++i) x[j + i] = v[i];
        }
    } else {
#pragma unroll
        for (int j = 0; j < VPL; ++j) x[j] = j < count ? load_logit(a.logits, a.in_type, row + e0 + j) : -INFINITY;
    }
    float top = 0.f, sum = 1.f;
    auto sigmoid = [](float v) { return 1.f / (1.f + expf(-v)); };
    auto softmax = [&](float v) { return expf(v - top) / sum; };
    // (without a bias the logits order the experts as their softmax does, and exactly; sums of two are sums of scores, though)
    const bool by_logit = a.score == ACC950_SCORE_SOFTMAX && !a.bias, two = a.groups > 1 && a.group_score == ACC950_GROUP_BEST_TWO;
    if (a.score == ACC950_SCORE_SOFTMAX) {
        top = -INFINITY; // (of the numbers: a NaN reaches every score through the sum)
#pragma unroll
        for (int j = 0; j < VPL; ++j) top = fmaxf(top, x[j]);
        top = over_lanes<L>(top, [](float u, float v) { return fmaxf(u, v); });
        if (top == -INFINITY) top = 0.f;
        sum = 0.f;
#pragma unroll
        for (int j = 0; j < VPL; ++j) sum += expf(x[j] - top);
        sum = over_lanes<L>(sum, [](float u, float v) { return u + v; });
        if (sum == 0.f) sum = 1.f;
    }
    if (a.score == ACC950_SCORE_SIGMOID) {
#pragma unroll
        for (int j = 0; j < VPL; ++j) p[j] = sigmoid(x[j]);
    } else if (!by_logit || two) {
#pragma unroll
        for (int j = 0; j < VPL; ++j) p[j] = softmax(x[j]);
    }
    if (a.bias) {
#pragma unroll
        for (int j = 0; j < VPL; j += VEC ? 4 : 1) {
            if (j >= count) continue;
            if constexpr (VEC) {
                const f32x4 b = *(const f32x4*)(a.bias + e0 + j);
#pragma unroll
                for (int i = 0; i < 4; ++i) p[j + i] += b[i];
            } else p[j] += a.bias[e0 + j];
        }
    }
    double key[VPL];
    auto keys_from = [&](bool from_logits) {
#pragma unroll
        for (int j = 0; j < VPL; ++j) {
            const float v = from_logits ? x[j] : p[j];
            const double k = key_of(v, e0 + j);
            key[j] = with_high(k, ((x[j] == -INFINITY) | (v == -INFINITY)) ? NO_KEY : high_word(k)); // (behind `count` x is -inf)
        }
    };
    keys_from(by_logit && !two);
    if (a.groups > 1) {
        double best = no_key(), second = no_key();
#pragma unroll
        for (int j = 0; j < VPL; ++j) {
            if (two) second = larger(second, smaller(best, key[j]));
            best = larger(best, key[j]);
        }
        for (int d = 1; d < lanes; d <<= 1) {
            const double other = __shfl_xor(best, d);
            if (two) second = larger(larger(second, __shfl_xor(second, d)), smaller(best, other));
            best = larger(best, other);
        }
        if (two && high_word(best) != NO_KEY) best = key_of_sum(value_of_key(best), high_word(second) != NO_KEY ? value_of_key(second) : 0.f, group);
        bool open = false;
        for (int n = 0; n < a.top_groups; ++n) {
            const double taken = over_lanes<L>(best, larger);
            if (__double_as_longlong(best) == __double_as_longlong(taken)) {
                open = true; // (a group with nothing to choose too: it has no keys)
                best = no_key();
            }
        }
        if (by_logit && two) keys_from(true);
#pragma unroll
        for (int j = 0; j < VPL; ++j) key[j] = open ? key[j] : with_high(key[j], NO_KEY);
    }
    int my_id = -1; // lane s: slot s
    for (int s = 0; s < a.top_k; ++s) {
        double best[VPL / 2];
#pragma unroll
        for (int j = 0; j < VPL / 2; ++j) best[j] = larger(key[2 * j], key[2 * j + 1]);
#pragma unroll
        for (int n = VPL / 4; n > 0; n /= 2)
#pragma unroll
            for (int j = 0; j < n; ++j) best[j] = larger(best[j], best[j + n]);
        const double taken = over_lanes<L>(best[0], larger);
        const int id = index_of_key(taken); // (without a key left: any, and all keys stay what they are)
        my_id = ((lane == s) & (high_word(taken) != NO_KEY)) ? id : my_id;
#pragma unroll
        for (int j = 0; j < VPL; ++j) key[j] = with_high(key[j], id - e0 == j ? NO_KEY : high_word(key[j]));
    }
    float w = 0.f, mine = -INFINITY; // score and logit of the lane's slot
    if (my_id >= 0) {
        mine = load_logit(a.logits, a.in_type, row + my_id);
        w = a.score == ACC950_SCORE_SIGMOID ? sigmoid(mine) : softmax(mine);
    }
    if (a.renormalise) {
        float total = over_lanes<L>(w, [](float u, float v) { return u + v; });
        if (total < SCORES_LOST) {
            const float largest = over_lanes<L>(mine, [](float u, float v) { return fmaxf(u, v); });
            w = largest == -INFINITY ? 0.f : expf(mine - largest);
            total = over_lanes<L>(w, [](float u, float v) { return u + v; });
        }
        w = total == 0.f ? 0.f : w / total;
    }
    if (lane < a.top_k) {
        a.ids[token * a.top_k + lane] = my_id;
        a.weights[token * a.top_k + lane] = my_id < 0 ? 0.f : w * a.scale;
    }
}

// 8192x128 in bf16 6.2 us (4.7 MB), 16384x256 14 us: a wave to a token, with its reductions and a shuffle for each slot; the exponentials of all experts, to the last
// place as going forward, are about 1 us of the first.
// dlogits.  With g the gradient of the scores taken (g_s = scale * dw_s, or renormalised scale * (dw_s - sum dw w') / total, w' = p / total):
// sigmoid: p (1 - p) g for the experts taken, 1 - p being 1 / (1 + exp(x)), for the difference would have lost its bits where p is nearly 1; softmax: p (g - sum over the
// taken of p g), g 0 for the others.
template <int VPL>
__global__ void __launch_bounds__(256) route_backward_kernel(RouteArgs a)
{
    const int lane = threadIdx.x & 63;
    const int64_t token = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (token >= a.tokens) return;
    float x[VPL], p[VPL], g[VPL];
#pragma unroll
    for (int j = 0; j < VPL; ++j) {
        const int e = j * 64 + lane;
        x[j] = e < a.experts ? load_logit(a.logits, a.in_type, token * a.l_rs + e) : -INFINITY;
        g[j] = 0.f;
    }
    const int my_id = lane < a.top_k ? a.ids[token * a.top_k + lane] : -1;
    const bool have = my_id >= 0 && my_id < a.experts;
    float my_g = have ? a.dweights[token * a.top_k + lane] : 0.f;
    scores_of<VPL>(x, p, a.experts, a.score, lane);
    const bool sigmoid = a.score == ACC950_SCORE_SIGMOID;
    float my_p = 0.f, my_x = 0.f; // score and logit of this lane's slot
#pragma unroll
    for (int j = 0; j < VPL; ++j) {
        const float v = __shfl(p[j], my_id & 63), logit = __shfl(x[j], my_id & 63);
        if (have && my_id >> 6 == j) { my_p = v; my_x = logit; }
    }
    bool lost = false;
    if (a.renormalise) {
        float total = wave_sum(my_p);
        lost = total < SCORES_LOST;
        if (lost) {
            const float largest = of_order_bits(wave_max_u(order_bits(have ? my_x : -INFINITY)));
            my_p = have && largest > -INFINITY ? expf(my_x - largest) : 0.f;
            total = wave_sum(my_p);
        }
        const float shares = wave_sum(my_g * my_p);
        my_g = total == 0.f || !have ? 0.f : (my_g - shares / total) / total;
    }
    my_g *= a.scale;
    float dot = 0.f;
    const bool of_logits = sigmoid || lost; // my_g becomes the gradient of the slot's logit (and is that of its score otherwise)
    if (lost) my_g *= my_p; // (either score's: softmax's other term, the sum of these, is 0, and 1 - p is 1)
    else if (sigmoid) my_g = have ? my_p * (1.f / (1.f + expf(my_x))) * my_g : 0.f;
    else dot = wave_sum(my_p * my_g);
    for (int s = 0; s < a.top_k; ++s) {
        const int e = __builtin_amdgcn_readlane(have ? my_id : -1, s);
        const float gs = __shfl(my_g, s);
#pragma unroll
        for (int j = 0; j < VPL; ++j)
            if (j * 64 + lane == e) g[j] += gs;
    }
#pragma unroll
    for (int j = 0; j < VPL; ++j) {
        const int e = j * 64 + lane;
        if (e < a.experts)
            store_out(a.dlogits, a.in_type, token * a.g_rs + e, of_logits ? g[j] : p[j] * (g[j] - dot));
    }
}

// ---- order of the pairs by expert: a stable counting sort -----------------------------------------
// 131072 pairs of 256 experts 11.5 us, 24576 of 64 9: two launches of a few trips to memory each; up to 1024 pairs one launch, 3.2 us.
// Chunks of pairs are counted (one workgroup each), then every workgroup adds up the counts in front of its chunk and places its
// pairs; a pair's rank inside the chunk comes from its wave's ballots and the counts of the waves before.  No atomics: the
// order does not vary.
constexpr int PLAN_THREADS = 1024, PLAN_WAVES = PLAN_THREADS / 64, PLAN_CHUNKS = 128;

__host__ __device__ inline int plan_chunk(int pairs)
{
    const int c = (pairs + PLAN_CHUNKS - 1) / PLAN_CHUNKS;
    return c <= PLAN_THREADS ? PLAN_THREADS : (c + PLAN_THREADS - 1) / PLAN_THREADS * PLAN_THREADS;
}

// lanes of the wave with the same value (of `bits` bits)
__device__ __forceinline__ unsigned long long same_lanes(int v, int bits, bool active)
{
    unsigned long long m = __ballot(active);
    for (int b = 0; b < bits; ++b) {
        const unsigned long long set = __ballot(v >> b & 1);
        m &= (v >> b & 1) ? set : ~set;
    }
    return m;
}

__device__ __forceinline__ void plan_count(const PlanArgs& a, int chunk)
{
    __shared__ int hist[MAX_EXPERTS + 1];
    for (int e = threadIdx.x; e <= a.experts; e += PLAN_THREADS) hist[e] = 0;
    __syncthreads();
    const int64_t begin = (int64_t)blockIdx.x * chunk, end = begin + chunk < a.pairs ? begin + chunk : a.pairs;
    for (int64_t i = begin + threadIdx.x; i < end; i += PLAN_THREADS) {
        const int e = a.ids[i];
        atomicAdd(&hist[e >= 0 && e < a.experts ? e : a.experts], 1); // (whole numbers: any order gives the same count)
    }
    __syncthreads();
    for (int e = threadIdx.x; e <= a.experts; e += PLAN_THREADS) a.counts[(int64_t)blockIdx.x * (a.experts + 1) + e] = hist[e];
}

// COUNTED: there are several chunks and plan_count has run; otherwise the one workgroup counts its chunk itself.
template <bool COUNTED>
__device__ __forceinline__ void plan_place(const PlanArgs& a, int chunk, int chunks, int bits)
{
    __shared__ int next[MAX_EXPERTS + 1];                   // where the next pair of an expert goes
    __shared__ int wave_count[PLAN_WAVES][MAX_EXPERTS + 1]; // this pass's pairs of a wave
    __shared__ int wave_sums[PLAN_WAVES];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, buckets = a.experts + 1;
    if (a.zeros && blockIdx.x == 0 && tid < 16) a.zeros[tid] = 0;
    int before = 0, total = 0; // of bucket `tid`
    if constexpr (COUNTED) {
        // `parts` threads to a bucket, each with every parts-th chunk; their sums meet in LDS (wave_count is free yet)
        const int parts = buckets >= PLAN_THREADS ? 1 : PLAN_THREADS / buckets < 16 ? PLAN_THREADS / buckets : 16;
        int* sums = &wave_count[0][0];
        for (int u = tid; u < buckets * parts; u += PLAN_THREADS) {
            const int b = u % buckets, part = u / buckets;
            int front = 0, all = 0;
            for (int c0 = part; c0 < chunks; c0 += parts * 16) {
                int n[16];
#pragma unroll
                for (int k = 0; k < 16; ++k) n[k] = c0 + k * parts < chunks ? a.counts[(int64_t)(c0 + k * parts) * buckets + b] : 0;
#pragma unroll
                for (int k = 0; k < 16; ++k) {
                    all += n[k];
                    if (c0 + k * parts < (int)blockIdx.x) front += n[k];
                }
            }
            sums[u * 2] = front;
            sums[u * 2 + 1] = all;
        }
        __syncthreads();
        for (int b = tid; b < buckets; b += PLAN_THREADS) {
            int front = 0, all = 0;
            for (int part = 0; part < parts; ++part) {
                front += sums[(part * buckets + b) * 2];
                all += sums[(part * buckets + b) * 2 + 1];
            }
            if (b < a.experts) { before = front; total = all; }
            else next[b] = front; // (pairs without an expert: where they start is known below)
        }
        __syncthreads();
    } else {
        for (int e = tid; e < buckets; e += PLAN_THREADS) next[e] = 0;
        __syncthreads();
        for (int i = tid; i < a.pairs; i += PLAN_THREADS) {
            const int e = a.ids[i];
            atomicAdd(&next[e >= 0 && e < a.experts ? e : a.experts], 1);
        }
        __syncthreads();
        if (tid < a.experts) total = next[tid];
        __syncthreads();
    }
    int sum = total; // inclusive prefix over the experts
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int o = __shfl_up(sum, d);
        if (lane >= d) sum += o;
    }
    if (lane == 63) wave_sums[wave] = sum;
    __syncthreads();
    int base = 0, all = 0;
    for (int w = 0; w < PLAN_WAVES; ++w) {
        if (w < wave) base += wave_sums[w];
        all += wave_sums[w];
    }
    if (tid < a.experts) {
        next[tid] = base + sum - total + before;
        if (blockIdx.x == 0) a.offsets[tid] = base + sum - total;
    }
    if (tid == 0) {
        if (blockIdx.x == 0) a.offsets[a.experts] = all;
        next[a.experts] = all + (COUNTED ? next[a.experts] : 0); // pairs without an expert go behind
    }
    const int64_t begin = (int64_t)blockIdx.x * chunk, end = begin + chunk < a.pairs ? begin + chunk : a.pairs;
    for (int64_t i0 = begin; i0 < end; i0 += PLAN_THREADS) {
        for (int e = lane; e < buckets; e += 64) wave_count[wave][e] = 0;
        __syncthreads();
        const int64_t i = i0 + tid;
        const bool in = i < end;
        int e = in ? a.ids[i] : 0;
        if (e < 0 || e >= a.experts) e = a.experts;
        const unsigned long long same = same_lanes(e, bits, in);
        const int rank = __popcll(same & ((1ull << lane) - 1));
        if (in && rank == 0) wave_count[wave][e] = __popcll(same);
        __syncthreads();
        int at = 0;
        if (in) {
            at = next[e] + rank;
#pragma unroll
            for (int w = 0; w < PLAN_WAVES; ++w) { // (all at once, not one by one up to this wave)
                const int n = wave_count[w][e];
                at += w < wave ? n : 0;
            }
            a.order[at] = (int)i;
            a.position[i] = e < a.experts ? at : -1;
        }
        if (i0 + PLAN_THREADS >= end) return;
        __syncthreads(); // every `next` is read
        for (int b = tid; b < buckets; b += PLAN_THREADS) {
            int n = 0;
            for (int w = 0; w < PLAN_WAVES; ++w) n += wave_count[w][b];
            next[b] += n;
        }
        __syncthreads();
    }
}

__global__ void __launch_bounds__(PLAN_THREADS) plan_count_kernel(PlanArgs a, int chunk) { plan_count(a, chunk); }
template <bool COUNTED>
__global__ void __launch_bounds__(PLAN_THREADS) plan_place_kernel(PlanArgs a, int chunk, int chunks, int bits) { plan_place<COUNTED>(a, chunk, chunks, bits); }

// The plan's first step (its only one with ONE chunk) beside the quantising of the tokens' rows, which needs none of it.
template <int TYPE, bool VEC, bool ONE>
__global__ void __launch_bounds__(PLAN_THREADS) plan_quantize_kernel(PlanArgs a, int chunk, int chunks, int bits, F8QuantizeArgs q)
{
    if ((int)blockIdx.x >= chunks) f8_quantize_unit<TYPE, VEC, ACC950_ACT_NONE>(q, (blockIdx.x - chunks) * PLAN_WAVES + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), threadIdx.x & 63);
    else if constexpr (ONE) plan_place<false>(a, chunk, 1, bits);
    else plan_count(a, chunk);
}

// ---- weighted sum of a token's rows ---------------------------------------------------------------
// Bound by memory: six rows of 2048 in fp16 for each of 4096 tokens 26.9 us (118 MB, 4.5 TB/s).
template <int IN, int OUT, bool VEC>
__global__ void __launch_bounds__(256) combine_kernel(CombineArgs a)
{
    constexpr int PER = VEC ? (OUT == T_F32 ? 4 : 8) : 1;
    const int pieces = (a.cols + PER - 1) / PER;
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t t = a.few ? (int64_t)a.by_pieces((unsigned)i) : i / pieces;
    if (t >= a.tokens) return;
    const int c = (int)(i - t * pieces) * PER;
    float sum[PER] = {};
    constexpr int AT_ONCE = 4; // slots whose rows are on the way together
    constexpr int PIECES = VEC ? (IN == T_F32 ? PER / 4 : 1) : 1;
    for (int s0 = 0; s0 < a.top_k; s0 += AT_ONCE) {
        int row[AT_ONCE];
        float w[AT_ONCE];
        i32x4 raw[AT_ONCE][PIECES];
        float one[AT_ONCE];
#pragma unroll
        for (int u = 0; u < AT_ONCE; ++u) row[u] = s0 + u < a.top_k ? a.position[t * a.top_k + s0 + u] : -1;
#pragma unroll
        for (int u = 0; u < AT_ONCE; ++u) {
            if (row[u] < 0) continue;
            const int64_t at = (int64_t)row[u] * a.x_rs + c;
            w[u] = a.weights ? a.weights[t * a.top_k + s0 + u] : 1.f;
            if (IN == T_F16 && a.scale) w[u] *= a.scale[(int64_t)row[u] * a.s_rs + (c >> 5)];
            if constexpr (!VEC) one[u] = load_out(a.x, IN, at);
            else {
#pragma unroll
                for (int h = 0; h < PIECES; ++h) raw[u][h] = *(const i32x4*)((const char*)a.x + at * (IN == T_F32 ? 4 : 2) + h * 16);
            }
        }
#pragma unroll
        for (int u = 0; u < AT_ONCE; ++u) {
            if (row[u] < 0) continue;
            if constexpr (!VEC) sum[0] += w[u] * one[u];
            else if constexpr (IN == T_F32) {
#pragma unroll
                for (int e = 0; e < PER; ++e) sum[e] += w[u] * __int_as_float(raw[u][e / 4][e % 4]);
            } else {
#pragma unroll
                for (int e = 0; e < PER; ++e) {
                    const uint16_t h = (uint16_t)((unsigned)raw[u][0][e / 2] >> (e % 2 * 16));
                    sum[e] += w[u] * (IN == T_F16 ? f16_bits_to_float(h) : bf16_bits_to_float(h));
                }
            }
        }
    }
    const int64_t at = t * a.y_rs + c;
    if constexpr (!VEC) store_out(a.y, OUT, at, sum[0]);
    else if constexpr (OUT == T_F32) *(f32x4*)((float*)a.y + at) = f32x4{sum[0], sum[1], sum[2], sum[3]};
    else {
        i32x4 v;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const unsigned lo = OUT == T_F16 ? float_to_f16_bits(sum[2 * e]) : float_to_bf16_bits(sum[2 * e]);
            const unsigned hi = OUT == T_F16 ? float_to_f16_bits(sum[2 * e + 1]) : float_to_bf16_bits(sum[2 * e + 1]);
            v[e] = (int)(lo | hi << 16);
        }
        *(i32x4*)((uint16_t*)a.y + at) = v;
    }
}

template <int IN, int OUT>
hipError_t launch_combine(CombineArgs a, hipStream_t s)
{
    constexpr int PER = OUT == T_F32 ? 4 : 8;
    const bool vec = a.cols % PER == 0 && a.x_rs % PER == 0 && a.y_rs % PER == 0 && (((size_t)a.x | (size_t)a.y) & 15) == 0;
    const int64_t n = (int64_t)a.tokens * (vec ? a.cols / PER : a.cols), blocks = (n + 255) / 256;
    if (blocks > 0x7fffffffll) return hipErrorInvalidConfiguration;
    a.few = n < 0x7fffffffll - 256;
    a.by_pieces = F8Over((unsigned)(vec ? a.cols / PER : a.cols));
    if (vec) combine_kernel<IN, OUT, true><<<dim3((unsigned)blocks), dim3(256), 0, s>>>(a);
    else combine_kernel<IN, OUT, false><<<dim3((unsigned)blocks), dim3(256), 0, s>>>(a);
    return hipGetLastError();
}

template <typename F>
hipError_t by_lanes(int experts, F&& f)
{
    if (experts <= 64) f(std::integral_constant<int, 1>{});
    else if (experts <= 128) f(std::integral_constant<int, 2>{});
    else if (experts <= 256) f(std::integral_constant<int, 4>{});
    else if (experts <= 512) f(std::integral_constant<int, 8>{});
    else f(std::integral_constant<int, 16>{});
    return hipGetLastError();
}

} // namespace

hipError_t launch_route(const RouteArgs& a, hipStream_t s)
{
    if (a.tokens == 0) return hipSuccess;
    // 16 lanes to a token where a lane then has few experts or there are tokens enough to fill the chip with such waves: a quarter of the steps over
    // lanes.  Else 64: fewer experts to a lane, a shorter chain.  (us, 16 / 64: 16384 tokens of 256 experts in groups 15.0 / 23.9, 4096 7.4 / 8.7,
    // 2048 7.1 / 6.1, 8 6.8 / 5.1; 16384 of 64 experts 5.2 / 16.5, 8 3.2 / 3.7.)
    const int per = a.experts / a.groups;
    int lanes_log2 = 0, each = 0;
    auto spread = [&](int L) { // a group's lanes and what is left to each
        if (L < a.groups) return false;
        for (lanes_log2 = 0; (2 << lanes_log2) * a.groups <= L; ++lanes_log2) {}
        each = (per + (1 << lanes_log2) - 1) >> lanes_log2;
        return true;
    };
    const bool narrow = a.top_k <= 16 && spread(16) && each <= 16 && (each <= 4 || a.tokens >= 256 * each);
    if (!narrow) spread(64);
    const int64_t to = a.in_type == T_F32 ? 16 : 8;
    const bool vec = per % 4 == 0 && a.l_rs % 4 == 0 && ((size_t)a.logits & (to - 1)) == 0 && ((size_t)a.bias & 15) == 0;
    if (vec) each = (each + 3) / 4 * 4; // (a group's last lanes have less)
    const int token_lanes = narrow ? 16 : 64;
    const dim3 grid((unsigned)(((int64_t)a.tokens + 256 / token_lanes - 1) / (256 / token_lanes)));
    auto launch = [&](auto l, auto vpl) {
        if (vec) route_kernel<decltype(l)::value, decltype(vpl)::value, true><<<grid, dim3(256), 0, s>>>(a, per, lanes_log2, each);
        else route_kernel<decltype(l)::value, decltype(vpl)::value, false><<<grid, dim3(256), 0, s>>>(a, per, lanes_log2, each);
        return hipGetLastError();
    };
    std::integral_constant<int, 16> l16;
    std::integral_constant<int, 64> l64;
    if (narrow) return each <= 4 ? launch(l16, std::integral_constant<int, 4>{}) : each <= 8 ? launch(l16, std::integral_constant<int, 8>{}) : launch(l16, std::integral_constant<int, 16>{});
    return each <= 4 ? launch(l64, std::integral_constant<int, 4>{}) : each <= 16 ? launch(l64, std::integral_constant<int, 16>{}) : launch(l64, std::integral_constant<int, 32>{});
}

hipError_t launch_route_backward(const RouteArgs& a, hipStream_t s)
{
    if (a.tokens == 0) return hipSuccess;
    const dim3 grid((unsigned)(((int64_t)a.tokens + 3) / 4));
    return by_lanes(a.experts, [&](auto vpl) { route_backward_kernel<decltype(vpl)::value><<<grid, dim3(256), 0, s>>>(a); });
}

int64_t expert_plan_workspace(int64_t pairs, int64_t experts)
{
    const int64_t chunk = plan_chunk((int)pairs), chunks = (pairs + chunk - 1) / chunk;
    return chunks > 1 ? chunks * (experts + 1) * 4 : 0;
}

namespace {

struct PlanSteps {
    int chunk, chunks, bits;
    explicit PlanSteps(const PlanArgs& a) : chunk(plan_chunk(a.pairs)), chunks((int)(((int64_t)a.pairs + chunk - 1) / chunk)), bits(1)
    {
        if (chunks < 1) chunks = 1;
        while ((1 << bits) < a.experts + 1) ++bits;
    }
};

template <int TYPE, bool VEC>
hipError_t plan_and_quantize(const PlanArgs& a, const PlanSteps& p, F8QuantizeArgs q, hipStream_t s)
{
    const int64_t units = (int64_t)q.rows * ((q.cols + 511) / 512), blocks = p.chunks + (units + PLAN_WAVES - 1) / PLAN_WAVES;
    if (units > 0x7fffffffll - PLAN_WAVES) return hipErrorInvalidConfiguration;
    q.by_quads = F8Over((unsigned)((q.cols + 511) / 512));
    if (p.chunks == 1) plan_quantize_kernel<TYPE, VEC, true><<<dim3((unsigned)blocks), dim3(PLAN_THREADS), 0, s>>>(a, p.chunk, 1, p.bits, q);
    else {
        plan_quantize_kernel<TYPE, VEC, false><<<dim3((unsigned)blocks), dim3(PLAN_THREADS), 0, s>>>(a, p.chunk, p.chunks, p.bits, q);
        plan_place_kernel<true><<<dim3(p.chunks), dim3(PLAN_THREADS), 0, s>>>(a, p.chunk, p.chunks, p.bits);
    }
    return hipGetLastError();
}

} // namespace

hipError_t launch_expert_plan(const PlanArgs& a, hipStream_t s)
{
    const PlanSteps p(a);
    if (p.chunks == 1) plan_place_kernel<false><<<dim3(1), dim3(PLAN_THREADS), 0, s>>>(a, p.chunk, 1, p.bits);
    else {
        plan_count_kernel<<<dim3(p.chunks), dim3(PLAN_THREADS), 0, s>>>(a, p.chunk);
        plan_place_kernel<true><<<dim3(p.chunks), dim3(PLAN_THREADS), 0, s>>>(a, p.chunk, p.chunks, p.bits);
    }
    return hipGetLastError();
}

hipError_t launch_expert_plan_and_quantize(const PlanArgs& a, const F8QuantizeArgs& q, hipStream_t s)
{
    const PlanSteps p(a);
    if (q.in_type == T_F16) return f8_quantize_by_16<T_F16>(q) ? plan_and_quantize<T_F16, true>(a, p, q, s) : plan_and_quantize<T_F16, false>(a, p, q, s);
    return f8_quantize_by_16<T_BF16>(q) ? plan_and_quantize<T_BF16, true>(a, p, q, s) : plan_and_quantize<T_BF16, false>(a, p, q, s);
}

hipError_t launch_expert_combine(const CombineArgs& a, hipStream_t s)
{
    if (a.tokens == 0 || a.cols == 0) return hipSuccess;
    const bool f32 = a.in_type == T_F32;
    switch (a.type) {
    case T_F16: return f32 ? launch_combine<T_F32, T_F16>(a, s) : launch_combine<T_F16, T_F16>(a, s);
    case T_BF16: return f32 ? launch_combine<T_F32, T_BF16>(a, s) : a.in_type == T_F16 ? launch_combine<T_F16, T_BF16>(a, s) : launch_combine<T_BF16, T_BF16>(a, s);
    default: return launch_combine<T_F32, T_F32>(a, s);
    }
}

} // namespace acc950
