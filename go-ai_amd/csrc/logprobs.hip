// logprobs.hip -- log probabilities of given actions under a policy's logits, with the entropy and the best alternatives,
// and their gradient.
//
//   s_j = x_j / T over the allowed columns j (valid[j] != 0 and x_j > -inf)
//   lse = log sum_j exp(s_j),  log p_a = s_a - lse,  H = -sum_j p_j log p_j
//   d x_j = (g (delta_aj - p_j) - h p_j (log p_j + H)) / T        for a loss with d/d log p_a = g, d/dH = h
//
// The forward pass reads the logits once: every lane keeps the maximum m of the logits it has seen and, with t = (x - m) c,
// c = log2(e) / T, the sums l = sum 2^t and e = sum 2^t t; a maximum larger by d / c scales l by 2^-d and turns e into
// 2^-d (e - d l).  All terms of e have one sign, so H = ln 2 (log2 l - e / l) loses nothing to cancellation.  Sums are float32; those over
// the tiles of a long row carry what each addition rounded off (a lane's 2000 terms of 128001 columns, added one by one, were up to 4e-5
// off: equal terms round the same way over and over).
// A lane without columns has m = -FLT_MAX, l = e = 0: x - m is then never inf - inf, and l == 0 says that a row has no allowed
// column.  t may be -inf (a column that is not allowed, or an overflow): its power is 0, and t is bounded in front of the product.
#include <float.h>
#include <math.h>

#include <algorithm>
#include <utility>

#include "ctx.h"
#include "elem.h"
#include "goai_internal.h"

namespace goai {

constexpr int LP_TOP = GOAI_LOGPROBS_MAX_TOP;      // a wavefront's list of alternatives: one per lane
constexpr float LOG2E = 1.44269504088896340736f, LN2 = 0.69314718055994530942f;

struct LpStat {
    float m = -FLT_MAX, l = 0.0f, e = 0.0f;
};

// a factor that many terms share, to more than 24 bits: its rounding would move all of them the same way.  0 < lo: an infinite
// d stays infinite
struct LpFactor {
    float hi, lo;
};
__device__ __forceinline__ float lp_times(float d, LpFactor c) { return fmaf(d, c.lo, d * c.hi); }

__device__ __forceinline__ void lp_add(LpStat& s, float x, LpFactor c)       // x <= s.m
{
    const float t = lp_times(x - s.m, c), p = __builtin_amdgcn_exp2f(t);
    s.l += p;
    s.e = fmaf(p, fmaxf(t, -1000.0f), s.e);
}

__device__ __forceinline__ void lp_raise(LpStat& s, float m, LpFactor c)     // m >= s.m
{
    const float d = fminf(lp_times(m - s.m, c), 1000.0f), f = __builtin_amdgcn_exp2f(-d);
    s.e = f * fmaf(-d, s.l, s.e);
    s.l *= f;
    s.m = m;
}

// `low`: what the additions into s.l and s.e have rounded off (all of it where the sum is the larger of the two, as it is but for tiles behind
// a raise)
__device__ __forceinline__ void lp_raise(LpStat& s, LpStat& low, float m, LpFactor c)
{
    const float d = fminf(lp_times(m - s.m, c), 1000.0f), f = __builtin_amdgcn_exp2f(-d);
    s.e = f * fmaf(-d, s.l, s.e);
    low.e = f * fmaf(-d, low.l, low.e);
    s.l *= f;
    low.l *= f;
    s.m = m;
}
__device__ __forceinline__ void lp_carry(float& sum, float& low, float x)
{
    const float y = x + low, t = sum + y;
    low = y - (t - sum);
    sum = t;
}
// a tile's columns (all <= s.m), summed four ways by themselves
template <int N> __device__ __forceinline__ void lp_tile(LpStat& s, LpStat& low, const float (&x)[N], LpFactor c)
{
    LpStat a[4];
#pragma unroll
    for (int k = 0; k < 4; k++) a[k].m = s.m;
#pragma unroll
    for (int k = 0; k < N; k++) lp_add(a[k % 4], x[k], c);
    lp_carry(s.l, low.l, (a[0].l + a[1].l) + (a[2].l + a[3].l));
    lp_carry(s.e, low.e, (a[0].e + a[1].e) + (a[2].e + a[3].e));
}

// ---- cross-lane helpers: DPP moves within rows of 16 lanes and from row to row, which do without the LDS unit that shuffles go
// through (5 x 128001 rising columns, 20 alternatives: 27 -> 24 us a call) ----
template <int CTRL> __device__ __forceinline__ int lp_dpp(int x) { return __builtin_amdgcn_mov_dpp(x, CTRL, 0xf, 0xf, true); }
template <int CTRL> __device__ __forceinline__ float lp_dpp(float x) { return __int_as_float(lp_dpp<CTRL>(__float_as_int(x))); }
constexpr int SHR = 0x110, ROR = 0x120, WAVE_SHR1 = 0x138, MIRROR = 0x140, HALF_MIRROR = 0x141, XOR1 = 0xb1, XOR2 = 0x4e, XOR3 = 0x1b;
// lane 15 of each row to the row behind it (rows 1 and 3 take it), lane 31 to the rows 2 and 3; the other rows keep `keep`
__device__ __forceinline__ int lp_row15(int keep, int x) { return __builtin_amdgcn_update_dpp(keep, x, 0x142, 0xa, 0xf, false); }
__device__ __forceinline__ int lp_row31(int keep, int x) { return __builtin_amdgcn_update_dpp(keep, x, 0x143, 0xc, 0xf, false); }
__device__ __forceinline__ float lp_row15(float keep, float x) { return __int_as_float(lp_row15(__float_as_int(keep), __float_as_int(x))); }
__device__ __forceinline__ float lp_row31(float keep, float x) { return __int_as_float(lp_row31(__float_as_int(keep), __float_as_int(x))); }
__device__ __forceinline__ float lp_lane(float x, int lane) { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), lane)); }
__device__ __forceinline__ int lp_lane(int x, int lane) { return __builtin_amdgcn_readlane(x, lane); }

// over groups of L = 16 or 64 lanes, the result in all of them; `none` is the operation's neutral element
template <int L, class T, class F> __device__ __forceinline__ T lp_reduce(T x, T none, F&& f)
{
    x = f(x, lp_dpp<ROR + 8>(x));
    x = f(x, lp_dpp<ROR + 4>(x));
    x = f(x, lp_dpp<ROR + 2>(x));
    x = f(x, lp_dpp<ROR + 1>(x));
    if constexpr (L == 64) {
        x = f(x, lp_row15(none, x));
        x = f(x, lp_row31(none, x));
        x = lp_lane(x, 63);
    }
    return x;
}
template <int L> __device__ __forceinline__ float lp_max(float x)
{
    return lp_reduce<L>(x, -INFINITY, [](float a, float b) { return fmaxf(a, b); });
}
template <int L> __device__ __forceinline__ float lp_sum(float x)
{
    return lp_reduce<L>(x, 0.0f, [](float a, float b) { return a + b; });
}
template <int L> __device__ __forceinline__ int lp_count(int n)
{
    return lp_reduce<L>(n, 0, [](int a, int b) { return a + b; });
}

// the sum of n over the lanes of a group before this one
template <int L> __device__ __forceinline__ int lp_before_me(int n)
{
    int upto = n;
    upto += lp_dpp<SHR + 1>(upto);
    upto += lp_dpp<SHR + 2>(upto);
    upto += lp_dpp<SHR + 4>(upto);
    upto += lp_dpp<SHR + 8>(upto);
    if constexpr (L == 64) {
        upto += lp_row15(0, upto);
        upto += lp_row31(0, upto);
    }
    return upto - n;
}

// the statistics of all lanes' columns together
__device__ __forceinline__ LpStat lp_wave_join(LpStat s, LpFactor c)
{
    lp_raise(s, lp_max<64>(s.m), c);
    s.l = lp_sum<64>(s.l);
    s.e = lp_sum<64>(s.e);
    return s;
}

// Sixteen lanes' values in descending order (a bitonic network: every step keeps the larger of two lanes' values in the lower).
__device__ __forceinline__ float lp_sort16(float x, int lane)
{
    const float b0 = lane & 1 ? -INFINITY : INFINITY, b1 = lane & 2 ? -INFINITY : INFINITY, b2 = lane & 4 ? -INFINITY : INFINITY,
                b3 = lane & 8 ? -INFINITY : INFINITY;
    // med3 with +inf is the maximum, with -inf the minimum
    x = __builtin_amdgcn_fmed3f(x, lp_dpp<XOR1>(x), b0);
    x = __builtin_amdgcn_fmed3f(x, lp_dpp<XOR3>(x), b1);
    x = __builtin_amdgcn_fmed3f(x, lp_dpp<XOR1>(x), b0);
    x = __builtin_amdgcn_fmed3f(x, lp_dpp<HALF_MIRROR>(x), b2);
    x = __builtin_amdgcn_fmed3f(x, lp_dpp<XOR2>(x), b1);
    x = __builtin_amdgcn_fmed3f(x, lp_dpp<XOR1>(x), b0);
    x = __builtin_amdgcn_fmed3f(x, lp_dpp<MIRROR>(x), b3);
    x = __builtin_amdgcn_fmed3f(x, lp_dpp<XOR3>(lp_dpp<HALF_MIRROR>(x)), b2);
    x = __builtin_amdgcn_fmed3f(x, lp_dpp<XOR2>(x), b1);
    return __builtin_amdgcn_fmed3f(x, lp_dpp<XOR1>(x), b0);
}

// The top-th largest of a group's L lanes' own maxima (a lane without columns: -inf): at least `top` columns reach it.
// -FLT_MAX if there are none.
template <int L> __device__ __forceinline__ float lp_threshold(float lane_max, int top, int lane)
{
    float s = lp_sort16(lane_max, lane & 15);
    if constexpr (L == 64) {
        // two sorted halves, one of them turned round, make a bitonic sequence: merged in log2 steps
        const float b0 = lane & 1 ? -INFINITY : INFINITY, b1 = lane & 2 ? -INFINITY : INFINITY, b2 = lane & 4 ? -INFINITY : INFINITY,
                    b3 = lane & 8 ? -INFINITY : INFINITY, b4 = lane & 16 ? -INFINITY : INFINITY, b5 = lane & 32 ? -INFINITY : INFINITY;
        auto merge16 = [&] {
            s = __builtin_amdgcn_fmed3f(s, lp_dpp<ROR + 8>(s), b3);
            s = __builtin_amdgcn_fmed3f(s, lp_dpp<XOR3>(lp_dpp<HALF_MIRROR>(s)), b2);
            s = __builtin_amdgcn_fmed3f(s, lp_dpp<XOR2>(s), b1);
            s = __builtin_amdgcn_fmed3f(s, lp_dpp<XOR1>(s), b0);
        };
        s = __builtin_amdgcn_fmed3f(s, __shfl_xor(s, 31), b4);
        merge16();
        s = __builtin_amdgcn_fmed3f(s, __shfl_xor(s, 63), b5);
        s = __builtin_amdgcn_fmed3f(s, __shfl_xor(s, 16), b4);
        merge16();
    }
    return fmaxf(L == 64 ? lp_lane(s, top - 1) : __shfl(s, (lane & (64 - L)) + top - 1), -FLT_MAX);
}

// bit (N - 1 - k) for x[k] >= t: bits = 2 bits + (x[k] >= t), a compare and an add with its carry.  The carry may be read two
// instructions after the compare at the earliest, so compares and adds go four by four.
template <int N> __device__ __forceinline__ unsigned lp_at_least(const float (&x)[N], float t)
{
    unsigned bits = 0;
    unsigned long long a, b, c, d, e;
#pragma unroll
    for (int k = 0; k + 4 <= N; k += 4)
        asm("v_cmp_ge_f32 %1, %6, %10\n\tv_cmp_ge_f32 %2, %7, %10\n\tv_cmp_ge_f32 %3, %8, %10\n\tv_cmp_ge_f32 %4, %9, %10\n\t"
            "v_addc_co_u32 %0, %5, %0, %0, %1\n\tv_addc_co_u32 %0, %5, %0, %0, %2\n\t"
            "v_addc_co_u32 %0, %5, %0, %0, %3\n\tv_addc_co_u32 %0, %5, %0, %0, %4"
            : "+v"(bits), "=&s"(a), "=&s"(b), "=&s"(c), "=&s"(d), "=&s"(e)
            : "v"(x[k]), "v"(x[k + 1]), "v"(x[k + 2]), "v"(x[k + 3]), "v"(t));
#pragma unroll
    for (int k = N / 4 * 4; k < N; k++) bits = 2 * bits + (x[k] >= t ? 1u : 0u);
    return bits;
}

// x[k] = -inf where byte k of `ok` is 0 (as above: four compares, four selections)
__device__ __forceinline__ void lp_mask4(float& x0, float& x1, float& x2, float& x3, unsigned ok)
{
    unsigned long long a, b, c, d;
    asm("v_cmp_ne_u32_sdwa %4, %8, %9 src0_sel:BYTE_0 src1_sel:DWORD\n\tv_cmp_ne_u32_sdwa %5, %8, %9 src0_sel:BYTE_1 src1_sel:DWORD\n\t"
        "v_cmp_ne_u32_sdwa %6, %8, %9 src0_sel:BYTE_2 src1_sel:DWORD\n\tv_cmp_ne_u32_sdwa %7, %8, %9 src0_sel:BYTE_3 src1_sel:DWORD\n\t"
        "v_cndmask_b32 %0, %10, %0, %4\n\tv_cndmask_b32 %1, %10, %1, %5\n\tv_cndmask_b32 %2, %10, %2, %6\n\t"
        "v_cndmask_b32 %3, %10, %3, %7"
        : "+v"(x0), "+v"(x1), "+v"(x2), "+v"(x3), "=&s"(a), "=&s"(b), "=&s"(c), "=&s"(d)
        : "v"(ok), "v"(0u), "v"(-INFINITY));
}

// floats as integers of the same order, and back
__device__ __forceinline__ int lp_key(int bits) { return bits ^ ((bits >> 31) & 0x7fffffff); }

// The candidates of a group of L lanes for its `top` best columns: at least `top` of them (all, if there are fewer), at most L;
// bits as in lp_at_least, `count` in the group.  Lane l holds vectors of V neighbouring columns, l V + q L V ...
// The first threshold, lp_threshold, is sharp while a lane seldom holds two of the best.  Where it leaves more than L, the range
// between it and the largest value is halved until it does not (3.5 % of the wavefronts for 8 of 362 columns over 16 lanes, some 3
// steps), and where that ends at one value that too many columns share, the range of columns that count among them.
template <int L, int V, int N> __device__ __forceinline__ unsigned lp_candidates(const float (&x)[N], float lane_max, float most, int top, int lane, int& count)
{
    const float T = lp_threshold<L>(lane_max, top, lane);
    unsigned bits = lp_at_least(x, T);
    count = lp_count<L>(__popc(bits));
    if (__any(count > L)) {
        int lo = lp_key(__float_as_int(T)), hi = lp_key(__float_as_int(most)) + 1;       // enough columns reach lo, too few reach hi
        unsigned above = 0;                                                              // those that reach hi
        while (__any(count > L && (unsigned)hi - (unsigned)lo > 1u)) {
            const int mid = (int)((unsigned)lo + (((unsigned)hi - (unsigned)lo) >> 1));
            const unsigned b = lp_at_least(x, __int_as_float(lp_key(mid)));
            const int n = lp_count<L>(__popc(b));
            if (count > L && (unsigned)hi - (unsigned)lo > 1u) {
                if (n >= top) {
                    lo = mid;
                    bits = b;
                    count = n;
                } else {
                    hi = mid;
                    above = b;
                }
            }
        }
        int c0 = 0, c1 = N * L;                              // too few, enough with the first so many columns of those at lo
        const unsigned ties = bits & ~above;
        const bool tied = count > L;
        while (__any(count > L && c1 - c0 > 1)) {
            const int mid = (c0 + c1) >> 1, q = mid / (L * V), mine = q * V + min(max(mid - (q * L + (lane & (L - 1))) * V, 0), V);
            const unsigned b = above | (ties & (mine ? ~0u << (N - mine) : 0u));
            const int n = lp_count<L>(__popc(b));
            if (tied && count > L) {
                if (n >= top) {
                    c1 = mid;
                    bits = b;
                    count = n;
                } else c0 = mid;
            }
        }
    }
    return bits;
}

// (v, i) comes before (w, j): larger logit, then lower column
__device__ __forceinline__ bool lp_before(float v, int i, float w, int j) { return v > w || (v == w && i < j); }

constexpr int LP_NONE = 0x40000000;        // columns from here on stand for "no column" (with v = -inf): cols <= 2^30

// How many of a group's L entries (one per lane, no two the same) come before the lane's own; L = 64: of the first `count`.
template <int... K> __device__ __forceinline__ int lp_rank16(float v, int i, std::integer_sequence<int, K...>)
{
    // (rotations of the same register: no one waits for the one before)
    return (0 + ... + (int)lp_before(lp_dpp<ROR + 1 + K>(v), lp_dpp<ROR + 1 + K>(i), v, i));
}
template <int L> __device__ __forceinline__ int lp_rank(float v, int i, int count)
{
    if constexpr (L == 16) return lp_rank16(v, i, std::make_integer_sequence<int, 15>());
    int rank = 0;
    for (int k = 0; k < count; k++) {
        const float w = lp_lane(v, k);
        const int j = lp_lane(i, k);
        rank += lp_before(w, j, v, i);
    }
    return rank;
}

// One wavefront's best columns, best first, one per lane.
struct LpList {
    float v = -INFINITY;
    int i = LP_NONE;
};

__device__ __forceinline__ void lp_insert(LpList& t, float cv, int ci, int lane)
{
    const unsigned long long before = __ballot(lp_before(t.v, t.i, cv, ci));
    const int pos = __popcll(before);
    const float sv = lp_dpp<WAVE_SHR1>(t.v);
    const int si = lp_dpp<WAVE_SHR1>(t.i);
    if (lane == pos) { t.v = cv; t.i = ci; }
    else if (lane > pos) { t.v = sv; t.i = si; }
}

__device__ __forceinline__ void lp_wave_sync()
{
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup");
}

struct LpArgs {
    const void* x;
    long xstride;
    const uint8_t* valid;
    long vstride;
    const int* actions;
    LpFactor inv_t, c2;                    // 1 / T, log2(e) / T
    int top;
    float *logp, *entropy, *lse;
    int* top_actions;
    float* top_logp;
    long rows;
    int cols;
};


// The given action's logit, read early (its address waits for another load): NaN for an action beyond the row, -inf where the column
// is not allowed, +inf (which no allowed finite logit is: a row with one is NaN anyway) for "no action".
template <int E> __device__ __forceinline__ float lp_given(const LpArgs& A, long row)
{
    using raw = typename Elem<E>::raw;
    const int a = A.actions ? A.actions[row] : -1;
    if (a >= A.cols) return NAN;
    if (a < 0) return INFINITY;
    const float x = elem_to_float<E>(((const raw*)A.x)[row * A.xstride + a]);
    return A.valid && !A.valid[row * A.vstride + a] ? -INFINITY : x == INFINITY ? NAN : x;
}

// lse, entropy and the given action's log probability of a row (one lane)
__device__ __forceinline__ void lp_write_row(const LpArgs& A, long row, const LpStat& s, float logl, float given)
{
    const bool none = s.l == 0.0f;                               // no allowed column
    if (A.lse) A.lse[row] = none ? -INFINITY : __builtin_amdgcn_fmed3f(lp_times(s.m, A.inv_t), -FLT_MAX, FLT_MAX) + logl;
    if (A.entropy) A.entropy[row] = none ? 0.0f : logl - LN2 * (s.e / s.l);
    if (A.logp) A.logp[row] = given == INFINITY ? 0.0f : given == -INFINITY ? -INFINITY : lp_times(given - s.m, A.inv_t) - logl;
}
__device__ __forceinline__ void lp_write_top(const LpArgs& A, long row, int rank, float v, int i, const LpStat& s, float logl)
{
    const bool some = i < LP_NONE;
    A.top_actions[row * A.top + rank] = some ? i : -1;
    A.top_logp[row * A.top + rank] = some ? lp_times(v - s.m, A.inv_t) - logl : -INFINITY;
}

// ---- short rows: all of a row in the registers of L lanes, NV vectors of V columns each; lane l's are (q L + l) V .. + V; the
// first FULL vectors of every lane lie within the row for sure ----
//
// The alternatives: T = lp_threshold of the lanes' maxima leaves few candidates (for 8 of 362 columns about 11).  The row goes to
// LDS, every lane looks up its candidates there (a bit each), one lane takes each, and a candidate's place is the number of those
// before it.

template <int E, int L, int V, int NV, int FULL, bool TOP> __global__ __launch_bounds__(256) void k_logprobs_short(LpArgs A)
{
    using raw = typename Elem<E>::raw;
    constexpr int N = NV * V;
    __shared__ float lds_x[TOP ? 256 * N : 1];                   // lane by lane
    __shared__ float lds_v[TOP ? 256 : 1];
    __shared__ int lds_i[TOP ? 256 : 1];
    const int lane = threadIdx.x & 63, sub = lane & (L - 1);
    const int group = (threadIdx.x & ~(L - 1));                  // this group's first slot in LDS
    const long mine_row = (long)blockIdx.x * (256 / L) + threadIdx.x / L;
    const bool active = mine_row < A.rows;                   // (the lanes behind the last row work on it too, and write nothing)
    const long row = active ? mine_row : A.rows - 1;
    // All loads are issued before the first is used.  A vector that would pass the row's end starts cols - V (cols >= V) instead; its
    // columns in front of the lane's own are another lane's.
    const int last = A.cols - V;
    const float given = lp_given<E>(A, row);
    float x[N];
    {
        const raw* p = (const raw*)A.x + row * A.xstride;
        ElemVec<E, V> t[NV];
#pragma unroll
        for (int q = 0; q < NV; q++) __builtin_memcpy(&t[q], p + min((q * L + sub) * V, last), sizeof(t[q]));
        unsigned ok[NV];                                         // a byte per column: not 0 where it is allowed
#pragma unroll
        for (int q = 0; q < NV; q++) ok[q] = ~0u;
        if (A.valid) {
            const uint8_t* valid = A.valid + row * A.vstride;
#pragma unroll
            for (int q = 0; q < NV; q++) __builtin_memcpy(&ok[q], valid + min((q * L + sub) * V, last), V);
        }
#pragma unroll
        for (int k = 0; k < N; k++) x[k] = elem_to_float<E>(t[k / V].a[k % V]);
        if (A.valid || FULL < NV) {
#pragma unroll
            for (int q = 0; q < NV; q++) {
                if (!A.valid && q < FULL) continue;
                if (q >= FULL) {
                    const int c = (q * L + sub) * V;
                    ok[q] &= (unsigned)(0xffffffffull << (8 * min(c - min(c, last), 4)));
                }
                if constexpr (V == 4) lp_mask4(x[q * V], x[q * V + 1], x[q * V + 2], x[q * V + 3], ok[q]);
                else x[q] = ok[q] & 255u ? x[q] : -INFINITY;
            }
        }
    }
    float lane_max = -INFINITY;
#pragma unroll
    for (int k = 0; k < N; k++) lane_max = fmaxf(lane_max, x[k]);
    LpStat s;
    s.m = fmaxf(lp_max<L>(lane_max), -FLT_MAX);
#pragma unroll
    for (int k = 0; k < N; k++) lp_add(s, x[k], A.c2);
    s.l = lp_sum<L>(s.l);
    s.e = lp_sum<L>(s.e);
    const float logl = logf(s.l);
    if (sub == 0 && active) lp_write_row(A, row, s, logl, given);
    if constexpr (TOP) {
        float* mine_x = lds_x + threadIdx.x * N;
#pragma unroll
        for (int k = 0; k < N; k++) mine_x[k] = x[k];
        int count;
        unsigned bits = lp_candidates<L, V>(x, lane_max, s.m, A.top, lane, count);
        int at = group + lp_before_me<L>(__popc(bits));
        lp_wave_sync();
        while (__any(bits != 0)) {
            if (bits) {
                const int k = __clz(bits) - (32 - N);
                bits &= ~(0x80000000u >> __clz(bits));
                lds_v[at] = mine_x[k];
                lds_i[at++] = min(((k / V) * L + sub) * V, last) + k % V;
            }
        }
        lp_wave_sync();
        const bool some = sub < count;
        const float v = some ? lds_v[group + sub] : -INFINITY;
        const int i = some ? lds_i[group + sub] : LP_NONE + sub;
        int rank = lp_rank<L>(v, i, L == 64 ? count : L);
        if (L == 64 && !some) rank = sub;                // behind all candidates
        if (active && rank < A.top) lp_write_top(A, row, rank, v, i, s, logl);
    }
}

// ---- long rows: W wavefronts take a segment of a row, each of them every W-th tile of it ----
//
// A wavefront keeps its list of alternatives across its lanes.  A tile's columns come after all earlier tiles', so only those
// strictly better than the last alternative listed can enter (k ln(n / k) of n, in random order): a few one by one, many -- the first
// tile's, and those of rows that rise -- as a list of the tile's own that is merged in.
constexpr int LP_E = 16;                                   // columns per lane and tile
constexpr int LP_TILE = 64 * LP_E;
// columns that enter a list one by one, more as a list of their own (1500 x 50021 float32, 20 alternatives: with 4 98 us, 12 71, 24 66,
// 48 67; 20000 x 2000: 60, 60, 52, 52)
constexpr int LP_FEW = 24;
constexpr int LP_SPLITS = 64;                              // at most: one list per lane when they are joined

struct LpPart {                                            // a segment's result in the workspace
    float m, l, e, pad;
};

// How many of a sorted list's `top` entries come before (v, i)
__device__ __forceinline__ int lp_search(const float* lv, const int* li, int top, float v, int i)
{
    int at = 0;
#pragma unroll
    for (int d = 64; d; d >>= 1)
        if (at + d <= top && lp_before(lv[at + d - 1], li[at + d - 1], v, i)) at += d;
    return at;
}

template <int E, int W, bool TOP>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(6))) void k_logprobs_long(LpArgs A, int splits, int segment,
                                                                                              LpPart* __restrict__ parts,
                                                                                              float* __restrict__ part_v, int* __restrict__ part_i)
{
    using raw = typename Elem<E>::raw;
    constexpr int V = E == 0 ? 4 : 8, NV = LP_E / V;
    __shared__ float lds_v[TOP ? 256 : 1];
    __shared__ int lds_i[TOP ? 256 : 1];
    __shared__ LpPart lds_s[4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const long unit = W == 4 ? (long)blockIdx.x : (long)blockIdx.x * 4 + wave;
    if (W == 1 && unit >= A.rows) return;
    const long row = W == 4 ? unit / splits : unit;
    const int split = W == 4 ? (int)(unit - row * splits) : 0;
    const int c0 = split * segment, c1 = min(A.cols, c0 + segment);
    const raw* p = (const raw*)A.x + row * A.xstride;
    const uint8_t* valid = A.valid ? A.valid + row * A.vstride : nullptr;
    const float given = splits == 1 ? lp_given<E>(A, row) : 0.0f;
    LpStat s, low;
    LpList t;
    float worst = -INFINITY;                               // the last alternative of the tiles before
    for (int base = c0 + (W == 4 ? wave : 0) * LP_TILE; base < c1; base += W * LP_TILE) {
        // the loads are issued before the first is used; a vector that would pass the row's end starts V columns before it, and its
        // columns in front of the lane's own are another lane's (rows of this kernel are longer than a vector)
        float x[LP_E];
        {
            ElemVec<E, V> u[NV];
            const int last = A.cols - V;
#pragma unroll
            for (int q = 0; q < NV; q++) __builtin_memcpy(&u[q], p + min(base + (q * 64 + lane) * V, last), sizeof(u[q]));
            unsigned ok[LP_E / 4];                         // a byte per column
            if (valid) {
#pragma unroll
                for (int q = 0; q < NV; q++) __builtin_memcpy(&ok[q * V / 4], valid + min(base + (q * 64 + lane) * V, last), V);
            }
#pragma unroll
            for (int k = 0; k < LP_E; k++) x[k] = elem_to_float<E>(u[k / V].a[k % V]);
            if (valid) {
#pragma unroll
                for (int k = 0; k < LP_E; k += 4) lp_mask4(x[k], x[k + 1], x[k + 2], x[k + 3], ok[k / 4]);
            }
            if (base + LP_TILE > A.cols) {
#pragma unroll
                for (int k = 0; k < LP_E; k++) {
                    const int c = base + ((k / V) * 64 + lane) * V;
                    x[k] = min(c, last) + k % V >= c ? x[k] : -INFINITY;
                }
            }
        }
        float lane_max = -INFINITY;
#pragma unroll
        for (int k = 0; k < LP_E; k++) lane_max = fmaxf(lane_max, x[k]);
        lp_raise(s, low, fmaxf(s.m, lane_max), A.c2);
        lp_tile(s, low, x, A.c2);
        if constexpr (TOP) {
            if (__any(lane_max > worst)) {
                const int last = A.cols - V;
                // more than a few: the tile's own list, by threshold and rank as a short row's, and the two lists merged
                if (lp_count<64>(__popc(lp_at_least(x, fmaxf(worst, -FLT_MAX)))) <= LP_FEW) {
                    const float bar = worst;
#pragma unroll
                    for (int k = 0; k < LP_E; k++) {
                        unsigned long long better = __ballot(x[k] > bar);
                        while (better) {
                            const int src = __ffsll((long long)better) - 1;
                            better &= better - 1;
                            lp_insert(t, lp_lane(x[k], src), min(base + ((k / V) * 64 + src) * V, last) + k % V, lane);
                        }
                    }
                } else {
                    float* wv = lds_v + wave * 64;
                    int* wi = lds_i + wave * 64;
                    int count;
                    const unsigned enter = lp_candidates<64, V>(x, lane_max, lp_max<64>(lane_max), A.top, lane, count);
                    int at = lp_before_me<64>(__popc(enter));
#pragma unroll
                    for (int k = 0; k < LP_E; k++)
                        if (enter & (1u << (LP_E - 1 - k))) {
                            wv[at] = x[k];
                            wi[at++] = min(base + ((k / V) * 64 + lane) * V, last) + k % V;
                        }
                    lp_wave_sync();
                    const bool some = lane < count;
                    float v = some ? wv[lane] : -INFINITY;
                    int i = some ? wi[lane] : LP_NONE + 64 + lane;
                    lp_wave_sync();
                    int rank = some ? lp_rank<64>(v, i, count) : lane;             // in the tile's list
                    if (__any(t.v != -INFINITY)) {
                        wv[lane] = t.v;
                        wi[lane] = t.i = t.i < LP_NONE ? t.i : LP_NONE + lane;
                        lp_wave_sync();
                        rank += lp_search(wv, wi, 64, v, i);                       // in both
                        lp_wave_sync();
                        const int mine = some ? rank : 64;                         // my column's place; the list's own entries move
                        wv[lane] = -INFINITY;                                      // behind those of the tile that come before them
                        wi[lane] = LP_NONE + lane;
                        lp_wave_sync();
                        int before = 0;
                        for (int k = 0; k < count; k++) {
                            const float w = lp_lane(v, k);
                            const int j = lp_lane(i, k);
                            before += lp_before(w, j, t.v, t.i);
                        }
                        if (lane + before < 64) {
                            wv[lane + before] = t.v;
                            wi[lane + before] = t.i;
                        }
                        rank = mine;
                    }
                    if (rank < 64) {
                        wv[rank] = v;
                        wi[rank] = i;
                    }
                    lp_wave_sync();
                    t.v = wv[lane];
                    t.i = wi[lane];
                    lp_wave_sync();
                }
                worst = lp_lane(t.v, A.top - 1);
            }
        }
    }
    s = lp_wave_join(s, A.c2);
    if constexpr (W == 1) {
        const float logl = logf(s.l);
        if (lane == 0) lp_write_row(A, row, s, logl, given);
        if (TOP && lane < A.top) lp_write_top(A, row, lane, t.v, t.i, s, logl);
        return;
    }
    __syncthreads();                                   // all waves' first tiles are done with the LDS arrays
    if (lane == 0) lds_s[wave] = LpPart{ s.m, s.l, s.e, 0.0f };
    if (TOP && lane < A.top) {
        lds_v[wave * A.top + lane] = t.v;
        lds_i[wave * A.top + lane] = t.i = t.i < LP_NONE ? t.i : LP_NONE + (int)threadIdx.x;     // (no two entries the same)
    }
    __syncthreads();
    s = LpStat();
    if (lane < 4) {
        s.m = lds_s[lane].m;
        s.l = lds_s[lane].l;
        s.e = lds_s[lane].e;
    }
    s = lp_wave_join(s, A.c2);
    const float logl = logf(s.l);
    if (threadIdx.x == 0) {
        if (splits == 1) lp_write_row(A, row, s, logl, given);
        else parts[unit] = LpPart{ s.m, s.l, s.e, 0.0f };
    }
    // the four lists together: an entry's place is its place in its own and the numbers of the others' entries before it
    if (TOP && lane < A.top) {
        int rank = lane;
#pragma unroll
        for (int k = 1; k < 4; k++) {
            const int w = (wave + k) & 3;
            rank += lp_search(lds_v + w * A.top, lds_i + w * A.top, A.top, t.v, t.i);
        }
        if (rank < A.top) {
            if (splits == 1) lp_write_top(A, row, rank, t.v, t.i, s, logl);
            else {
                part_v[unit * A.top + rank] = t.v;
                part_i[unit * A.top + rank] = t.i;
            }
        }
    }
}

// The segments of a row together: one workgroup per row.  The lists come to LDS; of every list's entry number j (j as small as
// `top` entries allow) the r-th largest is reached by `top` entries or more, few of them in general: they are the beginnings of their
// lists, and are ranked as a short row's candidates are.
template <int E, bool TOP>
__global__ __launch_bounds__(256) void k_logprobs_join(LpArgs A, int splits, const LpPart* __restrict__ parts, const float* __restrict__ part_v,
                                                       const int* __restrict__ part_i)
{
    __shared__ float lds_v[TOP ? LP_SPLITS * LP_TOP : 1], cand_v[TOP ? 64 : 1];
    __shared__ int lds_i[TOP ? LP_SPLITS * LP_TOP : 1], cand_i[TOP ? 64 : 1];
    const long row = blockIdx.x;
    const int lane = threadIdx.x & 63, top = A.top;
    if constexpr (TOP) {
        for (int k = threadIdx.x; k < splits * top; k += 256) {
            lds_v[k] = part_v[row * splits * top + k];
            const int i = part_i[row * splits * top + k];
            lds_i[k] = i < LP_NONE ? i : LP_NONE + k;
        }
    }
    LpStat s;
    if (lane < splits) {
        const LpPart q = parts[row * splits + lane];
        s.m = q.m;
        s.l = q.l;
        s.e = q.e;
    }
    const float given = lp_given<E>(A, row);
    s = lp_wave_join(s, A.c2);
    const float logl = logf(s.l);
    if (threadIdx.x == 0) lp_write_row(A, row, s, logl, given);
    if constexpr (TOP) {
        __syncthreads();
        if (threadIdx.x >= 64) return;
        const int j = (top - 1) / splits, r = (top + j) / (j + 1);             // r lists with j + 1 entries each: r <= splits
        const float T = lp_threshold<64>(lane < splits ? lds_v[lane * top + j] : -INFINITY, r, lane);
        // entries of this lane's list that come before (t, i)
        const auto reach = [&](float t, int i) { return lane < splits ? lp_search(lds_v + lane * top, lds_i + lane * top, top, t, i) : 0; };
        int mine = reach(T, LP_NONE), count = lp_count<64>(mine);      // those that are >= T
        if (count > 64) {                                  // halved as in lp_candidates: values, then columns of one value
            const auto halve = [&](int lo, int hi, auto&& before) {
                while (count > 64 && (unsigned)hi - (unsigned)lo > 1u) {
                    const int mid = __builtin_amdgcn_readfirstlane((int)((unsigned)lo + (((unsigned)hi - (unsigned)lo) >> 1)));
                    const int m = before(mid), n = lp_count<64>(m);
                    if (n >= top) {
                        lo = mid;
                        mine = m;
                        count = n;
                    } else hi = mid;
                }
                return lo;
            };
            const int lo = halve(lp_key(__float_as_int(T)), lp_key(__float_as_int(s.m)) + 1,
                                 [&](int mid) { return reach(__int_as_float(lp_key(mid)), LP_NONE); });
            halve(-LP_NONE, 0, [&](int mid) { return reach(__int_as_float(lp_key(lo)), -mid); });      // (the fewer, the larger mid)
        }
        const int at = lp_before_me<64>(mine);
        for (int k = 0; k < mine; k++) {
            cand_v[at + k] = lds_v[lane * top + k];
            cand_i[at + k] = lds_i[lane * top + k];
        }
        lp_wave_sync();
        const float v = lane < count ? cand_v[lane] : -INFINITY;
        const int i = lane < count ? cand_i[lane] : LP_NONE + lane;
        int rank = lp_rank<64>(v, i, count);
        if (lane >= count) rank = lane;
        if (rank < top) lp_write_top(A, row, rank, v, i, s, logl);
    }
}

struct LpGradArgs {
    const void* x;
    long xstride;
    const uint8_t* valid;
    long vstride;
    const int* actions;
    LpFactor inv_t;                        // as the forward pass has it: log p of the only column is 0 again
    const float *lse, *entropy, *g, *h;
    void* dx;
    long dstride;
    long rows;
    int cols;
};

// One pass: L lanes a row, up to LG_N vectors of V columns each; L = 256: workgroups (row, chunk of a long row).  Bound by reading the
// logits and the mask and writing the gradient.  The logits may be the output: a lane writes the columns that it alone reads.
constexpr int LG_N = 4;

template <int E, int L, int V> __global__ __launch_bounds__(256) void k_logprobs_grad(LpGradArgs A, int chunks)
{
    using raw = typename Elem<E>::raw;
    const int sub = threadIdx.x & (L - 1);
    long row;
    int c0 = 0;
    if constexpr (L == 256) {
        row = blockIdx.x / chunks;
        c0 = (int)(blockIdx.x - row * chunks) * (LG_N * L * V);
    } else {
        row = (long)blockIdx.x * (256 / L) + threadIdx.x / L;
        if (row >= A.rows) return;
    }
    const raw* x = (const raw*)A.x + row * A.xstride;
    raw* dx = (raw*)A.dx + row * A.dstride;
    // a vector that would pass the row's end is read from V columns before it (cols >= V)
    const int last = A.cols - V;
    ElemVec<E, V> u[LG_N];
#pragma unroll
    for (int q = 0; q < LG_N; q++)
        if (c0 + q * L * V < A.cols) __builtin_memcpy(&u[q], x + min(c0 + (q * L + sub) * V, last), sizeof(u[q]));
    uint8_t ok[LG_N][V];
    if (A.valid) {
        const uint8_t* valid = A.valid + row * A.vstride;
#pragma unroll
        for (int q = 0; q < LG_N; q++)
            if (c0 + q * L * V < A.cols) __builtin_memcpy(ok[q], valid + min(c0 + (q * L + sub) * V, last), V);
    } else {
#pragma unroll
        for (int k = 0; k < LG_N * V; k++) ok[k / V][k % V] = 1;
    }
    const int a = A.actions ? A.actions[row] : -1;
    const float lse = A.lse[row], H = A.h ? A.entropy[row] : 0.0f, h = A.h ? A.h[row] : 0.0f;
    const float g = a < 0 ? 0.0f : a >= A.cols ? NAN : A.g[row], scale = A.inv_t.hi + A.inv_t.lo;
#pragma unroll
    for (int q = 0; q < LG_N; q++) {
        const int c = c0 + (q * L + sub) * V, cc = min(c, last);
        if (c >= A.cols) break;
        float d[V];
#pragma unroll
        for (int k = 0; k < V; k++) {
            const float v = elem_to_float<E>(u[q].a[k]);
            const float lp = __builtin_amdgcn_fmed3f(lp_times(v, A.inv_t), -FLT_MAX, FLT_MAX) - lse, p = __builtin_amdgcn_exp2f(lp * LOG2E);
            // p log p is 0 at p = 0, also where log p is -inf
            const float t = fmaf(h, p * fmaxf(lp + H, -1000.0f), g * p);
            d[k] = ok[q][k] && v != -INFINITY ? ((cc + k == a ? g : 0.0f) - t) * scale : 0.0f;
        }
        if (c == cc) elem_store<E, V>(dx + c, d);
        else {
#pragma unroll
            for (int k = 0; k < V; k++)
                if (cc + k >= c) dx[cc + k] = elem_from_float<E>(d[k]);
        }
    }
}

static LpFactor lp_factor(double c)
{
    float hi = (float)c;
    if ((double)hi >= c) hi = nextafterf(hi, 0.0f);
    return LpFactor{ hi, (float)(c - (double)hi) };
}

#define LP_DISPATCH(elem, ...)                                       \
    switch (elem) {                                                  \
        case 0: { constexpr int E = 0; __VA_ARGS__; } break;         \
        case 1: { constexpr int E = 1; __VA_ARGS__; } break;         \
        default: { constexpr int E = 2; __VA_ARGS__; } break;        \
    }

constexpr int LP_SHORT = 384;                       // longest row that stays in registers (30000 x 1000 float32: 28 us there, 23 below)

// Long rows: from LP_MANY rows on they fill the GPU a wavefront each (20000 x 2000 float32, 5 alternatives: 40 us, with four wavefronts a
// row 85; 2048 x 40000: 67 and 70; 1024 x 40000: 56 and 37); fewer rows take four wavefronts a segment, in as many segments as fill
// it (LP_FILL; 5 x 128001: 18.5 us, with 256 21.4; 700 x 8000: 15 us, with 1024, which splits the rows, 18).  A segment is a multiple of four tiles, one for each.
constexpr int64_t LP_MANY = 2048, LP_FILL = 512;
static int lp_segment(int64_t rows, int cols)
{
    const int64_t want = std::min<int64_t>((LP_FILL + rows - 1) / rows, LP_SPLITS), unit = 4 * LP_TILE;
    return (int)(((cols + want - 1) / want + unit - 1) / unit * unit);
}
static int lp_splits(int64_t rows, int cols) { return cols <= LP_SHORT ? 1 : (cols - 1) / lp_segment(rows, cols) + 1; }

int64_t action_logprobs_workspace(int64_t rows, int cols, int top)
{
    const int64_t splits = lp_splits(std::max<int64_t>(rows, 1), cols);
    return splits == 1 ? 0 : rows * splits * (int64_t)(sizeof(LpPart) + 8 * top);
}

constexpr long LP_GRID = 1 << 22;                   // workgroups per launch

// f(arguments of some rows), at most `most` rows at a time
template <int E, class F> static void lp_chunks(LpArgs A, long most, F&& f)
{
    for (long left = A.rows; left > 0; left -= A.rows) {
        A.rows = std::min(left, most);
        f(A);
        A.x = (const char*)A.x + A.rows * A.xstride * (long)sizeof(typename Elem<E>::raw);
        if (A.valid) A.valid += A.rows * A.vstride;
        if (A.actions) A.actions += A.rows;
        if (A.logp) A.logp += A.rows;
        if (A.entropy) A.entropy += A.rows;
        if (A.lse) A.lse += A.rows;
        if (A.top) {
            A.top_actions += A.rows * A.top;
            A.top_logp += A.rows * A.top;
        }
    }
}

template <int E, int L, int V, int NV, int FULL> static void lp_launch_short(const LpArgs& all, hipStream_t st)
{
    const long per = 256 / L;
    lp_chunks<E>(all, LP_GRID * per, [&](const LpArgs& A) {
        const unsigned grid = (unsigned)((A.rows + per - 1) / per);
        if (A.top) k_logprobs_short<E, L, V, NV, FULL, true><<<grid, 256, 0, st>>>(A);
        else k_logprobs_short<E, L, V, NV, FULL, false><<<grid, 256, 0, st>>>(A);
    });
}

template <int E> static void lp_launch(const LpArgs& A, void* workspace, hipStream_t st)
{
    // sixteen lanes per row: up to eight alternatives (of sixteen lanes' maxima the eighth is still a sharp threshold; 65536 x 362
    // bfloat16: 21 us, with a wavefront per row 46; 300000 x 82 float32: 48 and 145); more: a wavefront per row
    if (A.cols <= LP_SHORT && A.top <= 8) {
        if (A.cols <= 32) lp_launch_short<E, 16, 1, 2, 0>(A, st);
        else if (A.cols <= 64) lp_launch_short<E, 16, 4, 1, 0>(A, st);
        else if (A.cols <= 128) lp_launch_short<E, 16, 4, 2, 1>(A, st);
        else if (A.cols <= 192) lp_launch_short<E, 16, 4, 3, 2>(A, st);
        else lp_launch_short<E, 16, 4, 6, 3>(A, st);
    } else if (A.cols <= LP_SHORT) {
        if (A.cols <= 128) lp_launch_short<E, 64, 1, 2, 0>(A, st);
        else lp_launch_short<E, 64, 1, 6, 2>(A, st);
    } else {
        const int segment = lp_segment(A.rows, A.cols), splits = lp_splits(A.rows, A.cols);
        LpPart* parts = (LpPart*)workspace;
        float* pv = (float*)(parts + A.rows * splits);
        int* pi = (int*)(pv + A.rows * splits * A.top);
        // (splits > 1 only for fewer than LP_FILL rows: one round)
        const bool many = A.rows >= LP_MANY;
        lp_chunks<E>(A, LP_GRID, [&](const LpArgs& B) {
            const unsigned grid = many ? (unsigned)((B.rows + 3) / 4) : (unsigned)(B.rows * splits);
            if (many && B.top) k_logprobs_long<E, 1, true><<<grid, 256, 0, st>>>(B, 1, B.cols, parts, pv, pi);
            else if (many) k_logprobs_long<E, 1, false><<<grid, 256, 0, st>>>(B, 1, B.cols, parts, pv, pi);
            else if (B.top) k_logprobs_long<E, 4, true><<<grid, 256, 0, st>>>(B, splits, segment, parts, pv, pi);
            else k_logprobs_long<E, 4, false><<<grid, 256, 0, st>>>(B, splits, segment, parts, pv, pi);
        });
        if (splits == 1) return;
        if (A.top) k_logprobs_join<E, true><<<(unsigned)A.rows, 256, 0, st>>>(A, splits, parts, pv, pi);
        else k_logprobs_join<E, false><<<(unsigned)A.rows, 256, 0, st>>>(A, splits, parts, pv, pi);
    }
}

int launch_action_logprobs(const void* logits, int elem, int64_t stride, const uint8_t* valid, int64_t valid_stride, const int32_t* actions,
                           double temperature, int top, float* logp, float* entropy, float* lse, int32_t* top_actions, float* top_logp,
                           int64_t rows, int cols, void* workspace, hipStream_t st)
{
    const LpArgs A{ logits, (long)stride, valid, (long)valid_stride, actions, lp_factor(1.0 / temperature),
                    lp_factor(1.44269504088896340736 / temperature), top, logp, entropy, lse, top_actions, top_logp, (long)rows, cols };
    LP_DISPATCH(elem, lp_launch<E>(A, workspace, st));
    GOAI_HIP_CHECK(hipGetLastError());
    return GOAI_OK;
}

template <int E, int L, int V> static void lp_launch_grad(LpGradArgs A, hipStream_t st)
{
    const int chunks = L == 256 ? (A.cols + LG_N * L * V - 1) / (LG_N * L * V) : 1;
    const long most = std::max<long>(1, LP_GRID / chunks) * (256 / L);
    for (long left = A.rows; left > 0; left -= A.rows) {
        A.rows = std::min(left, most);
        k_logprobs_grad<E, L, V><<<(unsigned)(L == 256 ? A.rows * chunks : (A.rows + 256 / L - 1) / (256 / L)), 256, 0, st>>>(A, chunks);
        const long size = sizeof(typename Elem<E>::raw);
        A.x = (const char*)A.x + A.rows * A.xstride * size;
        A.dx = (char*)A.dx + A.rows * A.dstride * size;
        if (A.valid) A.valid += A.rows * A.vstride;
        if (A.actions) A.actions += A.rows;
        A.lse += A.rows;
        if (A.entropy) A.entropy += A.rows;
        if (A.g) A.g += A.rows;
        if (A.h) A.h += A.rows;
    }
}
template <int E> static void lp_launch_grad(const LpGradArgs& A, hipStream_t st)
{
    constexpr int V = E == 0 ? 4 : 8;                   // 16 bytes; 8 of a short row, which has few vectors for its lanes (300000 x 26
    if (A.cols < 4) lp_launch_grad<E, 16, 1>(A, st);    // bfloat16: 21 us, with 16 bytes 30)
    else if (A.cols <= LG_N * 16 * 4) lp_launch_grad<E, 16, 4>(A, st);
    // lanes a row: 50000 x 362 bfloat16 20 us with 16, 22 with 64; 30000 x 1500 38 us with 64, 49 with 256
    else if (A.cols <= LG_N * 16 * V) lp_launch_grad<E, 16, V>(A, st);
    else if (A.cols <= LG_N * 64 * V) lp_launch_grad<E, 64, V>(A, st);
    else lp_launch_grad<E, 256, V>(A, st);
}

int launch_action_logprobs_grad(const void* logits, int elem, int64_t stride, const uint8_t* valid, int64_t valid_stride,
                                const int32_t* actions, double temperature, const float* lse, const float* entropy, const float* d_logp,
                                const float* d_entropy, void* d_logits, int64_t d_stride, int64_t rows, int cols, hipStream_t st)
{
    LpGradArgs A{ logits, (long)stride, valid, (long)valid_stride, d_logp ? actions : nullptr, lp_factor(1.0 / temperature), lse, entropy, d_logp,
                  d_entropy, d_logits, (long)d_stride, (long)rows, cols };
    LP_DISPATCH(elem, lp_launch_grad<E>(A, st));
    GOAI_HIP_CHECK(hipGetLastError());
    return GOAI_OK;
}

}  // namespace goai
