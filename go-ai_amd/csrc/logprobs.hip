// logprobs.hip -- log probabilities of given actions under a policy's logits, with the entropy and the best alternatives,
// and their gradient.
//
//   s_j = x_j / T over the allowed columns j (valid[j] != 0 and x_j > -inf)
//   lse = log sum_j exp(s_j),  log p_a = s_a - lse,  H = -sum_j p_j log p_j
//   d x_j = (g (delta_aj - p_j) - h p_j (log p_j + H)) / T        for a loss with d/d log p_a = g, d/dH = h
//
// The forward pass reads the logits once: every lane keeps the maximum m of the logits it has seen and, with t = (x - m) c,
// c = log2(e) / T, the sums l = sum 2^t and e = sum 2^t t; a maximum larger by d / c scales l by 2^-d and turns e into
// 2^-d (e - d l).  All terms of e have one sign, so H = ln 2 (log2 l - e / l) loses nothing to cancellation.  Sums are float32.
// A lane without columns has m = -FLT_MAX, l = e = 0: x - m is then never inf - inf, and l == 0 says that a row has no allowed
// column.  t may be -inf (a column that is not allowed, or an overflow): its power is 0, and t is bounded in front of the product.
#include <float.h>
#include <math.h>

#include <algorithm>

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

// the statistics of all lanes' columns together
__device__ __forceinline__ LpStat lp_wave_join(LpStat s, LpFactor c)
{
    float m = s.m;
    for (int d = 1; d < 64; d <<= 1) m = fmaxf(m, __shfl_xor(m, d));
    lp_raise(s, m, c);
    for (int d = 1; d < 64; d <<= 1) {
        s.l += __shfl_xor(s.l, d);
        s.e += __shfl_xor(s.e, d);
    }
    return s;
}

// One wavefront's best columns, best first, one per lane: larger logit, then lower column.
struct LpList {
    float v = -INFINITY;
    int i = 0x7fffffff;
};

__device__ __forceinline__ void lp_insert(LpList& t, float cv, int ci, int lane)
{
    const unsigned long long before = __ballot(t.v > cv || (t.v == cv && t.i < ci));
    const int pos = __popcll(before);
    const float sv = __shfl_up(t.v, 1);
    const int si = __shfl_up(t.i, 1);
    if (lane == pos) { t.v = cv; t.i = ci; }
    else if (lane > pos) { t.v = sv; t.i = si; }
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

// a row's outputs from its statistics (one wavefront; `t`: its list, best first)
template <int E>
__device__ __forceinline__ void lp_finish(const LpArgs& A, long row, LpStat s, const LpList& t, int lane)
{
    using raw = typename Elem<E>::raw;
    const bool none = s.l == 0.0f;                               // no allowed column
    const float logl = logf(s.l);
    const float lse = none ? -INFINITY : __builtin_amdgcn_fmed3f(lp_times(s.m, A.inv_t), -FLT_MAX, FLT_MAX) + logl;
    if (lane == 0) {
        if (A.lse) A.lse[row] = lse;
        if (A.entropy) A.entropy[row] = none ? 0.0f : logl - LN2 * (s.e / s.l);
        if (A.logp) {
            const int a = A.actions[row];
            float r = 0.0f;
            if (a >= A.cols) r = NAN;
            else if (a >= 0) {
                const float x = elem_to_float<E>(((const raw*)A.x)[row * A.xstride + a]);
                const bool there = x != -INFINITY && (!A.valid || A.valid[row * A.vstride + a]);
                r = there ? lp_times(x - s.m, A.inv_t) - logl : -INFINITY;
            }
            A.logp[row] = r;
        }
    }
    if (lane < A.top) {
        const bool some = t.v != -INFINITY;
        A.top_actions[row * A.top + lane] = some ? t.i : -1;
        A.top_logp[row * A.top + lane] = some ? lp_times(t.v - s.m, A.inv_t) - logl : -INFINITY;
    }
}

// One wavefront per row.
template <int E> __global__ __launch_bounds__(256) void k_logprobs(LpArgs A)
{
    using raw = typename Elem<E>::raw;
    const int lane = threadIdx.x & 63;
    for (long row = (long)blockIdx.x * 4 + (threadIdx.x >> 6); row < A.rows; row += (long)gridDim.x * 4) {
    const raw* x = (const raw*)A.x + row * A.xstride;
    const uint8_t* valid = A.valid ? A.valid + row * A.vstride : nullptr;
    LpStat s;
    LpList t;
    float worst = -INFINITY;                        // the last alternative listed so far: later columns must beat it
    for (int base = 0; base < A.cols; base += 64) {
        const int c = base + lane;
        const bool in = c < A.cols;
        const float v = in && (!valid || valid[c]) ? elem_to_float<E>(x[c]) : -INFINITY;
        if (v > s.m) lp_raise(s, v, A.c2);
        lp_add(s, v, A.c2);
        if (A.top) {
            unsigned long long better = __ballot(v > worst);
            while (better) {
                const int src = __ffsll((long long)better) - 1;
                better &= better - 1;
                lp_insert(t, __shfl(v, src), base + src, lane);
            }
            worst = __shfl(t.v, A.top - 1);
        }
    }
    s = lp_wave_join(s, A.c2);
    lp_finish<E>(A, row, s, t, lane);
    }
}

struct LpGradArgs {
    const void* x;
    long xstride;
    const uint8_t* valid;
    long vstride;
    const int* actions;
    float inv_t;
    const float *lse, *entropy, *g, *h;
    void* dx;
    long dstride;
    long rows;
    int cols;
};

template <int E> __device__ __forceinline__ float lp_grad_of(float x, bool ok, bool hot, float inv_t, float lse, float H, float g, float h)
{
    if (!ok || x == -INFINITY) return 0.0f;
    const float lp = __builtin_amdgcn_fmed3f(x * inv_t, -FLT_MAX, FLT_MAX) - lse, p = __builtin_amdgcn_exp2f(lp * LOG2E);
    const float pl = p > 0.0f ? p * (lp + H) : (p == 0.0f ? 0.0f : p);        // (NaN stays)
    return ((hot ? g : 0.0f) - g * p - h * pl) * inv_t;
}

template <int E> __global__ __launch_bounds__(256) void k_logprobs_grad(LpGradArgs A)
{
    using raw = typename Elem<E>::raw;
    const int lane = threadIdx.x & 63;
    for (long row = (long)blockIdx.x * 4 + (threadIdx.x >> 6); row < A.rows; row += (long)gridDim.x * 4) {
    const raw* x = (const raw*)A.x + row * A.xstride;
    raw* dx = (raw*)A.dx + row * A.dstride;
    const uint8_t* valid = A.valid ? A.valid + row * A.vstride : nullptr;
    const int a = A.actions ? A.actions[row] : -1;
    const float lse = A.lse[row], H = A.h ? A.entropy[row] : 0.0f, h = A.h ? A.h[row] : 0.0f;
    const float g = a < 0 ? 0.0f : a >= A.cols ? NAN : A.g[row];
    for (int c = lane; c < A.cols; c += 64)
        dx[c] = elem_from_float<E>(lp_grad_of<E>(elem_to_float<E>(x[c]), !valid || valid[c], c == a, A.inv_t, lse, H, g, h));
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

int launch_action_logprobs(const void* logits, int elem, int64_t stride, const uint8_t* valid, int64_t valid_stride, const int32_t* actions,
                           double temperature, int top, float* logp, float* entropy, float* lse, int32_t* top_actions, float* top_logp,
                           int64_t rows, int cols, hipStream_t st)
{
    const LpArgs A{ logits, (long)stride, valid, (long)valid_stride, actions, lp_factor(1.0 / temperature), lp_factor(1.44269504088896340736 / temperature), top, logp, entropy, lse, top_actions, top_logp,
                    (long)rows, cols };
    LP_DISPATCH(elem, k_logprobs<E><<<(unsigned)std::min<int64_t>((rows + 3) / 4, 1 << 20), 256, 0, st>>>(A));
    GOAI_HIP_CHECK(hipGetLastError());
    return GOAI_OK;
}

int launch_action_logprobs_grad(const void* logits, int elem, int64_t stride, const uint8_t* valid, int64_t valid_stride,
                                const int32_t* actions, double temperature, const float* lse, const float* entropy, const float* d_logp,
                                const float* d_entropy, void* d_logits, int64_t d_stride, int64_t rows, int cols, hipStream_t st)
{
    const LpGradArgs A{ logits, (long)stride, valid, (long)valid_stride, d_logp ? actions : nullptr, (float)(1.0 / temperature), lse, entropy, d_logp,
                        d_entropy, d_logits, (long)d_stride, (long)rows, cols };
    LP_DISPATCH(elem, k_logprobs_grad<E><<<(unsigned)std::min<int64_t>((rows + 3) / 4, 1 << 20), 256, 0, st>>>(A));
    GOAI_HIP_CHECK(hipGetLastError());
    return GOAI_OK;
}

}  // namespace goai
