// adamw.hip -- one AdamW step over many tensors in one launch, the moments in 32 or in 8 bits, and the gradients' global
// norm with its clipping coefficient.
//
//   g' = k g,  k = min(1, max_norm / |g|)      (|g| over all tensors; without clipping k = 1)
//   m  = b1 m + (1 - b1) g',   v = b2 v + (1 - b2) g'^2
//   p  = p (1 - lr wd) - (lr / (1 - b1^t)) m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// A step whose norm is not finite is skipped, and is no step of the bias corrections: t counts the others.  Only the GPU knows them in time, so
// the corrections of a step that may be skipped, or that follows one, are computed there.
//
// All of it is float32, every operation rounded on its own (the library is built with -ffp-contract=off), so that a moment
// in 8 bits is the same code wherever the step is computed.  The norm is summed in float64: a code next to the border of two
// would follow the last bit of k.
//
// Moments in 8 bits are held in blocks of AW_BLOCK elements (no block spans two tensors) with one float32 scale each:
//   m: e4m3 codes of m / scale, scale = largest |m| of the block / 448 (half a step: 2^-4 of the value, above 2^-15 of the largest);
//   v: codes of its root r = sqrt(v), c = 1 .. 255 for the float32 with the bits (c + AW_LEVEL0) << 19 (four exponent and four
//      fraction bits, the largest r of the block is 1.0 = code 255; half a step: 2^-5 of r), 0 for r = 0.  A root that is not zero
//      never becomes 0: m / (0 + eps) would throw the parameter away.
// The update itself uses the moments before they are rounded.  A block whose largest value is below 2^-100 is held as zeros.
//
// Rounding them to the nearest code every step would lose every change below half a code, and with beta2 = 0.999 a step moves a root by
// 0.05 % where half a code is 2^-5: a code would stand still while its block's largest root does and follow that one's scale
// otherwise (elements whose gradients fall tenfold keep a v 80 times too large 7000 steps later; the other elements of a block whose largest
// falls silent end at 0.13 of theirs), and a first moment of four steps of e4m3's smallest would stay for good.  So codes are rounded
// at random, with the expectation right: the lower code's or the upper's, as often as the value is near to it.  A root then scatters about its own
// value by sqrt(step / 2), 0.15 to 0.17 of it, with beta2's memory (v: 1/3), and its mean stays within a few percent.  The first AW_NEAREST = 16
// steps after the moments were set go to the nearest, which has half the error: while 1 / t is at least half a code of e4m3 (2^-4) the newest
// gradient's weight in fresh moments, (1 - beta) / (1 - beta^t) >= 1 / t, moves a code by itself, and 16 steps of loaded roots lose at most 16 of
// those 0.05 % (of loaded first moments what 16 steps move them by, which the steps behind make up for).  The random numbers are a hash of the step's number since then and the element: the same steps give the same bits.
#include <float.h>
#include <math.h>
#include <string.h>

#include <algorithm>
#include <new>
#include <vector>

#include "ctx.h"
#include "elem.h"
#include "goai_internal.h"

namespace goai {

constexpr int AW_BLOCK = 256;          // elements per scale of an 8-bit moment: eight on each of 32 lanes
constexpr int AW_CHUNK = 2048;         // elements per workgroup: eight per thread
constexpr int AW_LEVEL0 = 1777;        // (255 + AW_LEVEL0) << 19 is 1.0f
constexpr float AW_SMALLEST = 0x1p-100f;
constexpr int AW_LAUNCH = 256;         // tensors per launch: their gradients' addresses travel in the launch's arguments
constexpr int AW_NEAREST = 16;         // steps whose 8-bit moments are rounded to the nearest (above)
constexpr int AW_NORM_BLOCKS = 1024;   // workgroups (and float64 partial sums) of the norm (97 M: 599 us a step, with 512 or 2048 605)

struct AwTensor {
    void* p;
    long start, n;           // first element in the moments' flat arrays (a multiple of AW_BLOCK); elements
    float decay;
    int ptype, gtype;        // GOAI_ELEM_*
};
struct AwState {             // flat arrays over all tensors: float32, or codes and one scale per block
    void *m, *v;
    float *ms, *vs;
};
struct AwChunk {
    int tensor, chunk;
};
struct AwGrads {
    const void* g[AW_LAUNCH];
};
struct AwScal {
    double lr;
    float b1, omb1, b2, omb2, eps, c1, c2;     // c1 = 1 / sqrt(1 - b2^t), c2 = lr / (1 - b1^t)
    unsigned key;                              // of the step's random numbers
    bool random;                               // 8-bit moments are rounded at random
};
// The GPU's count of steps, for those whose number the host does not know when they are launched: the replays of a captured one, and
// steps that are skipped when their gradients' norm is not finite.
struct AwClock {
    long ticks, skipped;                       // since the moments were set
    double c1, c2;                             // the next step's (or the present one's)
    unsigned key;
    int random;
};
struct AwTick {
    AwClock* clock;
    long age, t;                               // steps that the clock does not count; this step's number, skipped ones counted
    double lr, b1, b2;
};

}  // namespace goai

struct goai_adamw {
    int device = 0, bits = 32;
    long elems = 0;                            // of the moments' flat arrays
    goai::AwState state{};
    std::vector<goai::AwTensor> tensors;
    std::vector<int> first;                    // first chunk of each tensor (and the total)
    long age = 0;                              // steps since the moments were set, those that the clock counts aside
    bool ticking = false;                      // there was a step that the clock counts: from then on it counts all
    char* d_mem = nullptr;                     // one allocation: the norm's partial sums, the clock, tensors, chunks
    double* d_partials = nullptr;              // AW_NORM_BLOCKS
    goai::AwClock* d_clock = nullptr;
    goai::AwTensor* d_tensors = nullptr;
    goai::AwChunk* d_chunks = nullptr;
};

namespace goai {

// N neighbouring elements from i on, as floats (zeros from `n` on); tensors are aligned to their element type only.  FULL: all of
// them are inside for sure, and all loads of a thread are in flight together
template <int E, bool FULL = false, int N> __device__ __forceinline__ void aw_load(const void* base, long i, long n, float (&out)[N])
{
    const typename Elem<E>::raw* q = (const typename Elem<E>::raw*)base + i;
    if (FULL || i + N <= n) elem_load<E, N>(q, out);
    else {
#pragma unroll
        for (int k = 0; k < N; k++) out[k] = i + k < n ? elem_to_float<E>(q[k]) : 0.0f;
    }
}
template <int E, bool FULL = false, int N> __device__ __forceinline__ void aw_store(void* base, long i, long n, const float (&x)[N])
{
    typename Elem<E>::raw* q = (typename Elem<E>::raw*)base + i;
    if (FULL || i + N <= n) elem_store<E, N>(q, x);
    else {
#pragma unroll
        for (int k = 0; k < N; k++)
            if (i + k < n) q[k] = elem_from_float<E>(x[k]);
    }
}

// The largest of 32 lanes' floats >= 0, which are ordered as their bits (a NaN above all).
template <int CTRL> __device__ __forceinline__ unsigned aw_dpp(unsigned x) { return (unsigned)__builtin_amdgcn_mov_dpp((int)x, CTRL, 0xf, 0xf, true); }
__device__ __forceinline__ float aw_max32(unsigned x)
{
    x = max(x, aw_dpp<0x128>(x));          // rotations within 16 lanes by 8, 4, 2, 1
    x = max(x, aw_dpp<0x124>(x));
    x = max(x, aw_dpp<0x122>(x));
    x = max(x, aw_dpp<0x121>(x));
    return __uint_as_float(max(x, (unsigned)__shfl_xor((int)x, 16)));
}

// Square roots, correctly rounded: y = 1 / sqrt(x) to an ulp, s = x y, and one correction s + (x - s s) y / 2.  Against sqrtf it gives
// the same for every x from 2^-102 on (the tests compare all significands); sqrtf's own correction steps take twice the instructions.
// 0: y is held finite.  Smaller x, infinities and NaN: sqrtf.
template <int N> __device__ __forceinline__ void aw_sqrt(const float (&x)[N], float (&s)[N])
{
    unsigned least = 0xffffffffu, most = 0;
#pragma unroll
    for (int k = 0; k < N; k++) {
        const unsigned bits = __float_as_uint(x[k]);
        least = min(least, bits - 1);      // 0 counts as the largest
        most = max(most, bits);
    }
    if (__any(least < __float_as_uint(0x1p-100f) || most >= 0x7f800000u)) {
#pragma unroll
        for (int k = 0; k < N; k++) s[k] = sqrtf(x[k]);
    } else {
#pragma unroll
        for (int k = 0; k < N; k++) {
            const float y = __builtin_amdgcn_fmed3f(__builtin_amdgcn_rsqf(x[k]), 0.0f, FLT_MAX), r = x[k] * y;
            s[k] = fmaf(fmaf(-r, r, x[k]), y * 0.5f, r);
        }
    }
}

// ---- random numbers: a lane's eight elements take one word for their first moments and one for their roots, turned by four bits an
// element (the top bits of two neighbours correlate by 1/16), as a bijection of every step's key each uniform by itself ----
__host__ __device__ __forceinline__ unsigned aw_mix(unsigned x)
{
    x = (x ^ (x >> 16)) * 0x9E3779B1u;
    x = (x ^ (x >> 15)) * 0x6A09E667u;
    return x ^ (x >> 16);
}
__host__ __device__ __forceinline__ unsigned aw_key(long age) { return aw_mix((unsigned)age * 0x9E3779B9u + 0x7F4A7C15u); }

struct AwRandom {
    unsigned mean, root;
};
__device__ __forceinline__ AwRandom aw_random(unsigned key, long j)      // j: the first of a lane's eight elements
{
    AwRandom w;
    w.mean = aw_mix((unsigned)(j >> 3) ^ key ^ ((unsigned)(j >> 35) * 0x9E3779B9u));
    w.root = aw_mix(w.mean + 0x9E3779B9u);
    return w;
}

// ---- moments in 8 bits: eight neighbouring codes per lane, a block on 32 lanes; `w`: rounded at random (nullptr: to the nearest) ----
struct AwCodes {
    unsigned w[2];
};
__device__ __forceinline__ void aw_mean_of(AwCodes code, float scale, float (&m)[8])
{
#pragma unroll
    for (int h = 0; h < 2; h++) {
        const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(code.w[h], false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(code.w[h], true);
        m[4 * h] = lo[0] * scale;
        m[4 * h + 1] = lo[1] * scale;
        m[4 * h + 2] = hi[0] * scale;
        m[4 * h + 3] = hi[1] * scale;
    }
}
__device__ __forceinline__ void aw_root_of(AwCodes code, float scale, float (&r)[8])
{
#pragma unroll
    for (int k = 0; k < 8; k++) {
        const unsigned c = (code.w[k / 4] >> (8 * (k % 4))) & 255u;
        r[k] = c ? __uint_as_float((c + AW_LEVEL0) << 19) * scale : 0.0f;
    }
}
__device__ __forceinline__ AwCodes aw_pack_mean(const float (&m)[8], float& scale, const AwRandom* w = nullptr)
{
    unsigned most = 0;
#pragma unroll
    for (int k = 0; k < 8; k++) most = max(most, __float_as_uint(m[k]) & 0x7fffffffu);
    const float big = aw_max32(most);
    const bool held = big >= AW_SMALLEST;
    const float inv = held ? (1.0f / big) * 448.0f : 0.0f;
    scale = held ? big * (1.0f / 448.0f) : 0.0f;
    AwCodes c{ { 0, 0 } };
    if (w) {
        // (the conversion adds the top 20 bits of its random number in front of its cut.  The largest must not pass 448, above which the
        // next code is NaN: the factor's two roundings are within 2^-22)
        const float below = inv * (1.0f - 0x1p-22f);
#pragma unroll
        for (int h = 0; h < 2; h++) {
            int x = 0;
            x = __builtin_amdgcn_cvt_sr_fp8_f32(m[4 * h] * below, __builtin_rotateleft32(w->mean, 16 * h), x, 0);
            x = __builtin_amdgcn_cvt_sr_fp8_f32(m[4 * h + 1] * below, __builtin_rotateleft32(w->mean, 16 * h + 4), x, 1);
            x = __builtin_amdgcn_cvt_sr_fp8_f32(m[4 * h + 2] * below, __builtin_rotateleft32(w->mean, 16 * h + 8), x, 2);
            x = __builtin_amdgcn_cvt_sr_fp8_f32(m[4 * h + 3] * below, __builtin_rotateleft32(w->mean, 16 * h + 12), x, 3);
            c.w[h] = (unsigned)x;
        }
        return c;
    }
#pragma unroll
    for (int h = 0; h < 2; h++) {
        const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(m[4 * h] * inv, m[4 * h + 1] * inv, 0, false);
        c.w[h] = (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(m[4 * h + 2] * inv, m[4 * h + 3] * inv, lo, true);
    }
    return c;
}
__device__ __forceinline__ AwCodes aw_pack_root(const float (&r)[8], float& scale, const AwRandom* w = nullptr)
{
    unsigned most = 0;
#pragma unroll
    for (int k = 0; k < 8; k++) most = max(most, __float_as_uint(r[k]));
    const float big = aw_max32(most);
    const bool held = big >= AW_SMALLEST;
    const float inv = held ? 1.0f / big : 0.0f;
    scale = held ? big : 0.0f;
    AwCodes code{ { 0, 0 } };
#pragma unroll
    for (int k = 0; k < 8; k++) {
        // in units of the code: to the nearest, ties to even, or with 19 random bits in front of the cut; what is not zero is 1 at least
        // (also where big is infinite)
        const int bits = __float_as_int(r[k] * inv);
        const int up = w ? (int)(__builtin_rotateleft32(w->root, 4 * k) >> 13) : 0x3FFFF + ((bits >> 19) & 1);
        const int c = (bits + up - (int)((unsigned)AW_LEVEL0 << 19)) >> 19;
        code.w[k / 4] |= (unsigned)min(max(c, (int)min(__float_as_uint(r[k]), 1u)), 255) << (8 * (k % 4));
    }
    return code;
}

// ---- the step ----
//
// Bound by memory: 28 bytes an element in float32, 16 with moments in 8 bits, 10 with bfloat16 parameters and gradients too, at
// some 55 vector instructions an element, 60 with codes at random (39 T lane instructions a second: 1.5 ps, 10 bytes at 5 TB/s take 2;
// 250 M elements 468 us to the nearest, 469 at random).  The quotient is a
// product with the reciprocal (an ulp or two of the update).
template <int N>
__device__ __forceinline__ void aw_math(float (&p)[N], const float (&g)[N], float (&m)[N], float (&v)[N], float (&root)[N], const AwScal& s, float k,
                                        float keep)
{
#pragma unroll
    for (int q = 0; q < N; q++) {
        const float gk = g[q] * k;
        m[q] = m[q] * s.b1 + gk * s.omb1;
        v[q] = v[q] * s.b2 + gk * gk * s.omb2;
    }
    aw_sqrt(v, root);
#pragma unroll
    for (int q = 0; q < N; q++) p[q] = p[q] * keep - (m[q] * __builtin_amdgcn_rcpf(root[q] * s.c1 + s.eps)) * s.c2;
}

// eight elements of a tensor with 8-bit moments, from i on
template <int PE, int GE, bool FULL>
__device__ __forceinline__ void aw_update8(const AwTensor& T, const AwState& S, const void* g_base, long i, const AwScal& s, float k, float keep)
{
    float p[8], g[8], m[8], v[8], root[8];
    const long j = T.start + i;
    aw_load<PE, FULL>(T.p, i, T.n, p);
    aw_load<GE, FULL>(g_base, i, T.n, g);
    aw_mean_of(*(const AwCodes*)((const char*)S.m + j), S.ms[j / AW_BLOCK], m);
    aw_root_of(*(const AwCodes*)((const char*)S.v + j), S.vs[j / AW_BLOCK], v);
#pragma unroll
    for (int q = 0; q < 8; q++) v[q] = v[q] * v[q];
    aw_math(p, g, m, v, root, s, k, keep);
    aw_store<PE, FULL>(T.p, i, T.n, p);
    float ms, vs;
    AwCodes cm, cv;
    if (s.random) {
        const AwRandom w = aw_random(s.key, j);
        cm = aw_pack_mean(m, ms, &w);
        cv = aw_pack_root(root, vs, &w);
    } else {
        cm = aw_pack_mean(m, ms);
        cv = aw_pack_root(root, vs);
    }
    *(AwCodes*)((char*)S.m + j) = cm;
    *(AwCodes*)((char*)S.v + j) = cv;
    if (j % AW_BLOCK == 0) {
        S.ms[j / AW_BLOCK] = ms;
        S.vs[j / AW_BLOCK] = vs;
    }
}

// four elements of a tensor with 32-bit moments, from i and from i + 1024 on
template <int PE, int GE, bool FULL>
__device__ __forceinline__ void aw_update32(const AwTensor& T, const AwState& S, const void* g_base, long i, const AwScal& s, float k, float keep)
{
    float p[2][4], g[2][4], m[2][4], v[2][4], root[4];
    float *mt = (float*)S.m + T.start, *vt = (float*)S.v + T.start;
#pragma unroll
    for (int h = 0; h < 2; h++) {
        aw_load<PE, FULL>(T.p, i + 1024 * h, T.n, p[h]);
        aw_load<GE, FULL>(g_base, i + 1024 * h, T.n, g[h]);
        aw_load<0, FULL>(mt, i + 1024 * h, T.n, m[h]);
        aw_load<0, FULL>(vt, i + 1024 * h, T.n, v[h]);
    }
#pragma unroll
    for (int h = 0; h < 2; h++) {
        aw_math(p[h], g[h], m[h], v[h], root, s, k, keep);
        aw_store<PE, FULL>(T.p, i + 1024 * h, T.n, p[h]);
        aw_store<0, FULL>(mt, i + 1024 * h, T.n, m[h]);
        aw_store<0, FULL>(vt, i + 1024 * h, T.n, v[h]);
    }
}

template <int BITS, int PE, int GE, bool FULL>
__device__ __forceinline__ void aw_update(const AwTensor& T, const AwState& S, const void* g, long c0, const AwScal& s, float k, float keep)
{
    if constexpr (BITS == 8) {
        const long i = c0 + threadIdx.x * 8;
        if (FULL || i / AW_BLOCK * AW_BLOCK < T.n) aw_update8<PE, GE, FULL>(T, S, g, i, s, k, keep);
    } else aw_update32<PE, GE, FULL>(T, S, g, c0 + threadIdx.x * 4, s, k, keep);
}

template <int BITS, int PE, int GE>
__device__ __forceinline__ void aw_update(const AwTensor& T, const AwState& S, const void* g, int chunk, const AwScal& s, float k, float keep)
{
    const long c0 = (long)chunk * AW_CHUNK;
    if (c0 + AW_CHUNK <= T.n) aw_update<BITS, PE, GE, true>(T, S, g, c0, s, k, keep);
    else aw_update<BITS, PE, GE, false>(T, S, g, c0, s, k, keep);
}

template <int BITS>
__global__ __launch_bounds__(256) void k_adamw(const AwTensor* __restrict__ tensors, const AwChunk* __restrict__ chunks, int base, AwState S,
                                               AwGrads grads, AwScal s, const double* __restrict__ scal, const float* __restrict__ clip,
                                               const AwClock* __restrict__ clock)
{
    // behind the norm, backwards: its last gradients are still in the memory-side cache (97 M elements: 599 -> 594 us)
    const AwChunk ch = chunks[clip ? gridDim.x - 1 - blockIdx.x : blockIdx.x];
    const AwTensor T = tensors[ch.tensor];
    const void* g = grads.g[ch.tensor - base];
    if (!g) return;
    const float k = clip ? clip[1] : 1.0f;
    if (k != k) return;                                    // the gradients' norm is not finite: the step is skipped
    if (scal) {
        s.lr = scal[0];
        s.c1 = (float)scal[1];
        s.c2 = (float)scal[2];
    } else if (clock) {
        s.c1 = (float)clock->c1;
        s.c2 = (float)clock->c2;
    }
    if (BITS == 8 && clock) {
        s.key = clock->key;
        s.random = clock->random != 0;
    }
    const float keep = (float)(1.0 - s.lr * (double)T.decay);
    switch (T.ptype * 3 + T.gtype) {
        case 0: aw_update<BITS, 0, 0>(T, S, g, ch.chunk, s, k, keep); break;
        case 1: aw_update<BITS, 0, 1>(T, S, g, ch.chunk, s, k, keep); break;
        case 2: aw_update<BITS, 0, 2>(T, S, g, ch.chunk, s, k, keep); break;
        case 3: aw_update<BITS, 1, 0>(T, S, g, ch.chunk, s, k, keep); break;
        case 4: aw_update<BITS, 1, 1>(T, S, g, ch.chunk, s, k, keep); break;
        case 5: aw_update<BITS, 1, 2>(T, S, g, ch.chunk, s, k, keep); break;
        case 6: aw_update<BITS, 2, 0>(T, S, g, ch.chunk, s, k, keep); break;
        case 7: aw_update<BITS, 2, 1>(T, S, g, ch.chunk, s, k, keep); break;
        default: aw_update<BITS, 2, 2>(T, S, g, ch.chunk, s, k, keep); break;
    }
}

// ---- the clock ----
__device__ __forceinline__ double aw_c1(double b2, long t) { return 1.0 / sqrt(1.0 - pow(b2, (double)t)); }
__device__ __forceinline__ double aw_c2(double lr, double b1, long t) { return lr / (1.0 - pow(b1, (double)t)); }
__device__ __forceinline__ long aw_number(long t, const AwClock* clock) { return max(1L, t - clock->skipped); }

__device__ __forceinline__ void aw_tick(const AwTick& k, bool skip)
{
    if (skip) {
        k.clock->skipped++;
        return;
    }
    const long age = k.age + k.clock->ticks++;
    k.clock->key = aw_key(age);
    k.clock->random = age >= AW_NEAREST;
}
// before a step that the clock counts and whose norm, if it has one, was computed before
__global__ __launch_bounds__(64) void k_adamw_tick(AwTick k, const float* __restrict__ clip)
{
    const long t = aw_number(k.t, k.clock);
    if (threadIdx.x == 0) {
        k.clock->c1 = aw_c1(k.b2, t);
        k.clock->c2 = aw_c2(k.lr, k.b1, t);
        aw_tick(k, clip && clip[1] != clip[1]);
    }
}
// the moments were set
__global__ void k_adamw_restart(AwClock* clock, long age)
{
    if (threadIdx.x == 0) {
        clock->ticks = -age;
        clock->skipped = 0;
    }
}
// what a captured step of number t reads
__global__ void k_adamw_scalars(AwTick k, double* __restrict__ out)
{
    if (threadIdx.x) return;
    const long t = aw_number(k.t, k.clock);
    out[0] = k.lr;
    out[1] = aw_c1(k.b2, t);
    out[2] = aw_c2(k.lr, k.b1, t);
}

// ---- the norm: float64 partial sums per workgroup, then one workgroup adds them in order (a launch of its own, 3 us: the last
// workgroup of the first launch doing it costs every workgroup a release of its XCD's L2: 44 us for 1 M elements) ----
__device__ __forceinline__ double aw_block_sum(double x, double* lds)
{
    for (int d = 1; d < 64; d <<= 1) x += __shfl_xor(x, d);
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = x;
    __syncthreads();
    x = (lds[0] + lds[1]) + (lds[2] + lds[3]);
    __syncthreads();
    return x;
}

template <int E, bool FULL> __device__ __forceinline__ double aw_square_sum(const void* g, long i, long n)
{
    float x[8];
    aw_load<E, FULL>(g, i, n, x);
    double a = 0.0, b = 0.0;
#pragma unroll
    for (int q = 0; q < 8; q += 2) {
        a = fma((double)x[q], (double)x[q], a);
        b = fma((double)x[q + 1], (double)x[q + 1], b);
    }
    return a + b;
}
template <bool FULL> __device__ __forceinline__ double aw_square_sum(int gtype, const void* g, long i, long n)
{
    return gtype == 0 ? aw_square_sum<0, FULL>(g, i, n) : gtype == 1 ? aw_square_sum<1, FULL>(g, i, n) : aw_square_sum<2, FULL>(g, i, n);
}

// add: a launch after the first of several
__global__ __launch_bounds__(256) void k_adamw_sumsq(const AwTensor* __restrict__ tensors, const AwChunk* __restrict__ chunks, int n_chunks, int base,
                                                     AwGrads grads, double* __restrict__ partials, int add)
{
    __shared__ double lds[4];
    double sum = 0.0;
    for (int b = blockIdx.x; b < n_chunks; b += gridDim.x) {
        const AwChunk ch = chunks[b];
        const AwTensor& T = tensors[ch.tensor];
        const void* g = grads.g[ch.tensor - base];
        const long c0 = (long)ch.chunk * AW_CHUNK, i = c0 + threadIdx.x * 8, n = g ? T.n : 0;
        sum += c0 + AW_CHUNK <= n ? aw_square_sum<true>(T.gtype, g, i, n) : aw_square_sum<false>(T.gtype, g, i, n);
    }
    sum = aw_block_sum(sum, lds);
    if (threadIdx.x == 0) partials[blockIdx.x] = add ? partials[blockIdx.x] + sum : sum;
}

// out[0] = norm, out[1] = the coefficient min(1, max_norm / norm); NaN where the norm is not finite.  With a clock it is a step's: the bias
// corrections are another wavefront's while the partial sums are on their way.
__global__ __launch_bounds__(256) void k_adamw_norm(const double* __restrict__ partials, int n, double max_norm, float* __restrict__ out, AwTick k)
{
    __shared__ double lds[4];
    double sum = 0.0;
    if (k.clock && threadIdx.x == 64) k.clock->c1 = aw_c1(k.b2, aw_number(k.t, k.clock));
    if (k.clock && threadIdx.x == 128) k.clock->c2 = aw_c2(k.lr, k.b1, aw_number(k.t, k.clock));
    for (int i = threadIdx.x; i < n; i += 256) sum += partials[i];
    sum = aw_block_sum(sum, lds);
    if (threadIdx.x == 0) {
        const double norm = sqrt(sum);
        out[0] = (float)norm;
        out[1] = !(norm < (double)INFINITY) ? NAN : norm > max_norm ? (float)(max_norm / norm) : 1.0f;
        if (k.clock) aw_tick(k, !(norm < (double)INFINITY));       // (behind the barriers: the others have read the clock)
    }
}

// ---- one of the moments (ROOT: the second) from float32 tensors, 8-bit ones to a float32 array of the flat layout ----
template <int BITS, bool ROOT>
__global__ __launch_bounds__(256) void k_adamw_load(const AwTensor* __restrict__ tensors, const AwChunk* __restrict__ chunks, int base, AwState S,
                                                    AwGrads from)
{
    const AwChunk ch = chunks[blockIdx.x];
    const AwTensor T = tensors[ch.tensor];
    const long i = (long)ch.chunk * AW_CHUNK + threadIdx.x * 8, j = T.start + i;
    if (i / AW_BLOCK * AW_BLOCK >= T.n) return;
    float x[8];
    aw_load<0>(from.g[ch.tensor - base], i, T.n, x);
    if constexpr (BITS == 32) aw_store<0>((float*)(ROOT ? S.v : S.m) + T.start, i, T.n, x);
    else {
        float scale;
        if constexpr (ROOT) {
            float r[8];
            aw_sqrt(x, r);
            *(AwCodes*)((char*)S.v + j) = aw_pack_root(r, scale);
        } else *(AwCodes*)((char*)S.m + j) = aw_pack_mean(x, scale);
        if (j % AW_BLOCK == 0) (ROOT ? S.vs : S.ms)[j / AW_BLOCK] = scale;
    }
}

// (the codes between a tensor's end and the next one's start are 0)
__global__ __launch_bounds__(256) void k_adamw_unpack(AwState S, float* __restrict__ m_out, float* __restrict__ v_out, long quads)
{
    for (long q = (long)blockIdx.x * 256 + threadIdx.x; q < quads; q += (long)gridDim.x * 256) {
        const float ms = S.ms[q / (AW_BLOCK / 4)], vs = S.vs[q / (AW_BLOCK / 4)];
        float m[8], r[8];
        aw_mean_of(AwCodes{ { ((const unsigned*)S.m)[q], 0 } }, ms, m);
        aw_root_of(AwCodes{ { ((const unsigned*)S.v)[q], 0 } }, vs, r);
        ((float4*)m_out)[q] = make_float4(m[0], m[1], m[2], m[3]);
        ((float4*)v_out)[q] = make_float4(r[0] * r[0], r[1] * r[1], r[2] * r[2], r[3] * r[3]);
    }
}

// ---- host ----
static long aw_padded(int64_t n) { return (long)((n + AW_BLOCK - 1) / AW_BLOCK) * AW_BLOCK; }

int64_t adamw_state_elems(int n, const int64_t* numels)
{
    int64_t total = 0;
    for (int i = 0; i < n; i++) total += aw_padded(numels[i]);
    return total;
}

static void aw_free(goai_adamw* o)
{
    if (!o) return;
    (void)hipFree(o->d_mem);
    delete o;
}

int adamw_check(int n, void* const* params, const int32_t* ptypes, const int32_t* gtypes, const int64_t* numels, const float* decays, int bits,
                const void* m, const void* v, const float* ms, const float* vs)
{
    GOAI_REQUIRE(n >= 1, "adamw: no tensors");
    GOAI_REQUIRE(params && ptypes && gtypes && numels && decays, "adamw: NULL table");
    GOAI_REQUIRE(bits == 8 || bits == 32, "adamw: state_bits must be 8 or 32");
    GOAI_REQUIRE(m && v && (bits == 32 || (ms && vs)), "adamw: NULL moments");
    GOAI_REQUIRE((((uintptr_t)m | (uintptr_t)v) & 15) == 0 && (((uintptr_t)ms | (uintptr_t)vs) & 3) == 0, "adamw: moments must be 16-byte aligned");
    int64_t chunks = 0;
    std::vector<std::pair<uintptr_t, uintptr_t>> spans;
    for (int i = 0; i < n; i++) {
        GOAI_REQUIRE(elem_ok(ptypes[i]) && elem_ok(gtypes[i]), "adamw: element type must be GOAI_ELEM_F32, GOAI_ELEM_BF16 or GOAI_ELEM_F16");
        GOAI_REQUIRE(numels[i] >= 0 && numels[i] < (1LL << 40), "adamw: tensor size out of range");
        GOAI_REQUIRE(isfinite(decays[i]) && decays[i] >= 0.0f, "adamw: weight decay must be finite and not negative");
        chunks += (numels[i] + AW_CHUNK - 1) / AW_CHUNK;
        if (!numels[i]) continue;
        const uintptr_t at = (uintptr_t)params[i];
        GOAI_REQUIRE(at != 0, "adamw: NULL parameter");
        GOAI_REQUIRE(at % elem_bytes(ptypes[i]) == 0, "adamw: a parameter is not aligned to its element type");
        spans.emplace_back(at, at + (uintptr_t)numels[i] * elem_bytes(ptypes[i]));
    }
    GOAI_REQUIRE(chunks < (1LL << 23), "adamw: too many elements");
    std::sort(spans.begin(), spans.end());
    for (size_t i = 1; i < spans.size(); i++) GOAI_REQUIRE(spans[i].first >= spans[i - 1].second, "adamw: parameters overlap in memory");
    return GOAI_OK;
}

static int aw_build(goai_adamw* o, int n, void* const* params, const int32_t* ptypes, const int32_t* gtypes, const int64_t* numels,
                    const float* decays)
{
    std::vector<AwChunk> chunks;
    for (int i = 0; i < n; i++) {
        o->tensors.push_back(AwTensor{ params[i], o->elems, (long)numels[i], decays[i], ptypes[i], gtypes[i] });
        o->first.push_back((int)chunks.size());
        for (int64_t k = 0; k * AW_CHUNK < numels[i]; k++) chunks.push_back(AwChunk{ i, (int)k });
        o->elems += aw_padded(numels[i]);
    }
    o->first.push_back((int)chunks.size());
    const size_t nb = AW_NORM_BLOCKS * sizeof(double), pb = nb + sizeof(AwClock), tb = o->tensors.size() * sizeof(AwTensor),
                 cb = chunks.size() * sizeof(AwChunk);
    std::vector<char> image(pb + tb + cb);                                     // (zeros at first: the clock's)
    memcpy(image.data() + pb, o->tensors.data(), tb);
    if (cb) memcpy(image.data() + pb + tb, chunks.data(), cb);
    GOAI_HIP_CHECK(hipMalloc((void**)&o->d_mem, image.size()));
    GOAI_HIP_CHECK(hipMemcpy(o->d_mem, image.data(), image.size(), hipMemcpyHostToDevice));
    o->d_partials = (double*)o->d_mem;
    o->d_clock = (AwClock*)(o->d_mem + nb);
    o->d_tensors = (AwTensor*)(o->d_mem + pb);
    o->d_chunks = (AwChunk*)(o->d_mem + pb + tb);
    return GOAI_OK;
}

int adamw_init(goai_ctx* c, int n, void* const* params, const int32_t* ptypes, const int32_t* gtypes, const int64_t* numels, const float* decays,
               int bits, void* m, void* v, float* ms, float* vs, goai_adamw** out)
{
    goai_adamw* o = new goai_adamw();
    o->device = c->device;
    o->bits = bits;
    o->state = AwState{ m, v, ms, vs };
    int rc;
    try {
        rc = aw_build(o, n, params, ptypes, gtypes, numels, decays);
    } catch (...) {
        aw_free(o);
        throw;
    }
    if (rc) {
        aw_free(o);
        return rc;
    }
    *out = o;
    return GOAI_OK;
}

int adamw_destroy(goai_ctx* c, goai_adamw* o)
{
    GOAI_REQUIRE(!c || o->device == c->device, "adamw: the optimiser lives on another GPU");
    OnDevice on_device;
    GOAI_HIP_CHECK(on_device.enter(o->device));
    if (c) GOAI_HIP_CHECK(hipStreamSynchronize(c->stream));
    else GOAI_HIP_CHECK(hipDeviceSynchronize());
    aw_free(o);
    return GOAI_OK;
}

// the launches of one pass over the tensors: AW_LAUNCH tensors at a time
template <class F> static int aw_launches(const goai_adamw* o, const void* const* grads, F&& launch)
{
    const int n = (int)o->tensors.size();
    for (int base = 0; base < n; base += AW_LAUNCH) {
        const int end = std::min(n, base + AW_LAUNCH);
        AwGrads g;
        memset(&g, 0, sizeof(g));
        for (int i = base; i < end; i++) g.g[i - base] = grads[i];
        launch(base, o->d_chunks + o->first[base], o->first[end] - o->first[base], g);
        GOAI_HIP_CHECK(hipGetLastError());
    }
    return GOAI_OK;
}

static int aw_check_grads(goai_ctx* c, const goai_adamw* o, const void* const* grads)
{
    GOAI_REQUIRE(o->device == c->device, "adamw: the optimiser lives on another GPU");
    for (size_t i = 0; i < o->tensors.size(); i++)
        GOAI_REQUIRE((uintptr_t)grads[i] % elem_bytes(o->tensors[i].gtype) == 0, "adamw: a gradient is not aligned to its element type");
    return GOAI_OK;
}

static int aw_norm(goai_ctx* c, goai_adamw* o, const void* const* grads, double max_norm, float* out, const AwTick& tick)
{
    const int grid = std::max(1, std::min(AW_NORM_BLOCKS, o->first.back()));
    const int rc = aw_launches(o, grads, [&](int base, const AwChunk* chunks, int n, const AwGrads& g) {
        k_adamw_sumsq<<<grid, 256, 0, c->stream>>>(o->d_tensors, chunks, n, base, g, o->d_partials, base != 0);
    });
    if (rc) return rc;
    k_adamw_norm<<<1, 256, 0, c->stream>>>(o->d_partials, grid, max_norm, out, tick);
    GOAI_HIP_CHECK(hipGetLastError());
    return GOAI_OK;
}

int adamw_grad_norm(goai_ctx* c, goai_adamw* o, const void* const* grads, double max_norm, float* out)
{
    const int rc = aw_check_grads(c, o, grads);
    return rc ? rc : aw_norm(c, o, grads, max_norm, out, AwTick{});
}

int adamw_step(goai_ctx* c, goai_adamw* o, const void* const* grads, int64_t t, double lr, double beta1, double beta2, double eps,
               double max_norm, float* clip, const double* scalars)
{
    int rc = aw_check_grads(c, o, grads);
    if (rc) return rc;
    if (!scalars) {
        hipStreamCaptureStatus cap = hipStreamCaptureStatusNone;
        GOAI_HIP_CHECK(hipStreamIsCapturing(c->stream, &cap));
        if (cap != hipStreamCaptureStatusNone) {
            set_error("adamw: a captured step needs `scalars` on the device (lr and the bias corrections change from replay to replay)");
            return GOAI_ERR_STATE;
        }
    }
    AwScal s{ lr, (float)beta1, (float)(1.0 - beta1), (float)beta2, (float)(1.0 - beta2), (float)eps,
              (float)(1.0 / sqrt(1.0 - pow(beta2, (double)t))), (float)(lr / (1.0 - pow(beta1, (double)t))), aw_key(o->age), o->age >= AW_NEAREST };
    // the clock counts steps that may be captured and steps that may be skipped, and once it has, all (scalars hold the corrections
    // themselves: a captured step without 8-bit moments needs no clock)
    if (scalars || clip) o->ticking = true;
    const AwClock* clock = clip || (o->ticking && (o->bits == 8 || !scalars)) ? o->d_clock : nullptr;
    const AwTick tick{ o->d_clock, o->age, (long)t, lr, beta1, beta2 };
    if (max_norm > 0.0) {
        if ((rc = aw_norm(c, o, grads, max_norm, clip, tick))) return rc;
    } else if (clock) {
        k_adamw_tick<<<1, 64, 0, c->stream>>>(tick, clip);
        GOAI_HIP_CHECK(hipGetLastError());
    }
    rc = aw_launches(o, grads, [&](int base, const AwChunk* chunks, int n, const AwGrads& g) {
        if (n == 0) return;
        if (o->bits == 32) k_adamw<32><<<n, 256, 0, c->stream>>>(o->d_tensors, chunks, base, o->state, g, s, scalars, clip, clock);
        else k_adamw<8><<<n, 256, 0, c->stream>>>(o->d_tensors, chunks, base, o->state, g, s, scalars, clip, clock);
    });
    if (rc == GOAI_OK && !o->ticking) o->age++;
    return rc;
}

// scalars of step t for a captured step, less the steps skipped so far
int adamw_scalars(goai_ctx* c, goai_adamw* o, int64_t t, double lr, double beta1, double beta2, double* scalars)
{
    GOAI_REQUIRE(o->device == c->device, "adamw: the optimiser lives on another GPU");
    k_adamw_scalars<<<1, 64, 0, c->stream>>>(AwTick{ o->d_clock, 0, (long)t, lr, beta1, beta2 }, scalars);
    GOAI_HIP_CHECK(hipGetLastError());
    return GOAI_OK;
}

int adamw_skipped(goai_ctx* c, goai_adamw* o, int64_t* skipped)
{
    GOAI_REQUIRE(!c || o->device == c->device, "adamw: the optimiser lives on another GPU");
    OnDevice on_device;
    GOAI_HIP_CHECK(on_device.enter(o->device));
    *skipped = 0;
    if (!o->ticking) return GOAI_OK;
    long n = 0;
    if (c) GOAI_HIP_CHECK(hipStreamSynchronize(c->stream));
    else GOAI_HIP_CHECK(hipDeviceSynchronize());
    GOAI_HIP_CHECK(hipMemcpy(&n, &o->d_clock->skipped, sizeof(n), hipMemcpyDeviceToHost));
    *skipped = n;
    return GOAI_OK;
}

int adamw_load_moments(goai_ctx* c, goai_adamw* o, const float* const* m, const float* const* v)
{
    GOAI_REQUIRE(o->device == c->device, "adamw: the optimiser lives on another GPU");
    for (size_t i = 0; i < o->tensors.size(); i++) {
        GOAI_REQUIRE(o->tensors[i].n == 0 || (m[i] && v[i]), "adamw: NULL moment");
        GOAI_REQUIRE((((uintptr_t)m[i] | (uintptr_t)v[i]) & 3) == 0, "adamw: a moment is not aligned to its element type");
    }
    const auto load = [&](const float* const* from, auto kernel) {
        return aw_launches(o, (const void* const*)from, [&](int base, const AwChunk* chunks, int n, const AwGrads& g) {
            if (n) kernel<<<n, 256, 0, c->stream>>>(o->d_tensors, chunks, base, o->state, g);
        });
    };
    if (o->ticking) {
        k_adamw_restart<<<1, 64, 0, c->stream>>>(o->d_clock, o->age);
        GOAI_HIP_CHECK(hipGetLastError());
    } else o->age = 0;
    const int rc = o->bits == 8 ? load(m, k_adamw_load<8, false>) : load(m, k_adamw_load<32, false>);
    if (rc) return rc;
    return o->bits == 8 ? load(v, k_adamw_load<8, true>) : load(v, k_adamw_load<32, true>);
}

int adamw_moments(goai_ctx* c, goai_adamw* o, float* m, float* v)
{
    GOAI_REQUIRE(o->device == c->device, "adamw: the optimiser lives on another GPU");
    GOAI_REQUIRE((((uintptr_t)m | (uintptr_t)v) & 15) == 0, "adamw: moments must be 16-byte aligned");
    if (o->bits == 32) {
        GOAI_HIP_CHECK(hipMemcpyAsync(m, o->state.m, o->elems * sizeof(float), hipMemcpyDeviceToDevice, c->stream));
        GOAI_HIP_CHECK(hipMemcpyAsync(v, o->state.v, o->elems * sizeof(float), hipMemcpyDeviceToDevice, c->stream));
        return GOAI_OK;
    }
    const long quads = o->elems / 4;
    if (quads) k_adamw_unpack<<<(unsigned)std::min<long>((quads + 255) / 256, 1 << 20), 256, 0, c->stream>>>(o->state, m, v, quads);
    GOAI_HIP_CHECK(hipGetLastError());
    return GOAI_OK;
}

}  // namespace goai
