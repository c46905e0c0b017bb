// elem.h -- the element types of caller-owned arrays that may be float32, bfloat16 or float16 (GOAI_ELEM_*), and their
// conversions; all arithmetic on them is float32.
#pragma once
#include <hip/hip_bfloat16.h>
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace goai {

template <int E> struct Elem;                                   // E = GOAI_ELEM_*
template <> struct Elem<0> { using raw = float; };
template <> struct Elem<1> { using raw = uint16_t; };           // bfloat16 bits
template <> struct Elem<2> { using raw = uint16_t; };           // float16 bits

template <int E> __device__ __forceinline__ float elem_to_float(typename Elem<E>::raw x)
{
    if constexpr (E == 0) return x;
    else if constexpr (E == 1) return __uint_as_float((unsigned)x << 16);
    else return (float)__builtin_bit_cast(_Float16, x);
}

// round to nearest even
template <int E> __device__ __forceinline__ typename Elem<E>::raw elem_from_float(float x)
{
    if constexpr (E == 0) return x;
    else if constexpr (E == 1) return __builtin_bit_cast(uint16_t, (__bf16)x);
    else return __builtin_bit_cast(uint16_t, (_Float16)x);
}

// N neighbouring elements by wide accesses; the address is aligned to the element type only (gfx950 takes that in global memory)
template <int E, int N> struct ElemVec {
    using raw = typename Elem<E>::raw;
    raw a[N];
};
template <int E, int N> __device__ __forceinline__ void elem_load(const typename Elem<E>::raw* p, float (&out)[N])
{
    ElemVec<E, N> v;
    __builtin_memcpy(&v, p, sizeof(v));
#pragma unroll
    for (int k = 0; k < N; k++) out[k] = elem_to_float<E>(v.a[k]);
}
template <int E, int N> __device__ __forceinline__ void elem_store(typename Elem<E>::raw* p, const float (&x)[N])
{
    ElemVec<E, N> v;
#pragma unroll
    for (int k = 0; k < N; k++) v.a[k] = elem_from_float<E>(x[k]);
    __builtin_memcpy(p, &v, sizeof(v));
}

inline int elem_bytes(int e) { return e == 0 ? 4 : 2; }
inline bool elem_ok(int e) { return e >= 0 && e <= 2; }

}  // namespace goai
