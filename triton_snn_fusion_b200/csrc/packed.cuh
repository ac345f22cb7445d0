// fp32 arithmetic on the few values of a thread, two at a time on the packed pipe.
#pragma once

#include "common.cuh"

#include <type_traits>

namespace snnb {
namespace {

// Each half of a packed instruction rounds like the scalar one.
__device__ __forceinline__ uint64_t pair(float x, float y) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ void unpair(uint64_t r, float &x, float &y) { asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(r)); }
// r = a * b + c
template <int N>
__device__ __forceinline__ void v_fma(const float (&a)[N], const float (&b)[N], const float (&c)[N], float (&r)[N]) {
  if constexpr (N == 1) {
    r[0] = fmaf(a[0], b[0], c[0]);
  } else {
#pragma unroll
    for (int k = 0; k < N; k += 2) {
      uint64_t o;
      asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(o) : "l"(pair(a[k], a[k + 1])), "l"(pair(b[k], b[k + 1])), "l"(pair(c[k], c[k + 1])));
      unpair(o, r[k], r[k + 1]);
    }
  }
}
template <int N> __device__ __forceinline__ void v_mul(const float (&a)[N], const float (&b)[N], float (&r)[N]) {
  if constexpr (N == 1) {
    r[0] = a[0] * b[0];
  } else {
#pragma unroll
    for (int k = 0; k < N; k += 2) {
      uint64_t o;
      asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(o) : "l"(pair(a[k], a[k + 1])), "l"(pair(b[k], b[k + 1])));
      unpair(o, r[k], r[k + 1]);
    }
  }
}
template <int N> __device__ __forceinline__ void v_add(const float (&a)[N], const float (&b)[N], float (&r)[N]) {
  if constexpr (N == 1) {
    r[0] = a[0] + b[0];
  } else {
#pragma unroll
    for (int k = 0; k < N; k += 2) {
      uint64_t o;
      asm("add.rn.f32x2 %0, %1, %2;" : "=l"(o) : "l"(pair(a[k], a[k + 1])), "l"(pair(b[k], b[k + 1])));
      unpair(o, r[k], r[k + 1]);
    }
  }
}
template <int N> __device__ __forceinline__ void v_set(float (&r)[N], float v) {
#pragma unroll
  for (int k = 0; k < N; ++k) r[k] = v;
}

// p: the start of a Pack<T, N> (its alignment is what allows whole words). A bf16 is the upper half of an fp32: one
// instruction a value from the word that holds two. WORDS false: the values were loaded one by one, and a word would have
// to be put together first, which waits for the loads.
template <typename T, int N, bool WORDS = true> __device__ __forceinline__ void widen(const T *p, float (&v)[N]) {
  if constexpr (WORDS && sizeof(T) == 2 && N % 2 == 0) {
#pragma unroll
    for (int k = 0; k < N; k += 2) {
      const uint32_t w = *reinterpret_cast<const uint32_t *>(p + k);
      if constexpr (std::is_same_v<T, __nv_bfloat16>) {
        v[k] = __uint_as_float(w << 16);
        v[k + 1] = __uint_as_float(w & 0xffff0000u);
      } else {
        const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w));
        v[k] = f.x;
        v[k + 1] = f.y;
      }
    }
  } else {
#pragma unroll
    for (int k = 0; k < N; ++k) v[k] = DT<T>::to_f(p[k]);
  }
}

template <int N> __device__ __forceinline__ void sh_load(const float *p, float (&v)[N]) {
  const Pack<float, N> r = *reinterpret_cast<const Pack<float, N> *>(p);
#pragma unroll
  for (int k = 0; k < N; ++k) v[k] = r.v[k];
}
template <int N> __device__ __forceinline__ void sh_store(float *p, const float (&v)[N]) {
  Pack<float, N> r;
#pragma unroll
  for (int k = 0; k < N; ++k) r.v[k] = v[k];
  *reinterpret_cast<Pack<float, N> *>(p) = r;
}

// Asynchronous copy of 16 bytes into shared memory, past the L1 cache: through it a copy on its way would take a whole line.
__device__ __forceinline__ void copy_async16(void *dst, const void *src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// a = 1 / (1 + e) and b = 1 - a = e a with e = exp(-g): both keep their relative accuracy, neither is the difference of the
// other from one. Below g = -87 e leaves the range in which its reciprocal is a normal number: a is zero then, and b, which
// would be zero or not a number, comes from the second term of its maximum (1 where a is zero, smaller than e a elsewhere).
// A gate that is not a number makes a one.
template <int N> __device__ __forceinline__ void v_sigmoid(const float (&g)[N], float (&a)[N], float (&b)[N]) {
  float one[N], t[N], k2[N];
  v_set(one, 1.f);
  v_set(k2, -1.4426950408889634f);
  v_mul(g, k2, t);
#pragma unroll
  for (int k = 0; k < N; ++k) asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(t[k]) : "f"(t[k]));
  v_add(t, one, a);
#pragma unroll
  for (int k = 0; k < N; ++k) asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(a[k]) : "f"(a[k]));
  v_mul(t, a, b);
  v_set(k2, -1073741824.f);
  v_fma(a, k2, one, t);
#pragma unroll
  for (int k = 0; k < N; ++k) b[k] = fmaxf(b[k], t[k]);
}

}  // namespace
}  // namespace snnb
