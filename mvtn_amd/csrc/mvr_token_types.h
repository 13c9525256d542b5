// mvr_token_types.h — what the kernels on view tokens (mvr_tokens.hip, mvr_attend.hip) share: element types, vectors of eight
// elements, sums over a wave, error reporting.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>
#include <stdio.h>

#include "../../include/mvr.h"

extern "C" __attribute__((visibility("hidden"))) void mvr_set_error_(const char *msg);

namespace mvr_tok {

typedef __bf16 bf16;
typedef _Float16 f16;

inline int fail(int code, const char *msg) {
  mvr_set_error_(msg);
  return code;
}
inline int bad(const char *msg) { return fail(MVR_ERR_INVALID_ARG, msg); }
inline int launched(const char *what) {
  const hipError_t e = hipGetLastError();
  if (e == hipSuccess) return MVR_OK;
  char buf[200];
  snprintf(buf, sizeof buf, "%s: %s", what, hipGetErrorString(e));
  return fail(MVR_ERR_HIP, buf);
}

// N consecutive elements on their way.  Whole vectors go through memcpy: 8- and 16-byte accesses whatever the alignment (rows of odd
// width start anywhere; the hardware takes unaligned vector accesses), the last vector of such a row element by element.
template <typename T, int N>
struct Raw {
  static constexpr int kWords = N * (int)sizeof(T) / 4;   // kept as words: 16-bit elements on their way take half a register each
  unsigned w[kWords];
  __device__ __forceinline__ void load(const T *p, int left) {
    if (left >= N) {
      __builtin_memcpy(w, p, sizeof w);
    } else {
#pragma unroll
      for (int k = 0; k < kWords; ++k) w[k] = 0;
      const unsigned short *h = reinterpret_cast<const unsigned short *>(p);
      if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int k = 0; k < N; ++k)
          if (k < left) __builtin_memcpy(&w[k], p + k, 4);
      } else {
#pragma unroll
        for (int k = 0; k < N; ++k)
          if (k < left) w[k / 2] |= (unsigned)h[k] << (16 * (k & 1));
      }
    }
  }
  __device__ __forceinline__ void get(float (&v)[N]) const {
#pragma unroll
    for (int k = 0; k < N; ++k) {
      if constexpr (sizeof(T) == 4) {
        v[k] = __builtin_bit_cast(float, w[k]);
      } else {
        const unsigned short h = (unsigned short)(w[k / 2] >> (16 * (k & 1)));
        v[k] = (float)__builtin_bit_cast(T, h);
      }
    }
  }
};
template <int N, typename T>
__device__ __forceinline__ void load_n(const T *p, int left, float (&v)[N]) {
  Raw<T, N> r;
  r.load(p, left);
  r.get(v);
}
template <int N, typename T>
__device__ __forceinline__ void store_n(T *p, int left, const float (&v)[N]) {
  if (left >= N) {
    T t[N];
#pragma unroll
    for (int k = 0; k < N; ++k) t[k] = (T)v[k];
    __builtin_memcpy(p, t, sizeof t);
  } else {
#pragma unroll
    for (int k = 0; k < N; ++k)
      if (k < left) p[k] = (T)v[k];
  }
}

// a barrier that waits for LDS only: global loads in flight stay in flight
__device__ __forceinline__ void lds_barrier() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

template <int CTRL>
__device__ __forceinline__ float dpp(float x) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, 0xF, 0xF, true));
}
// the two halves of a wave (or of each half) exchanged: x of this lane, x of the lane 32 (16) away
__device__ __forceinline__ float other_half(float x) {
  const unsigned u = __builtin_bit_cast(unsigned, x);
  auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  const unsigned other = (threadIdx.x & 32) ? r[0] : r[1];
  return __builtin_bit_cast(float, other);
}
__device__ __forceinline__ float wave_sum(float x) {   // in every lane; the order of the additions is fixed
  x += dpp<0xB1>(x);    // lanes 1 0 3 2
  x += dpp<0x4E>(x);    // lanes 2 3 0 1
  x += dpp<0x124>(x);   // rotated by 4 in a row of 16
  x += dpp<0x128>(x);   // by 8
  // (elements of the swaps' results go through variables: a bit cast straight from a vector element takes element 0)
  unsigned u = __builtin_bit_cast(unsigned, x);
  auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  unsigned r0 = r[0], r1 = r[1];
  u = __builtin_bit_cast(unsigned, __builtin_bit_cast(float, r0) + __builtin_bit_cast(float, r1));
  auto q = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  r0 = q[0], r1 = q[1];
  return __builtin_bit_cast(float, r0) + __builtin_bit_cast(float, r1);
}

}  // namespace mvr_tok
