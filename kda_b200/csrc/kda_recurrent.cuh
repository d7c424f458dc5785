// Shared by the token-recurrent kernels with a decay per key column (kda_recurrent.cu) and per head (delta_recurrent.cu).
#pragma once

#include "kda_common.cuh"
#include "kda_device.cuh"

namespace kda {

template <typename IO> struct IoTraits;
template <> struct IoTraits<float> {
  static __device__ __forceinline__ float ld(const float* p) { return *p; }
  static __device__ __forceinline__ void st4(float* p, float4 x) { *reinterpret_cast<float4*>(p) = x; }
  static __device__ __forceinline__ float4 ld4(const float* p) { return *reinterpret_cast<const float4*>(p); }
};
template <> struct IoTraits<__nv_bfloat16> {
  static __device__ __forceinline__ float ld(const __nv_bfloat16* p) { return __bfloat162float(*p); }
  static __device__ __forceinline__ void st4(__nv_bfloat16* p, float4 x) {
    uint2 u = make_uint2(pack_bf16(x.x, x.y), pack_bf16(x.z, x.w));
    *reinterpret_cast<uint2*>(p) = u;
  }
  static __device__ __forceinline__ float4 ld4(const __nv_bfloat16* p) {
    uint2 u = *reinterpret_cast<const uint2*>(p);
    float2 a = unpack_bf16(u.x), b = unpack_bf16(u.y);
    return make_float4(a.x, a.y, b.x, b.y);
  }
};

constexpr int REC_WARPS = 4;

// Sum over the 32 lanes of 32 per-lane values at once: lane L returns the total of v[L] (31 shuffles).
__device__ __forceinline__ float butterfly_sum32(float (&v)[32], int lane) {
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) {
    const bool up = (lane & o) != 0;
#pragma unroll
    for (int i = 0; i < o; ++i) {
      const float mine = up ? v[i + o] : v[i];
      const float other = up ? v[i] : v[i + o];
      v[i] = mine + __shfl_xor_sync(0xffffffffu, other, o);
    }
  }
  return v[0];
}

// E consecutive elements of a row as untouched bits: a conversion right behind the load would make the warp wait for it there.
// Plain loads, no read-only ones (__ldg) in these kernels: a chained kernel's lifetime overlaps that of the kernel in front, which may be writing
// these tensors, and read-only loads are defined only for data that nobody writes meanwhile (nor are they held behind chain_point()).
template <int E>
struct RowBits {
  uint32_t w[E];
  __device__ __forceinline__ void load(const void* base, size_t i, bool bf16) {
    if (bf16) {
      const __nv_bfloat16* p = static_cast<const __nv_bfloat16*>(base) + i;
      if constexpr (E == 1) w[0] = *reinterpret_cast<const unsigned short*>(p);
      else if constexpr (E == 2) w[0] = *reinterpret_cast<const uint32_t*>(p);
      else {
#pragma unroll
        for (int e = 0; e < E / 4; ++e) {
          const uint2 u = reinterpret_cast<const uint2*>(p)[e];
          w[2 * e] = u.x; w[2 * e + 1] = u.y;
        }
      }
    } else {
      const uint32_t* p = static_cast<const uint32_t*>(base) + i;
      if constexpr (E == 1) w[0] = *p;
      else {
#pragma unroll
        for (int e = 0; e < E / 2; ++e) {
          const uint2 u = reinterpret_cast<const uint2*>(p)[e];
          w[2 * e] = u.x; w[2 * e + 1] = u.y;
        }
      }
    }
  }
  __device__ __forceinline__ float get(int e, bool bf16) const {
    if (!bf16) return __uint_as_float(w[e]);
    const uint32_t u = w[e >> 1];
    return __uint_as_float((e & 1) ? u & 0xffff0000u : u << 16);
  }
};

// E (2 or 4) consecutive floats of a state row, streaming loads / stores of 8 or 16 bytes
template <int E>
__device__ __forceinline__ void ld_row(float (&d)[E], const float* p) {
  if constexpr (E == 4) {
    const float4 x = __ldcs(reinterpret_cast<const float4*>(p));
    d[0] = x.x; d[1] = x.y; d[2] = x.z; d[3] = x.w;
  } else {
    const float2 x = __ldcs(reinterpret_cast<const float2*>(p));
    d[0] = x.x; d[1] = x.y;
  }
}
template <int E>
__device__ __forceinline__ void st_row(float* p, const float (&d)[E]) {
  if constexpr (E == 4) __stcs(reinterpret_cast<float4*>(p), make_float4(d[0], d[1], d[2], d[3]));
  else __stcs(reinterpret_cast<float2*>(p), make_float2(d[0], d[1]));
}

// one decay per head (delta_recurrent.cu)
int recurrent_head_launch(const HeadArgs& a, cudaStream_t st);

}  // namespace kda
