// Shared by the kernels of the norms around a block (kda_norm.cu: the formulas).
#pragma once

#include "kda_common.cuh"
#include "kda_device.cuh"

namespace kda {

constexpr int NORM_MOST = 8192;         // columns
// Elements of a call from which rows travel through shared memory (kda_norm_ring.cu).  us, ring | direct, gated in bf16, then with an fp32 residual:
//   forward, 2^22 and 2^23 elements   128 columns 7.5 | 8.0, 11.0 | 14.2; 10.5 | 11.3, 18.4 | 22.4     4096: 9.3 | 8.0, 13.1 | 14.1; 12.1 | 13.9, 22.5 | 28.1
//   backward, 2^19 and 2^20           128 columns 8.5 | 6.6, 8.9 | 9.6; 9.7 | 9.0, 12.1 | 13.6         4096: 10.8 | 8.6, 11.3 | 13.6; 17.7 | 14.7, 21.2 | 24.1
constexpr int64_t ring_min(bool backward) { return backward ? 1 << 20 : 1 << 23; }

bool norm_ring_covers(const kda_norm_args& a, bool gated, bool backward);
size_t norm_ring_partials();
// launches it; *partials: the number of partial sums over rows that it leaves, as [partials][sums][cols]
int norm_ring(const kda_norm_args& a, bool gated, bool backward, float* partial, int* partials, cudaStream_t st);

int norm_ring_status(uint32_t* host_out);

inline bool norm_aligned(const kda_norm_args& a) {
  uintptr_t bits = 0;
  for (const void* p : {a.x, a.gate, a.residual, a.weight, a.post_weight, a.scale, static_cast<const void*>(a.y), static_cast<const void*>(a.r), a.dy, a.dr,
                        static_cast<const void*>(a.dx), static_cast<const void*>(a.dgate), static_cast<const void*>(a.dresidual)})
    bits |= reinterpret_cast<uintptr_t>(p);
  return (bits & 15u) == 0;
}

struct Bits { uint4 a, b; };            // eight values as they stand in memory: fp32, or bf16 in a

template <bool VEC>
struct Cols {                           // which columns a thread has: vector i of a row whose threads are `lane` of `lanes`
  int lane, lanes, cols;
  __device__ __forceinline__ bool any(int i) const { return VEC ? (i * lanes + lane) * 8 < cols : i * 8 * lanes + lane < cols; }
  __device__ __forceinline__ int at(int i, int j) const { return VEC ? (i * lanes + lane) * 8 + j : (i * 8 + j) * lanes + lane; }
  __device__ __forceinline__ bool has(int i, int j) const { return VEC || at(i, j) < cols; }
};

template <bool VEC>
__device__ __forceinline__ Bits fetch(const void* p, size_t row, int dtype, const Cols<VEC>& c, int i) {
  Bits r{make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
  const size_t base = row * c.cols;
  if constexpr (VEC) {
    if (c.any(i)) {
      if (dtype == KDA_BF16) r.a = *reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(p) + base + c.at(i, 0));
      else {
        const uint4* q = reinterpret_cast<const uint4*>(static_cast<const float*>(p) + base + c.at(i, 0));
        r.a = q[0];
        r.b = q[1];
      }
    }
  } else {
    uint32_t w[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      w[j] = 0;
      if (c.has(i, j)) w[j] = dtype == KDA_BF16 ? static_cast<const unsigned short*>(p)[base + c.at(i, j)] : static_cast<const uint32_t*>(p)[base + c.at(i, j)];
    }
    if (dtype == KDA_BF16) r.a = make_uint4(w[0] | w[1] << 16, w[2] | w[3] << 16, w[4] | w[5] << 16, w[6] | w[7] << 16);
    else {
      r.a = make_uint4(w[0], w[1], w[2], w[3]);
      r.b = make_uint4(w[4], w[5], w[6], w[7]);
    }
  }
  return r;
}
__device__ __forceinline__ void values(const Bits& r, int dtype, float (&v)[8]) {
  if (dtype == KDA_BF16) {
    const float2 a = unpack_bf16(r.a.x), b = unpack_bf16(r.a.y), c = unpack_bf16(r.a.z), d = unpack_bf16(r.a.w);
    v[0] = a.x; v[1] = a.y; v[2] = b.x; v[3] = b.y; v[4] = c.x; v[5] = c.y; v[6] = d.x; v[7] = d.y;
  } else {
    v[0] = __uint_as_float(r.a.x); v[1] = __uint_as_float(r.a.y); v[2] = __uint_as_float(r.a.z); v[3] = __uint_as_float(r.a.w);
    v[4] = __uint_as_float(r.b.x); v[5] = __uint_as_float(r.b.y); v[6] = __uint_as_float(r.b.z); v[7] = __uint_as_float(r.b.w);
  }
}
template <bool VEC>
__device__ __forceinline__ void load8(const void* p, size_t row, int dtype, const Cols<VEC>& c, int i, float (&v)[8]) { values(fetch<VEC>(p, row, dtype, c, i), dtype, v); }
template <bool VEC>
__device__ __forceinline__ void store8(void* p, size_t row, int dtype, const Cols<VEC>& c, int i, const float (&v)[8]) {
  if (!c.any(i)) return;
  const size_t base = row * c.cols;
  if constexpr (VEC) {
    if (dtype == KDA_BF16) {
      *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(p) + base + c.at(i, 0)) =
          make_uint4(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7]));
    } else {
      float4* q = reinterpret_cast<float4*>(static_cast<float*>(p) + base + c.at(i, 0));
      q[0] = make_float4(v[0], v[1], v[2], v[3]);
      q[1] = make_float4(v[4], v[5], v[6], v[7]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (c.has(i, j)) {
        if (dtype == KDA_BF16) static_cast<__nv_bfloat16*>(p)[base + c.at(i, j)] = __float2bfloat16_rn(v[j]);
        else static_cast<float*>(p)[base + c.at(i, j)] = v[j];
      }
  }
}

// The gate's activation and its slope.  For bf16 results the fast exponential and reciprocal do (their error grows with |z|: 4e-6 at 86).  EXACT, for float32 x: to float32's
// rounding.  Beyond +-88 sigmoid or what is left of it is below the normal float32 numbers, and zero; NaN stays.
template <bool EXACT>
__device__ __forceinline__ void act_of(float z, int activation, float& act, float& slope) {
  if constexpr (EXACT) {
    z = at_least(z, -88.f);
    const float zc = at_most(z, 88.f);
    float rest;
    const float sg = sigmoid_within(zc, rest);
    act = activation == KDA_ACT_SILU ? z * sg : sg;
    slope = activation == KDA_ACT_SILU ? sg * fmaf(zc, rest, 1.f) : sg * rest;
  } else {
    const float sg = sigmoid_fast(z);
    act = activation == KDA_ACT_SILU ? z * sg : sg;
    slope = activation == KDA_ACT_SILU ? sg * fmaf(z, 1.f - sg, 1.f) : sg * (1.f - sg);
  }
}

// eight columns of a parameter (1 where there is none), of the scale (its one value where it is a number)
template <bool VEC>
__device__ __forceinline__ void param8(const void* p, int dtype, float other, const Cols<VEC>& c, int i, float (&v)[8]) {
  if (p) load8<VEC>(p, 0, dtype, c, i, v);
  else
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = other;
}

}  // namespace kda
