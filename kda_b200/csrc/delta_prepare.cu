// Gated delta rule, one decay per token and head: what a chunk needs that does not depend on the state (see delta.cuh).
//
// One CTA per (chunk, head).  [K; Q] K^T is one product (128 x 64 x 128, its operands the input rows themselves); the decays, norms and beta multiply its
// fp32 result.  Tm = (I + A)^-1: the four 16 x 16 diagonal blocks by substitution in fp32, then two merges
// (T21 = -T2 A21 T1, at 16 and 32 rows), also in fp32: a merge by split bf16 products would take six dependent rounds on the tensor core.
// Pt = P Tm is a product again, in hi + lo parts, whose A operand's upper half is Tm's own tile (the rows it adds are not read).
// G is summed in double and kept as two floats: after a strong decay early in a chunk one float leaves 1e-5 in every later D_ij.
#include "delta.cuh"

namespace kda {
namespace delta {

namespace {

constexpr int PT = 256;      // 8 warps: TMEM lane quadrant = warp & 3, column half = warp >> 2

struct PrepSmem {
  unsigned char KQ[2][16384];      // [128 rows: k, then q][64 columns] x 2; once read, A and T (below)
  unsigned char TPh[16384], TPl[16384];
  double gs[2];
  float ghi[C], glo[C], beta[C], rk[C], rq[C], q2[2][C];
  uint64_t full, done;
  uint32_t tmem_slot;
};
static_assert(sizeof(PrepSmem) + 1024 <= 75 * 1024, "three CTAs per SM");

// element (i, j) of a 64 x 64 fp32 matrix; groups of four columns are permuted by the row so that a column of threads writes without conflicts
__device__ __forceinline__ int at(int i, int j) { return i * 64 + ((((j >> 2) ^ i) & 15) << 2) + (j & 3); }
__device__ __forceinline__ float4 at4(const float* m, int i, int j4) { return *reinterpret_cast<const float4*>(m + i * 64 + (((j4 ^ i) & 15) << 2)); }
__device__ __forceinline__ void axpy4(float4& y, float a, const float4& x) {
  y.x = fmaf(a, x.x, y.x); y.y = fmaf(a, x.y, y.y); y.z = fmaf(a, x.z, y.z); y.w = fmaf(a, x.w, y.w);
}

}  // namespace

__global__ void __launch_bounds__(PT, 3) delta_prepare_kernel(const __grid_constant__ PrepParams p) {
  chain_point();
  extern __shared__ unsigned char smem_raw[];
  PrepSmem& s = *reinterpret_cast<PrepSmem*>(smem_raw + pad_to_1024(smem_raw));
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, q4 = warp & 3, half = warp >> 2;
  const int c = blockIdx.x / p.H, h = blockIdx.x % p.H;
  if (p.clear_status && blockIdx.x == 0 && tid < 4) p.status[tid] = 0;
  if (c >= p.map.total()) return;
  const ChunkInfo ci = p.map.info(c);
  const size_t tile = static_cast<size_t>(c) * p.H + h;

  if (tid == 0) {
    mbar_init(&s.full, 1);
    mbar_init(&s.done, 1);
    fence_mbar_init();
    mbar_expect_tx(&s.full, 4 * 8192);
    for (int b = 0; b < 2; ++b) {
      tma_load_rows(s.KQ[b], &p.tm_k, 64 * b, h / p.grp, static_cast<int>(ci.tok0), &s.full);
      tma_load_rows(s.KQ[b] + 8192, &p.tm_q, 64 * b, h / p.grp, static_cast<int>(ci.tok0), &s.full);
    }
  }
  if (warp == 1) umma::tmem_alloc(&s.tmem_slot, 128);
  if (warp == 2 || warp == 3) {      // sums of g, in log2; rows behind the sequence's end neither decay nor write
    const int t = tid - 64;
    double x = 0.0;
    float b = 0.f;
    if (t < ci.len) {
      const size_t row = static_cast<size_t>(ci.tok0 + t) * p.H + h;
      float g = load_raw(p.g, row, p.g_dtype);
      if (g < -1e5f) g = -1e5f;      // -inf: the state is forgotten; differences of G stay numbers
      x = static_cast<double>(g) * 1.4426950408889634;
      b = load_raw(p.beta, row, p.beta_dtype);
    }
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const double y = __shfl_up_sync(0xffffffffu, x, off);
      if (lane >= off) x += y;
    }
    if (warp == 2 && lane == 31) s.gs[0] = x;
    asm volatile("bar.sync 1, 64;" ::: "memory");
    if (warp == 3) x += s.gs[0];
    s.ghi[t] = static_cast<float>(x);
    s.glo[t] = static_cast<float>(x - static_cast<double>(static_cast<float>(x)));
    s.beta[t] = b;
  }
  umma::fence_before_sync();
  __syncthreads();
  umma::fence_after_sync();
  const uint32_t tb = s.tmem_slot, tq = tb + (static_cast<uint32_t>(32 * q4) << 16);

  bool ok = mbar_wait(&s.full, 0);
  if (tid == 0 && ok) {
    constexpr uint32_t id = umma::instr_desc(128, 64, false, false);
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      const uint64_t d = umma::desc_kmajor(smem_u32(s.KQ[b]), 0);
      umma::mma4<umma::KSTEP_KMAJOR, umma::KSTEP_KMAJOR>(tb, d, d, id, b);
    }
    umma::commit(&s.done);
  }
  __syncwarp();
  if (p.use_l2norm && q4 >= 2) {      // |q|^2, half a row per thread (|k|^2 stands on the product's diagonal)
    const int t = 32 * (q4 - 2) + lane;
    float a = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      float x[8];
      unpack8(*reinterpret_cast<const uint4*>(piece(s.KQ[half] + 8192, t, e)), x);
#pragma unroll
      for (int i = 0; i < 8; ++i) a = fmaf(x[i], x[i], a);
    }
    s.q2[half][t] = a;
  }
  ok = ok && mbar_wait(&s.done, 0);
  umma::fence_after_sync();
  float S[32];
  if (__all_sync(0xffffffffu, ok)) {
    umma::tmem_ld16(tq + 32 * half, *reinterpret_cast<float(*)[16]>(&S[0]));
    umma::tmem_ld16(tq + 32 * half + 16, *reinterpret_cast<float(*)[16]>(&S[16]));
    umma::tmem_ld_wait();
  }
  const int i = 32 * (q4 & 1) + lane;      // this thread's row, of A (q4 < 2) or of P; its columns 32 half ..
  if (q4 < 2 && half == (i >> 5)) {
    float d = 0.f;
#pragma unroll
    for (int e = 0; e < 32; ++e) d = e == (i & 31) ? S[e] : d;
    s.rk[i] = p.use_l2norm ? rsqrtf(d + L2NORM_EPS) : 1.f;
  }
  ok = __syncthreads_and(ok);
  if (tid < C) s.rq[tid] = p.use_l2norm ? rsqrtf(s.q2[0][tid] + s.q2[1][tid] + L2NORM_EPS) : 1.f;
  __syncthreads();
  if (ok) {
    float* const A = reinterpret_cast<float*>(s.KQ[0]);
    float* const T = reinterpret_cast<float*>(s.KQ[1]);
    {
      const float gh = s.ghi[i], gl = s.glo[i], f = q4 < 2 ? s.beta[i] * s.rk[i] : p.scale * s.rq[i];
      const int last = i < ci.len ? (q4 < 2 ? i - 1 : i) : -1;      // columns beyond it are zero, whatever stands in the rows' products
#pragma unroll
      for (int e = 0; e < 32; ++e) {
        const int j = 32 * half + e;
        S[e] = j <= last ? S[e] * (f * s.rk[j]) * ex2((gh - s.ghi[j]) + (gl - s.glo[j])) : 0.f;
      }
    }
    if (q4 < 2) {
#pragma unroll
      for (int e = 0; e < 8; ++e) *reinterpret_cast<float4*>(&A[at(i, 32 * half + 4 * e)]) = make_float4(S[4 * e], S[4 * e + 1], S[4 * e + 2], S[4 * e + 3]);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const Split x = split8(&S[8 * e]);
        *reinterpret_cast<uint4*>(piece(s.TPh, 64 + i, 4 * half + e)) = x.hi;
        *reinterpret_cast<uint4*>(piece(s.TPl, 64 + i, 4 * half + e)) = x.lo;
      }
    }
    __syncthreads();
    // ---- Tm: diagonal blocks by substitution, a column per thread; meanwhile the others write VEC ------------------------------------------------
    if (tid < 64) {
      const int b = tid & ~15, col = tid & 15;
      float x[16];
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        float acc = r == col ? 1.f : 0.f;
#pragma unroll
        for (int j4 = 0; j4 < (r + 3) / 4; ++j4) {
          const float4 a = at4(A, b + r, (b >> 2) + j4);
          if (4 * j4 < r) acc = fmaf(-a.x, x[4 * j4], acc);
          if (4 * j4 + 1 < r) acc = fmaf(-a.y, x[4 * j4 + 1], acc);
          if (4 * j4 + 2 < r) acc = fmaf(-a.z, x[4 * j4 + 2], acc);
          if (4 * j4 + 3 < r) acc = fmaf(-a.w, x[4 * j4 + 3], acc);
        }
        x[r] = acc;
        T[at(b + r, b + col)] = acc;
      }
    } else if (tid >= 128 && tid < 192) {
      const int t = tid - 128;
      float* const v = reinterpret_cast<float*>(p.VEC + tile * T_VEC);
      const float gh = s.ghi[t], gl = s.glo[t], lh = s.ghi[63], ll = s.glo[63], e = ex2(gh + gl), rk = s.rk[t], rq = s.rq[t], b = s.beta[t];
      const bool there = t < ci.len;
      v[V_BETA + t] = b;
      v[V_KG + t] = there ? b * e * rk : 0.f;
      v[V_W + t] = there ? ex2((lh - gh) + (ll - gl)) * rk : 0.f;
      v[V_Q + t] = there ? p.scale * e * rq : 0.f;
      v[V_GHI + t] = gh;
      v[V_GLO + t] = gl;
      v[V_RK + t] = there ? rk : 0.f;
      v[V_RQ + t] = there ? rq : 0.f;
      if (t < 4) v[V_LAST + t] = ex2(lh + ll);
    }
    __syncthreads();
    // ---- merges: X = A21 T1 into the unused upper right of T, then T21 = -T2 X ---------------------------------------------------------------------
    {
      const int b = 32 * (tid >> 7), r = (tid >> 3) & 15, c4 = tid & 3, m0 = (tid & 4) ? 8 : 0;      // eight terms of four columns per thread, two threads a sum
      auto pairsum = [](float4 x) {
        x.x += __shfl_xor_sync(0xffffffffu, x.x, 4);
        x.y += __shfl_xor_sync(0xffffffffu, x.y, 4);
        x.z += __shfl_xor_sync(0xffffffffu, x.z, 4);
        x.w += __shfl_xor_sync(0xffffffffu, x.w, 4);
        return x;
      };
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int m = 0; m < 8; ++m) {      // T1 above its diagonal is not written: zero
        float4 t = at4(T, b + m0 + m, (b >> 2) + c4);
        const int d = m0 + m - 4 * c4;
        if (d < 0) t.x = 0.f;
        if (d < 1) t.y = 0.f;
        if (d < 2) t.z = 0.f;
        if (d < 3) t.w = 0.f;
        axpy4(acc, A[at(b + 16 + r, b + m0 + m)], t);
      }
      acc = pairsum(acc);
      if (!(tid & 4)) *reinterpret_cast<float4*>(&T[at(b + r, b + 16 + 4 * c4)]) = acc;
      __syncthreads();
      acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int m = 0; m < 8; ++m)
        if (m0 + m <= r) axpy4(acc, -T[at(b + 16 + r, b + 16 + m0 + m)], at4(T, b + m0 + m, (b >> 2) + 4 + c4));
      acc = pairsum(acc);
      if (!(tid & 4)) *reinterpret_cast<float4*>(&T[at(b + 16 + r, b + 4 * c4)]) = acc;
    }
    __syncthreads();
    {
      const int r = tid >> 3, c4 = tid & 7;
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
      for (int m = 0; m < 32; ++m) {
        float4 t = at4(T, m, c4);
        const int d = m - 4 * c4;
        if (d < 0) t.x = 0.f;
        if (d < 1) t.y = 0.f;
        if (d < 2) t.z = 0.f;
        if (d < 3) t.w = 0.f;
        axpy4(acc, A[at(32 + r, m)], t);
      }
      *reinterpret_cast<float4*>(&T[at(r, 32 + 4 * c4)]) = acc;
      __syncthreads();
      acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
      for (int m = 0; m < 32; ++m)
        if (m <= r) axpy4(acc, -T[at(32 + r, 32 + m)], at4(T, m, 8 + c4));
      *reinterpret_cast<float4*>(&T[at(32 + r, 4 * c4)]) = acc;
    }
    __syncthreads();
    {      // Tm as an operand
      const int r = tid >> 2, c0 = 16 * (tid & 3);
      float x[16];
#pragma unroll
      for (int e = 0; e < 4; ++e) *reinterpret_cast<float4*>(&x[4 * e]) = at4(T, r, (c0 >> 2) + e);
#pragma unroll
      for (int e = 0; e < 16; ++e)
        if (c0 + e > r) x[e] = 0.f;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const Split y = split8(&x[8 * e]);
        *reinterpret_cast<uint4*>(piece(s.TPh, r, (c0 >> 3) + e)) = y.hi;
        *reinterpret_cast<uint4*>(piece(s.TPl, r, (c0 >> 3) + e)) = y.lo;
      }
    }
    fence_proxy_async();
    umma::fence_before_sync();
    __syncthreads();
    umma::fence_after_sync();
    if (tid == 0) {      // [Tm; P] Tm: the lower half is wanted
      constexpr uint32_t id = umma::instr_desc(128, 64, false, true);
      const uint64_t ah = umma::desc_kmajor(smem_u32(s.TPh), 0), al = umma::desc_kmajor(smem_u32(s.TPl), 0);
      const uint64_t bh = umma::desc_mnmajor(smem_u32(s.TPh), 0, 8192), bl = umma::desc_mnmajor(smem_u32(s.TPl), 0, 8192);
      umma::mma4<umma::KSTEP_KMAJOR, umma::KSTEP_MNMAJOR>(tb + 64, ah, bh, id, 0);
      umma::mma4<umma::KSTEP_KMAJOR, umma::KSTEP_MNMAJOR>(tb + 64, ah, bl, id, 1);
      umma::mma4<umma::KSTEP_KMAJOR, umma::KSTEP_MNMAJOR>(tb + 64, al, bh, id, 1);
      umma::commit(&s.done);
    }
    __syncwarp();
    if (q4 >= 2) {
      ok = warp_wait(&s.done, 1);
      umma::fence_after_sync();
      if (ok) {
        umma::tmem_ld16(tq + 64 + 32 * half, *reinterpret_cast<float(*)[16]>(&S[0]));
        umma::tmem_ld16(tq + 64 + 32 * half + 16, *reinterpret_cast<float(*)[16]>(&S[16]));
        umma::tmem_ld_wait();
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const Split x = split8(&S[8 * e]);
          *reinterpret_cast<uint4*>(piece(s.TPh, 64 + i, 4 * half + e)) = x.hi;
          *reinterpret_cast<uint4*>(piece(s.TPl, 64 + i, 4 * half + e)) = x.lo;
        }
      }
      fence_proxy_async();
    }
    umma::fence_before_sync();
    ok = __syncthreads_and(ok);
    if (tid == 0 && ok) {
      bulk_s2g(p.TP + tile * T_TP, s.TPh, 16384);
      bulk_s2g(p.TP + tile * T_TP + 16384, s.TPl, 16384);
      bulk_commit();
      bulk_wait<0>();
    }
  }
  if (!ok && tid == 0) {      // a wait gave up: loads and products may still be under way
    atomicOr(p.status, KDA_STATUS_PREP_LOAD_WAIT);
    mbar_drain(&s.full);
    mbar_drain(&s.done);
  }
  __syncthreads();
  if (warp == 1) umma::tmem_dealloc(tb, 128);
}

int launch_prepare(const PrepParams& p, long long tiles, cudaStream_t st) {
  static DeviceOnce once;
  const int smem = static_cast<int>(sizeof(PrepSmem)) + 1024;
  const int rc = once.run([&] { return cudaFuncSetAttribute(delta_prepare_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem); });
  if (rc != KDA_OK) return rc;
  if (tiles > 0x7fffffffLL) return KDA_E_SHAPE;
  return static_cast<int>(launch_chained(delta_prepare_kernel, static_cast<unsigned>(tiles), PT, smem, st, p));
}

}  // namespace delta
}  // namespace kda
