// Gated delta rule, one decay per token and head: what a chunk needs that does not depend on the state (see delta.cuh).
//
// One CTA per (chunk, head), three of them on an SM.  [K; Q] K^T is one product (128 x 64 x 128, its operands the input rows themselves); the decays, norms and
// beta multiply its fp32 result.  Tm = (I + A)^-1: the four 16 x 16 diagonal blocks by substitution in fp32, then two merges
// T21 = -(T2 A21) T1, at 16 and 32 rows, by mma.sync on bf16 pairs: T2 A21 leaves the first product in the layout that the second takes its A in.
// Pt = P Tm is a product of the tensor core again, in pairs, whose A operand's upper half is Tm's own tile (the rows it adds are not read).
// G is summed in double and kept as two floats: after a strong decay early in a chunk one float leaves 1e-5 in every later D_ij.
// Bound by instruction issue and shared memory (with the merges as fp32 sums over shared memory 25 k warp instructions and 5.8 k wavefronts a tile: 578 us for
// 16,384 tiles).
#include "delta.cuh"

namespace kda {
namespace delta {

namespace {

constexpr int PT = 256;      // 8 warps: TMEM lane quadrant = warp & 3, column half = warp >> 2

struct PrepSmem {
  union {
    unsigned char KQ[2][16384];    // [128 rows: k, then q][64 columns] x 2
    struct {                       // once those are read:
      unsigned char Ah[8192], Al[8192];      // A as bf16 pairs, [64][64]
      float D[4][16][20];                    // its diagonal blocks in fp32
    };
  };
  unsigned char TPh[16384], TPl[16384];
  double gs[2];
  float ghi[C], glo[C], beta[C], rk[C], rq[C], q2[2][C];
  uint64_t full, done;
  uint32_t tmem_slot;
};
static_assert(sizeof(PrepSmem) + 1024 <= 75 * 1024, "three CTAs per SM");

// a pair of neighbours (row, col), (row, col + 1) as bf16 pairs
__device__ __forceinline__ void put2(unsigned char* hi, unsigned char* lo, int row, int col, float a, float b) {
  uint32_t h, l;
  split2(a, b, h, l);
  *reinterpret_cast<uint32_t*>(hi + umma::sw128(row, col)) = h;
  *reinterpret_cast<uint32_t*>(lo + umma::sw128(row, col)) = l;
}
// The 16 x 16 block at (row, col) of a tile as an A operand; the 16 x 16 block as a B operand of two products of eight columns.
__device__ __forceinline__ void frag_a(uint32_t (&f)[4], const unsigned char* tile, int row, int col, int lane) {
  ldsm_x4(f, smem_u32(tile) + umma::sw128(row + (lane & 15), col + 8 * (lane >> 4)));
}
__device__ __forceinline__ void frag_b(uint32_t (&f)[4], const unsigned char* tile, int row, int col, int lane) {
  ldsm_x4_t(f, smem_u32(tile) + umma::sw128(row + (lane & 15), col + 8 * (lane >> 4)));
}
struct FragPair { uint32_t h[4], l[4]; };
// c (16 x 16: two accumulators) += a b in pairs, without the product of the low parts
__device__ __forceinline__ void mma_pair(float (&c)[2][4], const FragPair& a, const FragPair& b) {
#pragma unroll
  for (int n = 0; n < 2; ++n) {
    mma16816(c[n], a.l, b.h[2 * n], b.h[2 * n + 1]);
    mma16816(c[n], a.h, b.l[2 * n], b.l[2 * n + 1]);
    mma16816(c[n], a.h, b.h[2 * n], b.h[2 * n + 1]);
  }
}
// an accumulated 16 x 16 block as the A operand of the next product: the accumulator's layout is the operand's
__device__ __forceinline__ FragPair as_a(const float (&c)[2][4]) {
  FragPair f;
#pragma unroll
  for (int n = 0; n < 2; ++n) {
    split2(c[n][0], c[n][1], f.h[2 * n], f.l[2 * n]);
    split2(c[n][2], c[n][3], f.h[2 * n + 1], f.l[2 * n + 1]);
  }
  return f;
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
    // ---- A and P: rows times decays ------------------------------------------------------------------------------------------------------------------
    const bool above = half > (q4 & 1);      // this warp's columns lie above the diagonal block row: zero
    if (!above) {
      const float gh = s.ghi[i], gl = s.glo[i], f = q4 < 2 ? s.beta[i] * s.rk[i] : p.scale * s.rq[i];
      const int last = i < ci.len ? (q4 < 2 ? i - 1 : i) : -1;      // columns beyond it are zero, whatever stands in the rows' products
#pragma unroll
      for (int e = 0; e < 32; e += 4) {
        const int j = 32 * half + e;
        const float4 h4 = *reinterpret_cast<const float4*>(&s.ghi[j]), l4 = *reinterpret_cast<const float4*>(&s.glo[j]), r4 = *reinterpret_cast<const float4*>(&s.rk[j]);
        S[e] = j <= last ? S[e] * (f * r4.x) * ex2((gh - h4.x) + (gl - l4.x)) : 0.f;
        S[e + 1] = j + 1 <= last ? S[e + 1] * (f * r4.y) * ex2((gh - h4.y) + (gl - l4.y)) : 0.f;
        S[e + 2] = j + 2 <= last ? S[e + 2] * (f * r4.z) * ex2((gh - h4.z) + (gl - l4.z)) : 0.f;
        S[e + 3] = j + 3 <= last ? S[e + 3] * (f * r4.w) * ex2((gh - h4.w) + (gl - l4.w)) : 0.f;
      }
    } else {
#pragma unroll
      for (int e = 0; e < 32; ++e) S[e] = 0.f;
    }
    {
      unsigned char* const hi = q4 < 2 ? s.Ah : s.TPh + 8192;
      unsigned char* const lo = q4 < 2 ? s.Al : s.TPl + 8192;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const Split x = split8(&S[8 * e]);
        *reinterpret_cast<uint4*>(piece(hi, i, 4 * half + e)) = x.hi;
        *reinterpret_cast<uint4*>(piece(lo, i, 4 * half + e)) = x.lo;
        if (q4 < 2) {      // Tm begins as zeros: what stays so is its part above the diagonal
          *reinterpret_cast<uint4*>(piece(s.TPh, i, 4 * half + e)) = make_uint4(0, 0, 0, 0);
          *reinterpret_cast<uint4*>(piece(s.TPl, i, 4 * half + e)) = make_uint4(0, 0, 0, 0);
        }
      }
      if (q4 < 2 && half == q4) {
        const int b = lane >> 4;      // the diagonal block of this row begins at column 16 b of its half
#pragma unroll
        for (int e = 0; e < 4; ++e)
          *reinterpret_cast<float4*>(&s.D[i >> 4][i & 15][4 * e]) = b ? make_float4(S[16 + 4 * e], S[17 + 4 * e], S[18 + 4 * e], S[19 + 4 * e])
                                                                       : make_float4(S[4 * e], S[4 * e + 1], S[4 * e + 2], S[4 * e + 3]);
      }
    }
    __syncthreads();
    // ---- Tm: diagonal blocks by substitution, a column per thread; meanwhile others write VEC ----------------------------------------------------------
    if (tid < 64) {
      const int b = tid >> 4, col = tid & 15;
      float x[16];
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        float acc = r == col ? 1.f : 0.f;
#pragma unroll
        for (int j4 = 0; j4 < (r + 3) / 4; ++j4) {
          const float4 a = *reinterpret_cast<const float4*>(&s.D[b][r][4 * j4]);
          if (4 * j4 < r) acc = fmaf(-a.x, x[4 * j4], acc);
          if (4 * j4 + 1 < r) acc = fmaf(-a.y, x[4 * j4 + 1], acc);
          if (4 * j4 + 2 < r) acc = fmaf(-a.z, x[4 * j4 + 2], acc);
          if (4 * j4 + 3 < r) acc = fmaf(-a.w, x[4 * j4 + 3], acc);
        }
        x[r] = acc;
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const __nv_bfloat16 hi = __float2bfloat16_rn(x[r]);
        const uint32_t off = umma::sw128(16 * b + r, 16 * b + col);
        *reinterpret_cast<__nv_bfloat16*>(s.TPh + off) = hi;
        *reinterpret_cast<__nv_bfloat16*>(s.TPl + off) = __float2bfloat16_rn(x[r] - __bfloat162float(hi));
      }
      __syncwarp();
      // ---- merge of 16: each of the two warps has written both diagonal blocks of its pair -------------------------------------------------------------
      const int r0 = 32 * warp;
      FragPair t2, a21, t1;
      frag_a(t2.h, s.TPh, r0 + 16, r0 + 16, lane);
      frag_a(t2.l, s.TPl, r0 + 16, r0 + 16, lane);
      frag_b(a21.h, s.Ah, r0 + 16, r0, lane);
      frag_b(a21.l, s.Al, r0 + 16, r0, lane);
      frag_b(t1.h, s.TPh, r0, r0, lane);
      frag_b(t1.l, s.TPl, r0, r0, lane);
      float y[2][4] = {}, z[2][4] = {};
      mma_pair(y, t2, a21);
      mma_pair(z, as_a(y), t1);
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        put2(s.TPh, s.TPl, r0 + 16 + (lane >> 2), r0 + 8 * n + 2 * (lane & 3), -z[n][0], -z[n][1]);
        put2(s.TPh, s.TPl, r0 + 24 + (lane >> 2), r0 + 8 * n + 2 * (lane & 3), -z[n][2], -z[n][3]);
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
    // ---- merge of 32: warps 0..3, 16 rows and 16 of the 32 columns each ----------------------------------------------------------------------------------
    if (warp < 4) {
      const int rb = warp & 1, n0 = 16 * (warp >> 1), r0 = 32 + 16 * rb;
      float y[2][2][4] = {}, z[2][4] = {};      // T2 A21: 16 rows, 32 columns
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        if (m > rb) break;                       // T2's upper right block is zero
        FragPair t2;
        frag_a(t2.h, s.TPh, r0, 32 + 16 * m, lane);
        frag_a(t2.l, s.TPl, r0, 32 + 16 * m, lane);
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          FragPair a21;
          frag_b(a21.h, s.Ah, 32 + 16 * m, 16 * n, lane);
          frag_b(a21.l, s.Al, 32 + 16 * m, 16 * n, lane);
          mma_pair(y[n], t2, a21);
        }
      }
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        FragPair t1;
        frag_b(t1.h, s.TPh, 16 * m, n0, lane);
        frag_b(t1.l, s.TPl, 16 * m, n0, lane);
        mma_pair(z, as_a(y[m]), t1);
      }
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        put2(s.TPh, s.TPl, r0 + (lane >> 2), n0 + 8 * n + 2 * (lane & 3), -z[n][0], -z[n][1]);
        put2(s.TPh, s.TPl, r0 + 8 + (lane >> 2), n0 + 8 * n + 2 * (lane & 3), -z[n][2], -z[n][3]);
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
      bulk_wait_read<0>();      // shared memory may go; the writes are complete with the kernel
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
