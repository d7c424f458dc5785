// Gated delta rule, one decay per token and head: what a chunk needs that does not depend on the state (see delta.cuh).
//
// Persistent CTAs, three on an SM, a tile per (chunk, head).  [K; Q] K^T is one product (128 x 64 x 128, its operands the input rows themselves); the decays, norms and
// beta multiply its fp32 result.  Tm = (I + A)^-1: the four 16 x 16 diagonal blocks by substitution in fp32, then two merges
// T21 = -(T2 A21) T1, at 16 and 32 rows, by mma.sync on bf16 pairs: T2 A21 leaves the first product in the layout that the second takes its A in.
// Pt = P Tm is a product of the tensor core again, in pairs, whose A operand's upper half is Tm's own tile (the rows it adds are not read).
// G is a sum of two floats each: after a strong decay early in a chunk one float leaves 1e-5 in every later D_ij.
// A tile is a row of short phases, each of them latency (14 k cycles a tile, 2 k of them instructions): the next tile's k and q are fetched once this one's have
// been read, its g and beta while this one is worked on (16,384 tiles of 8 x 4,096 tokens x 32 heads: 294 us, their bytes alone 165;
// 310 with a CTA per tile, whose loads, tensor memory and stores nobody hid;
// 578 with Tm's merges as fp32 sums over shared memory).
#include <algorithm>

#include "delta.cuh"

namespace kda {
namespace delta {

namespace {

constexpr int PT = 256;      // 8 warps: TMEM lane quadrant = warp & 3, column half = warp >> 2

struct PrepSmem {
  unsigned char KQ[2][16384];      // [128 rows: k, then q][64 columns] x 2
  unsigned char TPh[16384], TPl[16384];      // rows 0..63: A, which Tm replaces block by block; rows 64..127: P, then Pt
  float D[4][16][16];              // A's diagonal blocks in fp32, transposed
  float gs[2];
  struct Tile { int tok0, len, h; } next[2];      // where a tile is, by the thread that fetches it
  float ghi[C], glo[C], beta[C], rk[C], rq[C], q2[3][C];      // q2: of q's row halves, of k's rows
  float to16[C], to32[C];          // decay from a token to the end of its 16 tokens, of its 32
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
// the sum of two numbers as two floats each, to the last bit but a few of 48 (Knuth's sum with its rounding error, of the high parts)
struct Two { float hi, lo; };
__device__ __forceinline__ Two add(const Two& a, const Two& b) {
  const float s = a.hi + b.hi, v = s - a.hi, e = (a.hi - (s - v)) + (b.hi - v) + (a.lo + b.lo), hi = s + e;
  return {hi, e - (hi - s)};
}
// exp(G_i - G_j)
__device__ __forceinline__ float decay_between(const PrepSmem& s, int i, int j) { return ex2((s.ghi[i] - s.ghi[j]) + (s.glo[i] - s.glo[j])); }
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
  if (p.clear_status && blockIdx.x == 0 && tid < 4) p.status[tid] = 0;
  const int total = p.map.total() * p.H;      // (below 2^31: checked by the entry points)
  if (static_cast<int>(blockIdx.x) >= total) return;

  auto place = [&](int tile) {
    const ChunkInfo ci = p.map.info(tile / p.H);
    return PrepSmem::Tile{static_cast<int>(ci.tok0), ci.len, tile % p.H};
  };
  auto load = [&](const PrepSmem::Tile& x) {      // one thread: k's and q's rows
    mbar_expect_tx(&s.full, 4 * 8192);
    for (int b = 0; b < 2; ++b) {
      tma_load_rows(s.KQ[b], &p.tm_k, 64 * b, x.h / p.grp, x.tok0, &s.full);
      tma_load_rows(s.KQ[b] + 8192, &p.tm_q, 64 * b, x.h / p.grp, x.tok0, &s.full);
    }
  };
  const bool gater = warp == 4 || warp == 5;      // a token of the tile per thread
  const bool fetcher = tid == 192;                // (of a warp whose part of A or P is zero)
  float g_next = 0.f, b_next = 0.f;
  auto load_gates = [&](const PrepSmem::Tile& x) {         // rows behind the sequence's end neither decay nor write
    g_next = b_next = 0.f;
    if (tid - 128 < x.len) {
      const size_t row = static_cast<size_t>(x.tok0 + tid - 128) * p.H + x.h;
      g_next = load_raw(p.g, row, p.g_dtype);
      b_next = load_raw(p.beta, row, p.beta_dtype);
    }
  };
  if (fetcher) {
    mbar_init(&s.full, 1);
    mbar_init(&s.done, 1);
    fence_mbar_init();
    s.next[0] = place(blockIdx.x);
    load(s.next[0]);
  }
  if (warp == 1) umma::tmem_alloc(&s.tmem_slot, 128);
  umma::fence_before_sync();
  __syncthreads();
  umma::fence_after_sync();
  if (gater) load_gates(s.next[0]);
  const uint32_t tb = s.tmem_slot, tq = tb + (static_cast<uint32_t>(32 * q4) << 16);

  bool ok = true;
  unsigned phase = 0;
  for (int tile = blockIdx.x; tile < total; tile += gridDim.x, phase ^= 1u) {
    const int next = tile + gridDim.x;
    const int len = s.next[phase].len;
    if (fetcher && next < total) s.next[phase ^ 1] = place(next);
    ok = mbar_wait(&s.full, phase);
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
    // ---- beside the product: norms and sums of g ----
    if (!gater) {
      const int row = q4 < 2 ? 32 * q4 + lane : 64 + 32 * (q4 - 2) + lane;      // warps 0, 1: a row of k; 2, 3, 6, 7: half a row of q
      float a = 0.f;
      if (p.use_l2norm) {
        for (int b = q4 < 2 ? 0 : half; b <= (q4 < 2 ? 1 : half); ++b)
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            float x[8];
            unpack8(*reinterpret_cast<const uint4*>(piece(s.KQ[b], row, e)), x);
#pragma unroll
            for (int i = 0; i < 8; ++i) a = fmaf(x[i], x[i], a);
          }
      }
      if (q4 < 2) s.rk[row] = p.use_l2norm ? rsqrtf(a + L2NORM_EPS) : 1.f;
      else s.q2[half][row - 64] = a;
    } else {      // sums of g, in log2
      const int t = tid - 128;
      const float g = g_next < -1e5f ? -1e5f : g_next;      // -inf: the state is forgotten; differences of G stay numbers
      Two x{g * LOG2E, 0.f};
      x.lo = fmaf(g, LOG2E, -x.hi) + g * LOG2E_REST;
#pragma unroll
      for (int off = 1; off < 32; off <<= 1) {
        const Two y{__shfl_up_sync(0xffffffffu, x.hi, off), __shfl_up_sync(0xffffffffu, x.lo, off)};
        if (lane >= off) x = add(x, y);
      }
      if (warp == 4 && lane == 31) {
        s.gs[0] = x.hi;
        s.gs[1] = x.lo;
      }
      asm volatile("bar.sync 1, 64;" ::: "memory");
      if (warp == 5) x = add(x, Two{s.gs[0], s.gs[1]});
      s.ghi[t] = x.hi;
      s.glo[t] = x.lo;
      s.beta[t] = b_next;
      asm volatile("bar.sync 1, 64;" ::: "memory");
      s.to16[t] = decay_between(s, t | 15, t);
      s.to32[t] = decay_between(s, t | 31, t);
    }
    if (tid == 0) bulk_wait_read<0>();       // the tile before has left TP
    ok = __syncthreads_and(ok);
    if (gater && next < total) load_gates(s.next[phase ^ 1]);
    ok = ok && mbar_wait(&s.done, 0);
    umma::fence_after_sync();
    const int i = 32 * (q4 & 1) + lane;      // this thread's row, of A (q4 < 2) or of P; its columns 32 half ..
    float S[32];
    if (__all_sync(0xffffffffu, ok)) {
      umma::tmem_ld16(tq + 32 * half, *reinterpret_cast<float(*)[16]>(&S[0]));
      umma::tmem_ld16(tq + 32 * half + 16, *reinterpret_cast<float(*)[16]>(&S[16]));
      umma::tmem_ld_wait();
    }
    if (fetcher && ok && next < total) load(s.next[phase ^ 1]);
    // ---- A and P: rows times decays ------------------------------------------------------------------------------------------------------------------
    const float rq = p.use_l2norm ? rsqrtf(s.q2[0][i] + s.q2[1][i] + L2NORM_EPS) : 1.f;
    if (q4 == 2 + (i >> 5) && half == 0) s.rq[i] = rq;
    const float f = q4 < 2 ? s.beta[i] * s.rk[i] : p.scale * rq;
    if (half < (q4 & 1)) {      // 32 rows below 32 columns: the decay over the border between them is a factor of either side, both at most 1
      const float fr = i < len ? f * decay_between(s, i, 31) : 0.f;
#pragma unroll
      for (int e = 0; e < 32; e += 4) {
        const float4 d4 = *reinterpret_cast<const float4*>(&s.to32[e]), r4 = *reinterpret_cast<const float4*>(&s.rk[e]);
        S[e] = i < len ? S[e] * fr * (d4.x * r4.x) : 0.f;
        S[e + 1] = i < len ? S[e + 1] * fr * (d4.y * r4.y) : 0.f;
        S[e + 2] = i < len ? S[e + 2] * fr * (d4.z * r4.z) : 0.f;
        S[e + 3] = i < len ? S[e + 3] * fr * (d4.w * r4.w) : 0.f;
      }
    } else if (half == (q4 & 1)) {      // of a row's 32 columns the diagonal 16 take an exponential each; in front of them lie, in every other row, 16 below a border
      const bool low = lane >= 16;
      const float gh = s.ghi[i], gl = s.glo[i], fr = low && i < len ? f * decay_between(s, i, 32 * half + 15) : 0.f;
      const int last = i < len ? (q4 < 2 ? i - 1 : i) - (32 * half + (low ? 16 : 0)) : -1;      // columns beyond it are zero, whatever stands in the rows' products
#pragma unroll
      for (int e = 0; e < 16; e += 4) {
        const int j = 32 * half + e, jd = j + (low ? 16 : 0);
        const float4 d4 = *reinterpret_cast<const float4*>(&s.to16[j]), r4 = *reinterpret_cast<const float4*>(&s.rk[j]);
        const float4 h4 = *reinterpret_cast<const float4*>(&s.ghi[jd]), l4 = *reinterpret_cast<const float4*>(&s.glo[jd]), rd = *reinterpret_cast<const float4*>(&s.rk[jd]);
        const float dd[4] = {d4.x * r4.x, d4.y * r4.y, d4.z * r4.z, d4.w * r4.w}, hh[4] = {h4.x, h4.y, h4.z, h4.w}, ll[4] = {l4.x, l4.y, l4.z, l4.w},
                    rr[4] = {rd.x, rd.y, rd.z, rd.w};
#pragma unroll
        for (int j4 = 0; j4 < 4; ++j4) {
          const float x = e + j4 <= last ? (low ? S[16 + e + j4] : S[e + j4]) * (f * rr[j4]) * ex2((gh - hh[j4]) + (gl - ll[j4])) : 0.f;
          const float y = low && i < len ? S[e + j4] * fr * dd[j4] : 0.f;
          S[e + j4] = low ? y : x;
          S[16 + e + j4] = low ? x : 0.f;
        }
      }
    } else {      // this warp's columns lie above the diagonal block row
#pragma unroll
      for (int e = 0; e < 32; ++e) S[e] = 0.f;
    }
    {
      const int row = q4 < 2 ? i : 64 + i;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const Split x = split8(&S[8 * e]);
        *reinterpret_cast<uint4*>(piece(s.TPh, row, 4 * half + e)) = x.hi;
        *reinterpret_cast<uint4*>(piece(s.TPl, row, 4 * half + e)) = x.lo;
      }
      if (q4 < 2 && half == q4) {
        const int b = lane >> 4;      // the diagonal block of this row begins at column 16 b of its half
#pragma unroll
        for (int e = 0; e < 16; ++e) s.D[i >> 4][e][i & 15] = b ? S[16 + e] : S[e];
      }
    }
    umma::fence_before_sync();
    ok = __syncthreads_and(ok);
    if (!ok) break;
    // ---- Tm: diagonal blocks by substitution, a column per thread; meanwhile others write VEC ----------------------------------------------------------
    if (tid < 64) {
      const int b = tid >> 4, col = tid & 15;
      float x[16];      // column `col` of the inverse: a finished entry is taken out of all rows below it
#pragma unroll
      for (int r = 0; r < 16; ++r) x[r] = r == col ? 1.f : 0.f;
#pragma unroll
      for (int j = 0; j < 15; ++j) {
#pragma unroll
        for (int r4 = (j + 1) / 4; r4 < 4; ++r4) {
          const float4 a = *reinterpret_cast<const float4*>(&s.D[b][j][4 * r4]);
          if (4 * r4 > j) x[4 * r4] = fmaf(-a.x, x[j], x[4 * r4]);
          if (4 * r4 + 1 > j) x[4 * r4 + 1] = fmaf(-a.y, x[j], x[4 * r4 + 1]);
          if (4 * r4 + 2 > j) x[4 * r4 + 2] = fmaf(-a.z, x[j], x[4 * r4 + 2]);
          if (4 * r4 + 3 > j) x[4 * r4 + 3] = fmaf(-a.w, x[j], x[4 * r4 + 3]);
        }
      }
      const uint32_t at = column_at(s.TPh, 16 * b, 16 * b + col);
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        column_put(at, r, x[r]);
        column_put(at + 16384, r, x[r] - __bfloat162float(__float2bfloat16_rn(x[r])));
      }
      __syncwarp();
      // ---- merge of 16: each of the two warps has written both diagonal blocks of its pair; T21 takes A21's place -----------------------------------------
      const int r0 = 32 * warp;
      FragPair t2, a21, t1;
      frag_a(t2.h, s.TPh, r0 + 16, r0 + 16, lane);
      frag_a(t2.l, s.TPl, r0 + 16, r0 + 16, lane);
      frag_b(a21.h, s.TPh, r0 + 16, r0, lane);
      frag_b(a21.l, s.TPl, r0 + 16, r0, lane);
      frag_b(t1.h, s.TPh, r0, r0, lane);
      frag_b(t1.l, s.TPl, r0, r0, lane);
      float y[2][4] = {}, z[2][4] = {};
      mma_pair(y, t2, a21);
      mma_pair(z, as_a(y), t1);
      __syncwarp();
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        put2(s.TPh, s.TPl, r0 + 16 + (lane >> 2), r0 + 8 * n + 2 * (lane & 3), -z[n][0], -z[n][1]);
        put2(s.TPh, s.TPl, r0 + 24 + (lane >> 2), r0 + 8 * n + 2 * (lane & 3), -z[n][2], -z[n][3]);
      }
    } else if (tid >= 128 && tid < 192) {
      const int t = tid - 128;
      float* const v = reinterpret_cast<float*>(p.VEC + static_cast<size_t>(tile) * T_VEC);
      const float gh = s.ghi[t], gl = s.glo[t], lh = s.ghi[63], ll = s.glo[63], e = ex2(gh + gl), rk = s.rk[t], b = s.beta[t];
      const bool there = t < len;
      v[V_BETA + t] = b;
      v[V_KG + t] = there ? b * e * rk : 0.f;
      v[V_W + t] = there ? ex2((lh - gh) + (ll - gl)) * rk : 0.f;
      v[V_Q + t] = there ? p.scale * e * s.rq[t] : 0.f;
      v[V_GHI + t] = gh;
      v[V_GLO + t] = gl;
      v[V_RK + t] = there ? rk : 0.f;
      v[V_RQ + t] = there ? s.rq[t] : 0.f;
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
          frag_b(a21.h, s.TPh, 32 + 16 * m, 16 * n, lane);
          frag_b(a21.l, s.TPl, 32 + 16 * m, 16 * n, lane);
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
      asm volatile("bar.sync 2, 128;" ::: "memory");      // all four have read A21
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
    ok = mbar_wait(&s.done, 1);      // (everybody: the barrier's next phase is the next tile's first product)
    if (q4 >= 2) {
      umma::fence_after_sync();
      if (__all_sync(0xffffffffu, ok)) {
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
    if (!ok) break;
    if (tid == 0) {
      bulk_s2g(p.TP + static_cast<size_t>(tile) * T_TP, s.TPh, 16384);
      bulk_s2g(p.TP + static_cast<size_t>(tile) * T_TP + 16384, s.TPl, 16384);
      bulk_commit();
    }
  }
  if (!ok && tid == 0) {      // a wait gave up: loads and products may still be under way
    atomicOr(p.status, KDA_STATUS_PREP_LOAD_WAIT);
    mbar_drain(&s.full);
    mbar_drain(&s.done);
  }
  if (tid == 0) bulk_wait_read<0>();      // shared memory may go; the writes are complete with the kernel
  umma::fence_before_sync();
  __syncthreads();
  if (warp == 1) umma::tmem_dealloc(tb, 128);
}

int launch_prepare(const PrepParams& p, long long tiles, cudaStream_t st) {
  static DeviceOnce once;
  const int smem = static_cast<int>(sizeof(PrepSmem)) + 1024;
  const int rc = once.run([&] { return cudaFuncSetAttribute(delta_prepare_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem); });
  if (rc != KDA_OK) return rc;
  return static_cast<int>(launch_chained(delta_prepare_kernel, static_cast<unsigned>(std::min<long long>(tiles, 3LL * sm_count())), PT, smem, st, p));
}

}  // namespace delta
}  // namespace kda
