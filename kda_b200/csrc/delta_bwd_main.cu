// Gated delta rule, one decay per token and head: the gradients of a chunk (see delta.cuh), from the state in front of it (HS), the gradient of the
// state behind it (DH), v_new (VN) and f (DF).
//
// A persistent CTA per SM, a tile per (chunk, head).  Stacked operands, rows 0..63 the keys' and 64..127 the queries':
//   S  = [K; Q] K^T              G2 = [f; dO] VN^T            (128 x 64 x 128)
//   Y  = [f; dO] HS^T            Z  = VN DH^T                 (128 x 128 x 128; Z: the upper half counts)
//   E  = rows 0..63 -beta D G2 (j < i), rows 64..127 scale D G2 (j <= i), with the reciprocal norms of both rows; bf16
//   D4 = E K                     D5 = E^T [K; Q]              (D5: the upper half counts)
// so that a thread with a key's row has all of dk's terms in its TMEM lane, and one with a query's row all of dq's.  dG comes from the rows' products
// with k and q, dbeta from f v, k Y and the sums of a row's dA D <k, k>.  The next tile's HS, DH, VN, f, dO, v are fetched once their products are done, its k and q
// a tile ahead; dk and dq of a full chunk leave by TMA from k's and q's rows, which they overwrite.  16,384 tiles of 128 columns 641 us, 176 KB each: 0.69 of the copy
// rate; the rest is conversions between TMEM, registers and shared memory around the products.
#include <algorithm>

#include "delta.cuh"

namespace kda {
namespace delta {

namespace {

// sixteen warps (TMEM lane quadrant = warp & 3, column group = warp >> 2), one that issues the products, and one that has the loads, the stores and dg
// (with loads and stores the issuing warp came late for the second products: 707 instead of 807 us without its stores)
constexpr int CW = 16, NT = (CW + 2) * 32, W_ISSUE = CW;

struct MainSmem {
  unsigned char E[16384];              // [128][64]; as D5's A its second span is what follows, whose rows of the result nobody reads
  unsigned char KQ[2][2][16384];
  unsigned char FD[2][16384];          // [128 rows: f, dO][64 v] x 2
  unsigned char VN[2][8192];           // (Z's lower half reads beyond: the next span, then v)
  unsigned char V[2][8192];
  unsigned char HS[2][16384], DH[2][16384];
  float vec[2][V_LAST + 4];
  struct Sums {                        // of a tile, partial: of the four column groups
    float k[4][3][C], q[4][C];         // k rows: k (row terms), k (column terms), dbeta; q rows: q dq
    float z[8], h[CW];
  } sums[2];
  uint64_t fullA[2], fullB, ready, eReady, used, done, mS, mY, mD;
  uint32_t tmem_slot;
  volatile int dead;
};
static_assert(sizeof(MainSmem) + 1024 <= 227 * 1024, "MainSmem too large");
constexpr int T_S = 0, T_G2 = 64, T_D4 = 0, T_Y = 128, T_Z = 256, T_D5 = 384;      // TMEM columns: D4 takes the place of S and G2

__device__ __forceinline__ void store_any(void* p, size_t i, int dtype, float x) {
  if (dtype == KDA_BF16) static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(x);
  else static_cast<float*>(p)[i] = x;
}

}  // namespace

__global__ void __launch_bounds__(NT, 1) delta_bwd_main_kernel(const __grid_constant__ MainParams p, int spans) {
  chain_point();
  extern __shared__ unsigned char smem_raw[];
  MainSmem& s = *reinterpret_cast<MainSmem*>(smem_raw + pad_to_1024(smem_raw));
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, q4 = warp & 3, g = warp >> 2;
  const int total = p.map.total() * p.H;      // (below 2^31: checked by the entry points)
  if (tid == 0) {
    mbar_init(&s.fullA[0], 1);
    mbar_init(&s.fullA[1], 1);
    mbar_init(&s.fullB, 1);
    mbar_init(&s.ready, CW + 1);      // (one is the loading warp's, of done too: see warp_wait)
    mbar_init(&s.eReady, CW);
    mbar_init(&s.used, CW);
    mbar_init(&s.done, CW + 1);
    mbar_init(&s.mS, 1);
    mbar_init(&s.mY, 1);
    mbar_init(&s.mD, 1);
    s.dead = 0;
    fence_mbar_init();
  }
  if (warp == 0) umma::tmem_alloc(&s.tmem_slot, 512);
  umma::fence_before_sync();
  __syncthreads();
  umma::fence_after_sync();
  const uint32_t tb = s.tmem_slot, tq = tb + (static_cast<uint32_t>(32 * q4) << 16);

  if (warp < CW) {
    const int t = 32 * (q4 & 1) + lane;      // this thread's token, of k's rows or of q's
    const bool krow = q4 < 2;
    bool ok = true;
    int n = 0;
    for (int tile = blockIdx.x; tile < total; tile += gridDim.x, ++n) {
      const ChunkInfo ci = p.map.info(tile / p.H);
      const int h = tile % p.H;
      if (__any_sync(0xffffffffu, s.dead != 0)) { ok = false; break; }
      if (!(ok = warp_wait(&s.fullA[n & 1], (n >> 1) & 1) && warp_wait(&s.fullB, n & 1))) break;
      if (ci.len < C) {
        for (int b = 0; b < 4; ++b) clear_rows(s.KQ[n & 1][b >> 1] + (b & 1) * 8192, ci.len, tid, CW * 32);
        for (int b = 0; b < 2; ++b) clear_rows(s.FD[b] + 8192, ci.len, tid, CW * 32);
        fence_proxy_async();
      }
      warp_arrive(&s.ready, lane);
      const float* const vec = s.vec[n & 1];
      MainSmem::Sums& sums = s.sums[n & 1];
      const float vk = vec[V_KG + t], vw = vec[V_W + t], vq = vec[V_Q + t], rk = vec[V_RK + t], rq = vec[V_RQ + t];
      const float gh = vec[V_GHI + t], gl = vec[V_GLO + t];
      // ---- what needs only the tiles: f v (32 of the columns), <h, dh'> ----
      float fv = 0.f;
      if (krow && (g >> 1) < spans && t < ci.len) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float x[8], y[8];
          unpack8(*reinterpret_cast<const uint4*>(piece(s.FD[g >> 1], t, 4 * (g & 1) + e)), x);
          unpack8(*reinterpret_cast<const uint4*>(piece(s.V[g >> 1], t, 4 * (g & 1) + e)), y);
#pragma unroll
          for (int j = 0; j < 8; ++j) fv = fmaf(x[j], y[j], fv);
        }
      }
      float hd = 0.f;
#pragma unroll
      for (int b = 0; b < 2; ++b)
        for (int e = 0; e < spans; ++e) {      // (the same places of both tiles: their order does not matter)
          float x[8], y[8];
          unpack8(*reinterpret_cast<const uint4*>(s.HS[b] + (tid + CW * 32 * e) * 16), x);
          unpack8(*reinterpret_cast<const uint4*>(s.DH[b] + (tid + CW * 32 * e) * 16), y);
#pragma unroll
          for (int j = 0; j < 8; ++j) hd = fmaf(x[j], y[j], hd);
        }
      hd = warp_sum(hd);
      if (lane == 0) sums.h[warp] = hd;
      __syncwarp();
      if (lane == 0) mbar_arrive(&s.used);
      // ---- E: 16 columns ----
      if (!(ok = warp_wait(&s.mS, n & 1))) break;
      umma::fence_after_sync();
      float bsum = 0.f, e16[16];
      if (g >= 2 && (q4 & 1) == 0) {      // above the diagonal
#pragma unroll
        for (int e = 0; e < 16; ++e) e16[e] = 0.f;
      } else {
        umma::tmem_ld16(tq + T_G2 + 16 * g, e16);
        umma::tmem_ld_wait();
        const int last = (t < ci.len ? (krow ? t - 1 : t) : -1) - 16 * g;
        const float f = krow ? -rk : p.scale * rq;
#pragma unroll
        for (int e = 0; e < 16; e += 4) {
          const int j = 16 * g + e;
          const float4 h4 = *reinterpret_cast<const float4*>(vec + V_GHI + j), l4 = *reinterpret_cast<const float4*>(vec + V_GLO + j),
                       r4 = *reinterpret_cast<const float4*>(vec + V_RK + j);
          e16[e] = e <= last ? e16[e] * (f * r4.x) * ex2((gh - h4.x) + (gl - l4.x)) : 0.f;
          e16[e + 1] = e + 1 <= last ? e16[e + 1] * (f * r4.y) * ex2((gh - h4.y) + (gl - l4.y)) : 0.f;
          e16[e + 2] = e + 2 <= last ? e16[e + 2] * (f * r4.z) * ex2((gh - h4.z) + (gl - l4.z)) : 0.f;
          e16[e + 3] = e + 3 <= last ? e16[e + 3] * (f * r4.w) * ex2((gh - h4.w) + (gl - l4.w)) : 0.f;
        }
        if (krow) {
          float x[16];
          umma::tmem_ld16(tq + T_S + 16 * g, x);
          umma::tmem_ld_wait();
          const float vb = vec[V_BETA + t];
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            bsum = e <= last ? fmaf(e16[e], x[e], bsum) : bsum;
            e16[e] *= vb;
          }
        }
      }
      *reinterpret_cast<uint4*>(piece(s.E, 64 * (krow ? 0 : 1) + t, 2 * g)) = pack8(&e16[0]);
      *reinterpret_cast<uint4*>(piece(s.E, 64 * (krow ? 0 : 1) + t, 2 * g + 1)) = pack8(&e16[8]);
      fence_proxy_async();
      warp_arrive(&s.eReady, lane);
      // ---- the rows: 32 columns ----
      unsigned char* const row = s.KQ[n & 1][g >> 1] + (krow ? 0 : 8192);
      const int pc = 4 * (g & 1);
      float x[32], da = 0.f, db = 0.f, dy = 0.f, dz = 0.f;
      if (!(ok = warp_wait(&s.mY, n & 1))) break;
      umma::fence_after_sync();
#pragma unroll
      for (int e = 0; e < 32; e += 16) {      // what the first products give
        float a[16], in[16];
        unpack8(*reinterpret_cast<const uint4*>(piece(row, t, pc + (e >> 3))), &in[0]);
        unpack8(*reinterpret_cast<const uint4*>(piece(row, t, pc + (e >> 3) + 1)), &in[8]);
        umma::tmem_ld16(tq + T_Y + 32 * g + e, a);
        umma::tmem_ld_wait();
        const float f = krow ? -vk : vq;
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          dy = fmaf(in[j], a[j], dy);
          x[e + j] = f * a[j];
        }
        if (krow) {
          umma::tmem_ld16(tq + T_Z + 32 * g + e, a);
          umma::tmem_ld_wait();
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            dz = fmaf(in[j], a[j], dz);
            x[e + j] = fmaf(vw, a[j], x[e + j]);
          }
        }
      }
      if (!(ok = warp_wait(&s.mD, n & 1))) break;
      umma::fence_after_sync();
#pragma unroll
      for (int e = 0; e < 32; e += 16) {
        float a[16], in[16];
        unpack8(*reinterpret_cast<const uint4*>(piece(row, t, pc + (e >> 3))), &in[0]);
        unpack8(*reinterpret_cast<const uint4*>(piece(row, t, pc + (e >> 3) + 1)), &in[8]);
        umma::tmem_ld16(tq + T_D4 + 32 * g + e, a);
        umma::tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          da = fmaf(in[j], a[j], da);
          x[e + j] += a[j];
        }
        if (krow) {
          umma::tmem_ld16(tq + T_D5 + 32 * g + e, a);
          umma::tmem_ld_wait();
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            db = fmaf(in[j], a[j], db);
            x[e + j] += a[j];
          }
        }
      }
      if (krow) {
        sums.k[g][0][t] = fmaf(-vk, dy, da);
        sums.k[g][1][t] = fmaf(vw, dz, db);
        sums.k[g][2][t] = fv + bsum - ex2(gh + gl) * rk * dy;
        const float z = warp_sum(t < ci.len ? vw * dz : 0.f);
        if (lane == 0) sums.z[2 * g + q4] = z;
      } else {
        sums.q[g][t] = fmaf(vq, dy, da);
      }
      warp_arrive(&s.done, lane);
      if (p.use_l2norm) {      // through the normalisation: what lies along the row itself falls out
        if (!(ok = warp_wait(&s.done, n & 1))) break;
        float d = 0.f;
#pragma unroll
        for (int e = 0; e < 4; ++e) d += krow ? sums.k[e][0][t] + sums.k[e][1][t] : sums.q[e][t];
        d *= krow ? rk * rk : rq * rq;
#pragma unroll
        for (int e = 0; e < 32; e += 8) {
          float in[8];
          unpack8(*reinterpret_cast<const uint4*>(piece(row, t, pc + (e >> 3))), in);
#pragma unroll
          for (int j = 0; j < 8; ++j) x[e + j] = fmaf(-d, in[j], x[e + j]);
        }
      }
      if (ci.len == C) {
#pragma unroll
        for (int e = 0; e < 32; e += 8) *reinterpret_cast<uint4*>(piece(row, t, pc + (e >> 3))) = pack8(&x[e]);
        fence_proxy_async();
      } else if (t < ci.len) {
        __nv_bfloat16* const out = (krow ? p.dk : p.dq) + (static_cast<size_t>(ci.tok0 + t) * p.H + h) * p.kc;
#pragma unroll
        for (int e = 0; e < 32; e += 8)
          if (32 * g + e < p.kc) *reinterpret_cast<uint4*>(out + 32 * g + e) = pack8(&x[e]);
      }
      umma::fence_before_sync();
    }
    if (ok) warp_arrive(&s.ready, lane);                  // the last tile's rows stand in shared memory
    if (!ok) {
      s.dead = 1;
      if (lane == 0) atomicOr(p.status, KDA_STATUS_BWD_MAIN_MMA_WAIT);
    }
  } else if (warp == W_ISSUE) {
    if (lane == 0) {
      constexpr uint32_t idS = umma::instr_desc(128, 64, false, false),
                         id4 = umma::instr_desc(128, 128, false, true) /* Y and Z too: the states' rows are value columns */, id5 = umma::instr_desc(128, 128, true, true);
      const uint32_t aE = smem_u32(s.E);
      bool ok = true;
      int n = 0;
      for (int tile = blockIdx.x; tile < total; tile += gridDim.x, ++n) {
        const uint32_t aK = smem_u32(s.KQ[n & 1][0]);
        if (s.dead || !mbar_wait(&s.fullA[n & 1], (n >> 1) & 1) || !mbar_wait(&s.fullB, n & 1) || !mbar_wait(&s.ready, n & 1)) { ok = false; break; }
        umma::fence_after_sync();
#pragma unroll 1
        for (int b = 0; b < spans; ++b)
          umma::mma4<umma::KSTEP_KMAJOR, umma::KSTEP_KMAJOR>(tb + T_G2, umma::desc_kmajor(smem_u32(s.FD[b]), 0), umma::desc_kmajor(smem_u32(s.VN[b]), 0), idS, b);
#pragma unroll 1
        for (int b = 0; b < 2; ++b) {
          const uint64_t d = umma::desc_kmajor(aK + 16384 * b, 0);
          umma::mma4<umma::KSTEP_KMAJOR, umma::KSTEP_KMAJOR>(tb + T_S, d, d, idS, b);
        }
        umma::commit(&s.mS);
#pragma unroll 1
        for (int b = 0; b < spans; ++b) {
          umma::mma4<umma::KSTEP_KMAJOR, umma::KSTEP_MNMAJOR>(tb + T_Y, umma::desc_kmajor(smem_u32(s.FD[b]), 0), umma::desc_mnmajor(smem_u32(s.HS[0]), 4 * b, 16384), id4, b);
          umma::mma4<umma::KSTEP_KMAJOR, umma::KSTEP_MNMAJOR>(tb + T_Z, umma::desc_kmajor(smem_u32(s.VN[b]), 0), umma::desc_mnmajor(smem_u32(s.DH[0]), 4 * b, 16384), id4, b);
        }
        umma::commit(&s.mY);
        if (!mbar_wait(&s.eReady, n & 1)) { ok = false; break; }
        umma::fence_after_sync();
        umma::mma4<umma::KSTEP_KMAJOR, umma::KSTEP_MNMAJOR>(tb + T_D4, umma::desc_kmajor(aE, 0), umma::desc_mnmajor(aK, 0, 16384), id4, 0);
#pragma unroll 1
        for (int b = 0; b < 2; ++b)      // E's rows 0..63 with K's, 64..127 with Q's: one run of 128 rows in both
          umma::mma4<umma::KSTEP_MNMAJOR, umma::KSTEP_MNMAJOR>(tb + T_D5, umma::desc_mnmajor(aE, 4 * b, 16384), umma::desc_mnmajor(aK, 4 * b, 16384), id5, b);
        umma::commit(&s.mD);
      }
      if (!ok) {
        s.dead = 1;
        atomicOr(p.status, KDA_STATUS_BWD_MAIN_MMA_WAIT);
      }
    }
    __syncwarp();
  } else {
    // ================= loads, stores, dg and dbeta =================
    auto loadA = [&](int tile, int n) {
      const ChunkInfo ci = p.map.info(tile / p.H);
      const int h = tile % p.H, hq = h / p.grp, tok0 = static_cast<int>(ci.tok0), b = n & 1;
      mbar_expect_tx(&s.fullA[b], 4 * 8192 + VEC_COPY);
      for (int x = 0; x < 2; ++x) tma_load_rows(s.KQ[b][x], &p.tm_k, 64 * x, hq, tok0, &s.fullA[b]);
      for (int x = 0; x < 2; ++x) tma_load_rows(s.KQ[b][x] + 8192, &p.tm_q, 64 * x, hq, tok0, &s.fullA[b]);
      bulk_g2s(s.vec[b], p.VEC + static_cast<size_t>(tile) * T_VEC, VEC_COPY, &s.fullA[b]);
    };
    auto loadB = [&](int tile) {
      const ChunkInfo ci = p.map.info(tile / p.H);
      const int h = tile % p.H, tok0 = static_cast<int>(ci.tok0);
      const size_t at = static_cast<size_t>(tile);
      mbar_expect_tx(&s.fullB, spans * (4 * 8192 + 2 * 16384));
      for (int x = 0; x < spans; ++x) {
        bulk_g2s(s.FD[x], p.DF + at * T_VN + x * 8192, 8192, &s.fullB);
        bulk_g2s(s.VN[x], p.VN + at * T_VN + x * 8192, 8192, &s.fullB);
        tma_load_rows(s.FD[x] + 8192, &p.tm_do, 64 * x, h, tok0, &s.fullB);
        tma_load_rows(s.V[x], &p.tm_v, 64 * x, h, tok0, &s.fullB);
      }
      for (int x = 0; x < 2; ++x) {      // spans of 64 keys: the rows of the value columns that there are
        bulk_g2s(s.HS[x], p.HS + at * T_STATE + x * 16384, spans * 8192, &s.fullB);
        bulk_g2s(s.DH[x], p.DH + at * T_STATE + x * 16384, spans * 8192, &s.fullB);
      }
    };
    auto store = [&](int tile, int n) {      // dk, dq of a full chunk
      const ChunkInfo ci = p.map.info(tile / p.H);
      if (ci.len < C) return;
      const int h = tile % p.H, tok0 = static_cast<int>(ci.tok0);
      for (int x = 0; x < 2 && 64 * x < p.kc; ++x) {
        tma_store_rows(&p.tm_dk, 64 * x, h, tok0, s.KQ[n & 1][x]);
        tma_store_rows(&p.tm_dq, 64 * x, h, tok0, s.KQ[n & 1][x] + 8192);
      }
      bulk_commit();
    };
    bool ok = true;
    int n = 0;
    if (lane == 0 && static_cast<int>(blockIdx.x) < total) {
      mbar_arrive(&s.ready);
      mbar_arrive(&s.done);
      loadA(blockIdx.x, 0);
      loadB(blockIdx.x);
    }
    for (int tile = blockIdx.x; tile < total; tile += gridDim.x, ++n) {
      const int next = tile + gridDim.x;
      if (__any_sync(0xffffffffu, s.dead != 0)) { ok = false; break; }
      if (!(ok = warp_wait(&s.ready, n & 1))) break;      // everybody is past the tile before
      if (lane == 0) {
        mbar_arrive(&s.ready);
        if (n > 0) store(tile - gridDim.x, n - 1);
        if (next < total) {
          bulk_wait_read<0>();
          loadA(next, n + 1);
        }
      }
      if (next < total) {
        if (!(ok = warp_wait(&s.mY, n & 1) && warp_wait(&s.used, n & 1))) break;
        if (lane == 0) loadB(next);
      }
      if (!(ok = warp_wait(&s.done, n & 1))) break;
      if (lane == 0) mbar_arrive(&s.done);
      {      // dg: the sum of dG from a token to the chunk's end, two tokens a lane (these sums are written again behind the load of the tile after the next)
        const ChunkInfo ci = p.map.info(tile / p.H);
        const int h = tile % p.H;
        const float* const vec = s.vec[n & 1];
        const MainSmem::Sums& sums = s.sums[n & 1];
        float tail = lane < CW ? sums.h[lane] * vec[V_LAST] : 0.f;
        if (lane < 8) tail += sums.z[lane];
        tail = warp_sum(tail);
        float d[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int r = 2 * lane + j;
          d[j] = 0.f;
#pragma unroll
          for (int e = 0; e < 4; ++e) d[j] += sums.q[e][r] + sums.k[e][0][r] - sums.k[e][1][r];
          if (r >= ci.len) d[j] = 0.f;
        }
        float sum = d[0] + d[1];
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
          const float y = __shfl_down_sync(0xffffffffu, sum, off);
          if (lane + off < 32) sum += y;
        }
        // sum: over this lane's two tokens and all behind them
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int r = 2 * lane + j;
          if (r < ci.len) {
            const size_t at = static_cast<size_t>(ci.tok0 + r) * p.H + h;
            store_any(p.dg, at, p.g_dtype, (j ? sum - d[0] : sum) + tail);
            store_any(p.dbeta, at, p.beta_dtype, sums.k[0][2][r] + sums.k[1][2][r] + sums.k[2][2][r] + sums.k[3][2][r]);
          }
        }
      }
    }
    if (ok && n > 0) {
      ok = warp_wait(&s.ready, n & 1);
      if (ok && lane == 0) store(blockIdx.x + (n - 1) * gridDim.x, n - 1);
    }
    if (!ok) {
      s.dead = 1;
      if (lane == 0) atomicOr(p.status, KDA_STATUS_BWD_MAIN_LOAD_WAIT);
    }
    if (lane == 0) bulk_wait_read<0>();      // the stores read shared memory that goes with the CTA
    __syncwarp();
  }
  __syncthreads();
  if (tid == 0 && s.dead) {      // somebody gave up: loads and products may still be under way
    uint64_t* const all[] = {&s.fullA[0], &s.fullA[1], &s.fullB, &s.mS, &s.mY, &s.mD};
    for (uint64_t* b : all) mbar_drain(b);
  }
  umma::fence_before_sync();
  __syncthreads();
  if (warp == 0) umma::tmem_dealloc(tb, 512);
}

int launch_bwd_main(const MainParams& p, long long tiles, int spans, cudaStream_t st) {
  static DeviceOnce once;
  const int smem = static_cast<int>(sizeof(MainSmem)) + 1024;
  const int rc = once.run([&] { return cudaFuncSetAttribute(delta_bwd_main_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem); });
  if (rc != KDA_OK) return rc;
  const unsigned grid = static_cast<unsigned>(std::min<long long>(tiles, sm_count()));
  return static_cast<int>(launch_chained(delta_bwd_main_kernel, grid, NT, smem, st, p, spans));
}

}  // namespace delta
}  // namespace kda
