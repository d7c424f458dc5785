// Gated delta rule, one decay per token and head: the backward walk with a CTA per (sequence, head) (delta_bwd_scan.cu: several).
//
// The transposed form of delta_scan_t.cu: TMEM lane = value column, the operands that the walk produces are A and stay in tensor memory.  Per chunk:
//   1   dh'^T K^T                   (128 v x 64 tokens, K = 128 keys;  x = w K dh')
//   2   x^T Tm + dO^T Pt            (128 v x 64 tokens, K = 64;  f)
//   3   y^T K + (scale exp(G) dO)^T Q   (128 v x 128 keys, K = 64;  y = -beta exp(G) f), added to the gradient that the registers hold and decay
// The terms with dO do not depend on the chain and run behind product 1.  x (then y) takes the columns that its own thread has just read product 1 from.
// f leaves through dO's tile, dv through a tile of its own.  8 x 4,096 tokens x 32 heads 473 us (two rounds of units), 3.7 a chunk.
#include "delta.cuh"

namespace kda {
namespace delta {

namespace {

constexpr int CW = 16, NT = CREW_THREADS, W_ISSUE = CW;

struct RTSmem {
  unsigned char KQ[2][2][16384];        // two stages, of dO and of what leaves as dv too
  unsigned char dO[2][2][8192];         // [64 t][64 v] x 2
  unsigned char dV[2][2][8192];
  unsigned char TP[2][16384];
  unsigned char H[2][16384];            // dh' as it leaves: [128 v][64 keys] x 2
  alignas(16) float vec[2][VEC_COPY / 4];
  uint64_t fullA[2], freeA[2], fullB, freeB;
  uint64_t hReady, dReady, xReady, yReady, oReady, m1, m2, m3;
  uint32_t tmem_slot;
  volatile int dead;
};
static_assert(sizeof(RTSmem) + 1024 <= 227 * 1024, "RTSmem too large");

// TMEM columns: dh' hi, lo; product 1, then x or y (16 columns per group of tokens: eight hi, eight lo); scaled dO hi, lo; dO; products 2 and 3
constexpr int AH = 0, AL = 64, D1 = 128, OH = 192, OL = 224, DO = 256, D2 = 288, D3 = 352;

}  // namespace

__global__ void __launch_bounds__(NT, 1) delta_bwd_scan_t_kernel(const __grid_constant__ RScanParams p) {
  chain_point();
  extern __shared__ unsigned char smem_raw[];
  RTSmem& s = *reinterpret_cast<RTSmem*>(smem_raw + pad_to_1024(smem_raw));
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, q4 = warp & 3;
  const int seq = p.map.started(blockIdx.x / p.H), h = blockIdx.x % p.H;
  const int c0 = p.map.first_chunk(seq), nchunks = p.map.first_chunk(seq + 1) - c0;
  const long long tok_begin = p.map.first_token(seq), tok_end = p.map.first_token(seq + 1);

  if (tid == 0) {
    for (int b = 0; b < 2; ++b) {
      mbar_init(&s.fullA[b], 1);
      mbar_init(&s.freeA[b], 1);
    }
    mbar_init(&s.fullB, 1);
    mbar_init(&s.freeB, 1);
    mbar_init(&s.hReady, CW);
    mbar_init(&s.dReady, CW);
    mbar_init(&s.xReady, CW);
    mbar_init(&s.yReady, CW);
    mbar_init(&s.oReady, CW + 1);      // (one is the loading warp's: see warp_wait)
    mbar_init(&s.m1, 1);
    mbar_init(&s.m2, 1);
    mbar_init(&s.m3, 1);
    s.dead = 0;
    fence_mbar_init();
  }
  if (warp == 0) umma::tmem_alloc(&s.tmem_slot, 512);
  umma::fence_before_sync();
  __syncthreads();
  umma::fence_after_sync();
  const uint32_t tb = s.tmem_slot, tq = tb + (static_cast<uint32_t>(32 * q4) << 16);

  if (warp < CW) {
    compute_registers();
    // ================= the chain =================
    const int v = 32 * q4 + lane, g = warp >> 2, k0 = 32 * g, t0 = 16 * g;      // value column; first key and first token of this thread
    const size_t sb = (static_cast<size_t>(seq) * p.H + h) * p.kc * p.vc + v;
    float S[32];
#pragma unroll
    for (int e = 0; e < 32; ++e) S[e] = p.d_ht && k0 + e < p.kc && v < p.vc ? p.d_ht[sb + static_cast<size_t>(k0 + e) * p.vc] : 0.f;
    bool ok = true;
    for (int i = 0; i < nchunks; ++i) {
      const long long tok0 = tok_begin + static_cast<long long>(nchunks - 1 - i) * C;
      const int len = tok_end - tok0 < C ? static_cast<int>(tok_end - tok0) : C;
      if (__any_sync(0xffffffffu, s.dead != 0)) { ok = false; break; }
#pragma unroll
      for (int e = 0; e < 32; e += 16) {
        const Split a = split8(&S[e]), b = split8(&S[e + 8]);
        umma::tmem_st8(tq + AH + (k0 + e) / 2, a.hi, b.hi);
        umma::tmem_st8(tq + AL + (k0 + e) / 2, a.lo, b.lo);
        *reinterpret_cast<uint4*>(piece(s.H[g >> 1], v, 4 * (g & 1) + e / 8)) = a.hi;
        *reinterpret_cast<uint4*>(piece(s.H[g >> 1], v, 4 * (g & 1) + e / 8 + 1)) = b.hi;
      }
      umma::tmem_st_wait();
      if (!(ok = warp_wait(&s.fullA[i & 1], (i >> 1) & 1))) break;
      const float* const vec = s.vec[i & 1];
      if (len < C) {
#pragma unroll
        for (int b = 0; b < 4; ++b) clear_rows(s.KQ[i & 1][b >> 1] + (b & 1) * 8192, len, tid, CW * 32);
      }
      fence_proxy_async();
      warp_arrive(&s.hReady, lane);
      const float last = vec[V_LAST];
      // ---- beside product 1: dO and scaled dO as operands ----
      const uint32_t at_o = column_at(s.dO[i & 1][v >> 6], t0, v & 63), at_v = column_at(s.dV[i & 1][v >> 6], t0, v & 63);
      {
        float d[16], q[16];
        uint32_t w[8];
        row16(vec + V_Q + t0, q);
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const uint32_t x = t0 + j < len ? column_get(at_o, j) : 0u;
          w[j / 2] = j & 1 ? w[j / 2] | x << 16 : x;
          d[j] = __uint_as_float(x << 16) * q[j];
        }
        umma::tmem_st8(tq + DO + t0 / 2, make_uint4(w[0], w[1], w[2], w[3]), make_uint4(w[4], w[5], w[6], w[7]));
        const Split a = split8(&d[0]), b = split8(&d[8]);
        umma::tmem_st8(tq + OH + t0 / 2, a.hi, b.hi);
        umma::tmem_st8(tq + OL + t0 / 2, a.lo, b.lo);
        umma::tmem_st_wait();
      }
      warp_arrive(&s.dReady, lane);
      // ---- x ----
      float f[16], w[16];
      row16(vec + V_W + t0, w);
      if (!(ok = warp_wait(&s.m1, i & 1))) break;
      umma::fence_after_sync();
      umma::tmem_ld16(tq + D1 + t0, f);
      umma::tmem_ld_wait();
      {
#pragma unroll
        for (int j = 0; j < 16; ++j) f[j] *= w[j];
        const Split a = split8(&f[0]), b = split8(&f[8]);
        umma::tmem_st8(tq + D1 + t0, a.hi, b.hi);
        umma::tmem_st8(tq + D1 + t0 + 8, a.lo, b.lo);
        umma::tmem_st_wait();
      }
      warp_arrive(&s.xReady, lane);
      row16(vec + V_KG + t0, w);
      // ---- f, y ----
      if (!(ok = warp_wait(&s.m2, i & 1))) break;
      umma::fence_after_sync();
      umma::tmem_ld16(tq + D2 + t0, f);
      umma::tmem_ld_wait();
      {
#pragma unroll
        for (int j = 0; j < 16; ++j) w[j] *= -f[j];
        const Split a = split8(&w[0]), b = split8(&w[8]);
        umma::tmem_st8(tq + D1 + t0, a.hi, b.hi);
        umma::tmem_st8(tq + D1 + t0 + 8, a.lo, b.lo);
        umma::tmem_st_wait();
      }
      warp_arrive(&s.yReady, lane);
      row16(vec + V_BETA + t0, w);
#pragma unroll
      for (int j = 0; j < 16; ++j) column_put(at_o, j, f[j]);
      if (len == C) {
#pragma unroll
        for (int j = 0; j < 16; ++j) column_put(at_v, j, w[j] * f[j]);
      } else if (v < p.vc) {
#pragma unroll
        for (int j = 0; j < 16; ++j)
          if (t0 + j < len) p.dv[(static_cast<size_t>(tok0 + t0 + j) * p.H + h) * p.vc + v] = __float2bfloat16_rn(w[j] * f[j]);
      }
      fence_proxy_async();
      warp_arrive(&s.oReady, lane);
      // ---- the gradient of the state ----
      if (!(ok = warp_wait(&s.m3, i & 1))) break;
      umma::fence_after_sync();
#pragma unroll
      for (int e = 0; e < 32; e += 16) {
        umma::tmem_ld16(tq + D3 + k0 + e, f);
        umma::tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < 16; ++j) S[e + j] = fmaf(S[e + j], last, f[j]);
      }
      umma::fence_before_sync();
    }
    if (!ok) {
      s.dead = 1;
      if (lane == 0) atomicOr(p.status, KDA_STATUS_BWD_SCAN_MMA_WAIT);
    } else if (p.dh0 && v < p.vc) {
#pragma unroll
      for (int e = 0; e < 32; ++e)
        if (k0 + e < p.kc) p.dh0[sb + static_cast<size_t>(k0 + e) * p.vc] = S[e];
    }
  } else {
    helper_registers();
    if (warp == W_ISSUE) {
      if (lane == 0) {
        constexpr uint32_t id1 = umma::instr_desc(128, 64, false, false), id2 = umma::instr_desc(128, 64, false, true), id3 = umma::instr_desc(128, 128, false, true);
        const uint32_t aT = smem_u32(s.TP[0]);
        const uint64_t dT = umma::desc_mnmajor(aT, 0, 8192), dP = umma::desc_mnmajor(aT + 8192, 0, 8192);      // their low parts: 16 KiB behind
        bool ok = true;
        for (int i = 0; i < nchunks && ok; ++i) {
          const uint32_t aK = smem_u32(s.KQ[i & 1][0]);
          const uint64_t dK = umma::desc_kmajor(aK, 0), dKm = umma::desc_mnmajor(aK, 0, 16384), dQm = umma::desc_mnmajor(aK + 8192, 0, 16384);
          if (s.dead || !mbar_wait(&s.fullA[i & 1], (i >> 1) & 1) || !mbar_wait(&s.hReady, i & 1)) { ok = false; break; }
          umma::fence_after_sync();
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const uint64_t b = dK + (k >> 2) * 1024u + (k & 3) * umma::KSTEP_KMAJOR;
            umma::mma_ts(tb + D1, tb + AH + 8 * k, b, id1, k > 0);
            umma::mma_ts(tb + D1, tb + AL + 8 * k, b, id1, 1);
          }
          umma::commit(&s.m1);
          bulk_s2g(p.DH + (static_cast<size_t>(c0 + nchunks - 1 - i) * p.H + h) * T_STATE, s.H[0], 16384);
          bulk_s2g(p.DH + (static_cast<size_t>(c0 + nchunks - 1 - i) * p.H + h) * T_STATE + 16384, s.H[1], 16384);
          bulk_commit();
          if (!mbar_wait(&s.fullB, i & 1) || !mbar_wait(&s.dReady, i & 1)) { ok = false; break; }
          umma::fence_after_sync();
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            umma::mma_ts(tb + D2, tb + DO + 8 * k, dP + k * umma::KSTEP_MNMAJOR, id2, k > 0);
            umma::mma_ts(tb + D2, tb + DO + 8 * k, dP + 1024u + k * umma::KSTEP_MNMAJOR, id2, 1);
          }
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            umma::mma_ts(tb + D3, tb + OH + 8 * k, dQm + k * umma::KSTEP_MNMAJOR, id3, k > 0);
            umma::mma_ts(tb + D3, tb + OL + 8 * k, dQm + k * umma::KSTEP_MNMAJOR, id3, 1);
          }
          if (!mbar_wait(&s.xReady, i & 1)) { ok = false; break; }
          umma::fence_after_sync();
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const uint64_t b = dT + k * umma::KSTEP_MNMAJOR;
            umma::mma_ts(tb + D2, tb + D1 + 16 * k, b, id2, 1);
            umma::mma_ts(tb + D2, tb + D1 + 16 * k + 8, b, id2, 1);
            umma::mma_ts(tb + D2, tb + D1 + 16 * k, b + 1024u, id2, 1);
          }
          umma::commit(&s.m2);
          umma::commit(&s.freeB);
          if (!mbar_wait(&s.yReady, i & 1)) { ok = false; break; }
          umma::fence_after_sync();
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            umma::mma_ts(tb + D3, tb + D1 + 16 * k, dKm + k * umma::KSTEP_MNMAJOR, id3, 1);
            umma::mma_ts(tb + D3, tb + D1 + 16 * k + 8, dKm + k * umma::KSTEP_MNMAJOR, id3, 1);
          }
          bulk_wait_read<0>();      // m3 also says that dh's tile may be overwritten
          umma::commit(&s.m3);
          umma::commit(&s.freeA[i & 1]);
        }
        if (!ok) {
          s.dead = 1;
          atomicOr(p.status, KDA_STATUS_BWD_SCAN_MMA_WAIT);
        }
        bulk_wait_read<0>();
      }
      __syncwarp();
    } else if (warp == W_ISSUE + 1) {
      if (lane == 0) {
        const int hq = h / p.grp;
        auto first = [&](int i) { return static_cast<int>(tok_begin + static_cast<long long>(nchunks - 1 - i) * C); };
        auto tile_of = [&](int i) { return static_cast<size_t>(c0 + nchunks - 1 - i) * p.H + h; };
        auto loadA = [&](int i) {
          const int b = i & 1, tok0 = first(i);
          mbar_expect_tx(&s.fullA[b], 6 * 8192 + VEC_COPY);
          for (int x = 0; x < 2; ++x) tma_load_rows(s.KQ[b][x], &p.tm_k, 64 * x, hq, tok0, &s.fullA[b]);
          for (int x = 0; x < 2; ++x) tma_load_rows(s.KQ[b][x] + 8192, &p.tm_q, 64 * x, hq, tok0, &s.fullA[b]);
          for (int x = 0; x < 2; ++x) tma_load_rows(s.dO[b][x], &p.tm_do, 64 * x, h, tok0, &s.fullA[b]);
          bulk_g2s(s.vec[b], p.VEC + tile_of(i) * T_VEC, VEC_COPY, &s.fullA[b]);
        };
        auto loadB = [&](int i) {
          mbar_expect_tx(&s.fullB, 2 * 16384);
          bulk_g2s(s.TP[0], p.TP + tile_of(i) * T_TP, 32768, &s.fullB);
        };
        bool ok = true;
        mbar_arrive(&s.oReady);
        if (nchunks > 0) {
          loadA(0);
          loadB(0);
          if (nchunks > 1) loadA(1);
        }
        for (int i = 0; i < nchunks; ++i) {
          if (i + 2 < nchunks) bulk_prefetch(p.TP + tile_of(i + 2) * T_TP, 32768);      // into L2
          if (i + 1 < nchunks) {
            if (s.dead || !mbar_wait(&s.freeB, i & 1)) { ok = false; break; }
            loadB(i + 1);
          }
          if (s.dead || !mbar_wait(&s.oReady, i & 1)) { ok = false; break; }
          mbar_arrive(&s.oReady);
#pragma unroll
          for (int x = 0; x < 2; ++x) bulk_s2g(p.DF + tile_of(i) * T_VN + x * 8192, s.dO[i & 1][x], 8192);
          if (tok_end - first(i) >= C) {
            for (int x = 0; x < 2 && 64 * x < p.vc; ++x) tma_store_rows(&p.tm_dv, 64 * x, h, first(i), s.dV[i & 1][x]);
          }
          bulk_commit();
          if (i + 2 < nchunks) {
            if (!mbar_wait(&s.freeA[i & 1], (i >> 1) & 1)) { ok = false; break; }
            bulk_wait_read<0>();
            loadA(i + 2);
          }
        }
        if (!ok) {
          s.dead = 1;
          atomicOr(p.status, KDA_STATUS_BWD_SCAN_LOAD_WAIT);
        }
        bulk_wait_read<0>();      // the stores read shared memory that goes with the CTA
      }
      __syncwarp();
    }
  }
  __syncthreads();
  if (tid == 0 && s.dead) {      // somebody gave up: loads and products may still be under way
    uint64_t* const all[] = {&s.fullA[0], &s.fullA[1], &s.fullB, &s.m1, &s.m2, &s.m3};
    for (uint64_t* b : all) mbar_drain(b);
  }
  umma::fence_before_sync();
  __syncthreads();
  if (warp == 0) umma::tmem_dealloc(tb, 512);
}

int launch_bwd_scan_t(const RScanParams& p, int units, cudaStream_t st) {
  static DeviceOnce once;
  const int smem = static_cast<int>(sizeof(RTSmem)) + 1024;
  const int rc = once.run([&] { return crew_ready(delta_bwd_scan_t_kernel, smem); });
  if (rc != KDA_OK) return rc;
  return static_cast<int>(launch_chained(delta_bwd_scan_t_kernel, static_cast<unsigned>(units), NT, smem, st, p));
}

}  // namespace delta
}  // namespace kda
