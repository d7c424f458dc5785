// Gated delta rule, one decay per token and head: the backward walk, from a sequence's last chunk to its first (see delta.cuh).
//
// The counterpart of delta_scan.cu: a CTA has VC value columns of one (sequence, head), the gradient of the state in fp32 registers (TMEM lane = key
// row).  Per chunk, three dependent products:
//   1   K dh'                     (M = 64, K = 128;  x = w K dh')
//   2   Tm^T x                    (M = 64, K = 64;   f = that + Pt^T dO)
//   3   K^T y                     (M = 128, K = 64;  y = -beta exp(G) f;  dh = exp(G_last) dh' + that + Q^T (scale exp(G) dO))
// Pt^T dO and Q^T (..) depend on dO alone and run beside the chain.  dh', x, y and the scaled dO are bf16 pairs, hi and lo side by side in one operand.
// With 64 columns f and dv leave by bulk copies, through operands that are done (dO's tile, the scaled dO's).
// Bound by the chain of a chunk: 2.7 us with 32 columns, 3.5 with 64.
#include "delta.cuh"

namespace kda {
namespace delta {

namespace {

constexpr int NW = 10, NT = NW * 32, W_ISSUE = 8;

template <int VC>
struct RSmem {
  unsigned char KQ[2][2][16384];
  unsigned char TP[2][16384];
  unsigned char dO[8192];                      // [64 t][64 v]
  unsigned char H[VC == 32 ? 1 : 2][16384];    // dh': [128 keys][hi, lo]
  unsigned char X[VC == 32 ? 1 : 2][8192];     // x, then y: [64 t][hi, lo]
  unsigned char Os[VC == 32 ? 1 : 2][8192];    // scale exp(G) dO: [64 t][hi, lo]
  float vec[2][VEC_COPY / 4];
  uint64_t fullA[2], freeA[2], fullB, freeB;
  uint64_t hReady, dReady, xReady, yReady, oReady, m1, m2, m3;
  uint32_t tmem_slot;
  volatile int dead;
};
static_assert(sizeof(RSmem<64>) + 1024 <= 227 * 1024, "RSmem too large");

}  // namespace

template <int VC>
__global__ void __launch_bounds__(NT, 1) delta_bwd_scan_kernel(const __grid_constant__ RScanParams p) {
  chain_point();
  using Smem = RSmem<VC>;
  constexpr int HC = VC / 2, QC = VC / 4;
  constexpr bool BULK = VC == 64;
  constexpr int D1 = 0, D2 = 2 * VC, D3 = 4 * VC, DO = 6 * VC;
  constexpr uint32_t TM = VC == 32 ? 256 : 512;
  extern __shared__ unsigned char smem_raw[];
  Smem& s = *reinterpret_cast<Smem*>(smem_raw + pad_to_1024(smem_raw));
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, q4 = warp & 3, half = (warp >> 2) & 1;
  const int slices = ((p.vc + 63) & ~63) / VC;
  const int unit = blockIdx.x / slices, v0 = (blockIdx.x % slices) * VC;
  const int seq = p.map.started(unit / p.H), h = unit % p.H;
  const int c0 = p.map.first_chunk(seq), nchunks = p.map.first_chunk(seq + 1) - c0;
  const long long tok_begin = p.map.first_token(seq), tok_end = p.map.first_token(seq + 1);

  if (tid == 0) {
    for (int b = 0; b < 2; ++b) {
      mbar_init(&s.fullA[b], 1);
      mbar_init(&s.freeA[b], 1);
    }
    mbar_init(&s.fullB, 1);
    mbar_init(&s.freeB, 1);
    mbar_init(&s.hReady, 8);
    mbar_init(&s.dReady, 8);
    mbar_init(&s.xReady, 8);
    mbar_init(&s.yReady, 8);
    mbar_init(&s.oReady, 8);
    mbar_init(&s.m1, 1);
    mbar_init(&s.m2, 1);
    mbar_init(&s.m3, 1);
    s.dead = 0;
    fence_mbar_init();
  }
  if (warp == 0) umma::tmem_alloc(&s.tmem_slot, TM);
  umma::fence_before_sync();
  __syncthreads();
  umma::fence_after_sync();
  const uint32_t tb = s.tmem_slot, tq = tb + (static_cast<uint32_t>(32 * q4) << 16);

  if (warp < 8) {
    // ================= the chain =================
    const int key = 32 * q4 + lane, col = HC * half;
    const int t = 16 * q4 + (lane & 15);                     // token: lanes 0..15 of a quadrant hold its rows of an accumulator with M = 64
    const bool has = lane < 16;
    const int dcol = QC * (2 * half + (lane >> 4));          // the columns of dO's row t that this thread scales
    const size_t sb = ((static_cast<size_t>(seq) * p.H + h) * p.kc + key) * p.vc + v0 + col;
    float S[HC];
#pragma unroll
    for (int e = 0; e < HC; e += 4) {
      const float4 f = p.d_ht && key < p.kc && v0 + col + e < p.vc ? *reinterpret_cast<const float4*>(p.d_ht + sb + e) : make_float4(0.f, 0.f, 0.f, 0.f);
      S[e] = f.x; S[e + 1] = f.y; S[e + 2] = f.z; S[e + 3] = f.w;
    }
    auto load = [&](int d, int e, float (&x)[16]) {
      float y[16];
      umma::tmem_ld16(tq + d + col + e, x);
      umma::tmem_ld16(tq + d + VC + col + e, y);
      umma::tmem_ld_wait();
#pragma unroll
      for (int j = 0; j < 16; ++j) x[j] += y[j];
    };
    bool ok = true;
    for (int i = 0; i < nchunks; ++i) {
      const int c = nchunks - 1 - i;
      const long long tok0 = tok_begin + static_cast<long long>(c) * C;
      const int len = tok_end - tok0 < C ? static_cast<int>(tok_end - tok0) : C;
      const size_t tile = static_cast<size_t>(c0 + c) * p.H + h;
      if (__any_sync(0xffffffffu, s.dead != 0)) { ok = false; break; }
#pragma unroll
      for (int e = 0; e < HC; e += 8) {
        const Split x = split8(&S[e]);
        put<VC>(s.H[0], 128, key, col + e, x);
        leave_state(p.DH + tile * T_STATE, key, v0 + col + e, x.hi);
      }
      if (!(ok = warp_wait(&s.fullA[i & 1], (i >> 1) & 1))) break;
      const float* const vec = s.vec[i & 1];
      const float vb = vec[V_BETA + t], vk = vec[V_KG + t], vw = vec[V_W + t], vq = vec[V_Q + t], last = vec[V_LAST];
      if (len < C) {
#pragma unroll
        for (int b = 0; b < 4; ++b) clear_rows(s.KQ[i & 1][b >> 1] + (b & 1) * 8192, len, tid, 256);
      }
      fence_proxy_async();
      warp_arrive(&s.hReady, lane);
      // ---- beside product 1: dO scaled ----
      if (!(ok = warp_wait(&s.fullB, i & 1))) break;
#pragma unroll
      for (int e = 0; e < QC; e += 8) {
        const int dc = (VC == 32 ? v0 & 63 : 0) + dcol + e;
        uint4* const at = reinterpret_cast<uint4*>(piece(s.dO, t, dc >> 3));
        if (t >= len) *at = make_uint4(0, 0, 0, 0);
        float x[8];
        unpack8(*at, x);
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] *= vq;
        put<VC>(s.Os[0], 64, t, dcol + e, split8(x));
      }
      fence_proxy_async();
      warp_arrive(&s.dReady, lane);
#pragma unroll
      for (int e = 0; e < HC; ++e) S[e] *= last;
      // ---- x ----
      if (!(ok = warp_wait(&s.m1, i & 1))) break;
      umma::fence_after_sync();
#pragma unroll
      for (int e = 0; e < HC; e += 16) {
        float x[16];
        load(D1, e, x);
#pragma unroll
        for (int j = 0; j < 16; ++j) x[j] *= vw;
        if (has) {
          put<VC>(s.X[0], 64, t, col + e, split8(&x[0]));
          put<VC>(s.X[0], 64, t, col + e + 8, split8(&x[8]));
        }
      }
      fence_proxy_async();
      warp_arrive(&s.xReady, lane);
      // ---- f: dv, the tile for the per-chunk gradients, y ----
      if (!(ok = warp_wait(&s.m2, i & 1))) break;
      umma::fence_after_sync();
      uint4 kf[HC / 8], kv[HC / 8];
#pragma unroll
      for (int e = 0; e < HC; e += 16) {
        float x[16], y[16];
        load(D2, e, x);
        umma::tmem_ld16(tq + DO + col + e, y);
        umma::tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          x[j] += y[j];
          y[j] = vb * x[j];
        }
        kf[e / 8] = pack8(&x[0]); kf[e / 8 + 1] = pack8(&x[8]);
        kv[e / 8] = pack8(&y[0]); kv[e / 8 + 1] = pack8(&y[8]);
#pragma unroll
        for (int j = 0; j < 16; ++j) x[j] *= -vk;
        if (has) {
          put<VC>(s.X[0], 64, t, col + e, split8(&x[0]));
          put<VC>(s.X[0], 64, t, col + e + 8, split8(&x[8]));
        }
      }
      fence_proxy_async();
      warp_arrive(&s.yReady, lane);
      if constexpr (BULK) {
        if (has) {
#pragma unroll
          for (int e = 0; e < HC / 8; ++e) {
            *reinterpret_cast<uint4*>(piece(s.dO, t, (col >> 3) + e)) = kf[e];
            if (len == C) *reinterpret_cast<uint4*>(piece(s.Os[0], t, (col >> 3) + e)) = kv[e];
          }
        }
        fence_proxy_async();
        warp_arrive(&s.oReady, lane);
      }
      if (has && (!BULK || len < C)) {
        __nv_bfloat16* const dv = p.dv + (static_cast<size_t>(tok0 + t) * p.H + h) * p.vc + v0 + col;
#pragma unroll
        for (int e = 0; e < HC / 8; ++e) {
          const int v = v0 + col + 8 * e;
          if constexpr (!BULK) *reinterpret_cast<uint4*>(piece(p.DF + tile * T_VN + (v >> 6) * 8192, t, (v & 63) >> 3)) = kf[e];
          if (t < len && v < p.vc) *reinterpret_cast<uint4*>(dv + 8 * e) = kv[e];
        }
      }
      if (!(ok = warp_wait(&s.m3, i & 1))) break;
      umma::fence_after_sync();
#pragma unroll
      for (int e = 0; e < HC; e += 16) {
        float x[16];
        load(D3, e, x);
#pragma unroll
        for (int j = 0; j < 16; ++j) S[e + j] += x[j];
      }
      umma::fence_before_sync();
    }
    if (!ok) {
      s.dead = 1;
      if (lane == 0) atomicOr(p.status, KDA_STATUS_BWD_SCAN_MMA_WAIT);
    } else if (p.dh0 && key < p.kc) {
#pragma unroll
      for (int e = 0; e < HC; e += 4)
        if (v0 + col + e < p.vc) *reinterpret_cast<float4*>(p.dh0 + sb + e) = make_float4(S[e], S[e + 1], S[e + 2], S[e + 3]);
    }
  } else if (warp == W_ISSUE) {
    if (lane == 0) {
      constexpr int N = 2 * VC;
      constexpr uint32_t id1 = umma::instr_desc(64, N, false, true), idT = umma::instr_desc(64, N, true, true), idTl = umma::instr_desc(64, VC, true, true),
                         id3 = umma::instr_desc(128, N, true, true);
      const uint32_t aT = smem_u32(s.TP[0]);
      const uint64_t dH = umma::desc_mnmajor(smem_u32(s.H[0]), 0, 16384), dX = umma::desc_mnmajor(smem_u32(s.X[0]), 0, 8192),
                     dOs = umma::desc_mnmajor(smem_u32(s.Os[0]), 0, 8192), dO = umma::desc_mnmajor(smem_u32(s.dO) + (VC == 32 ? (v0 & 63) * 2 : 0), 0, 8192);
      bool ok = true;
      for (int i = 0; i < nchunks && ok; ++i) {
        const uint32_t aK = smem_u32(s.KQ[i & 1][0]);
        if (s.dead || !mbar_wait(&s.fullA[i & 1], (i >> 1) & 1) || !mbar_wait(&s.hReady, i & 1)) { ok = false; break; }
        umma::fence_after_sync();
#pragma unroll
        for (int b = 0; b < 2; ++b)
          umma::mma4<umma::KSTEP_KMAJOR, umma::KSTEP_MNMAJOR>(tb + D1, umma::desc_kmajor(aK + 16384 * b, 0), dH + 4ull * b * umma::KSTEP_MNMAJOR, id1, b);
        umma::commit(&s.m1);
        if (!mbar_wait(&s.fullB, i & 1) || !mbar_wait(&s.dReady, i & 1)) { ok = false; break; }
        umma::fence_after_sync();
        umma::mma4<umma::KSTEP_MNMAJOR, umma::KSTEP_MNMAJOR>(tb + DO, umma::desc_mnmajor(aT + 8192, 0, 8192), dO, idTl, 0);
        umma::mma4<umma::KSTEP_MNMAJOR, umma::KSTEP_MNMAJOR>(tb + DO, umma::desc_mnmajor(aT + 16384 + 8192, 0, 8192), dO, idTl, 1);
        umma::mma4<umma::KSTEP_MNMAJOR, umma::KSTEP_MNMAJOR>(tb + D3, umma::desc_mnmajor(aK + 8192, 0, 16384), dOs, id3, 0);
        if (!mbar_wait(&s.xReady, i & 1)) { ok = false; break; }
        umma::fence_after_sync();
        umma::mma4<umma::KSTEP_MNMAJOR, umma::KSTEP_MNMAJOR>(tb + D2, umma::desc_mnmajor(aT, 0, 8192), dX, idT, 0);
        umma::mma4<umma::KSTEP_MNMAJOR, umma::KSTEP_MNMAJOR>(tb + D2, umma::desc_mnmajor(aT + 16384, 0, 8192), dX, idTl, 1);
        umma::commit(&s.m2);
        umma::commit(&s.freeB);
        if (!mbar_wait(&s.yReady, i & 1)) { ok = false; break; }
        umma::fence_after_sync();
        umma::mma4<umma::KSTEP_MNMAJOR, umma::KSTEP_MNMAJOR>(tb + D3, umma::desc_mnmajor(aK, 0, 16384), dX, id3, 1);
        umma::commit(&s.m3);
        umma::commit(&s.freeA[i & 1]);
      }
      if (!ok) {
        s.dead = 1;
        atomicOr(p.status, KDA_STATUS_BWD_SCAN_MMA_WAIT);
      }
    }
    __syncwarp();
  } else {
    if (lane == 0) {
      const int hq = h / p.grp;
      auto first = [&](int i) { return static_cast<int>(tok_begin + static_cast<long long>(nchunks - 1 - i) * C); };
      auto tile_of = [&](int i) { return static_cast<size_t>(c0 + nchunks - 1 - i) * p.H + h; };
      auto loadA = [&](int i) {
        const int b = i & 1, tok0 = first(i);
        mbar_expect_tx(&s.fullA[b], 4 * 8192 + VEC_COPY);
        for (int x = 0; x < 2; ++x) tma_load_rows(s.KQ[b][x], &p.tm_k, 64 * x, hq, tok0, &s.fullA[b]);
        for (int x = 0; x < 2; ++x) tma_load_rows(s.KQ[b][x] + 8192, &p.tm_q, 64 * x, hq, tok0, &s.fullA[b]);
        bulk_g2s(s.vec[b], p.VEC + tile_of(i) * T_VEC, VEC_COPY, &s.fullA[b]);
      };
      auto loadB = [&](int i) {
        mbar_expect_tx(&s.fullB, 2 * 16384 + 8192);
        tma_load_rows(s.dO, &p.tm_do, v0 & ~63, h, first(i), &s.fullB);
        bulk_g2s(s.TP[0], p.TP + tile_of(i) * T_TP, 32768, &s.fullB);
      };
      bool ok = true;
      if (nchunks > 0) {
        loadA(0);
        loadB(0);
        if (nchunks > 1) loadA(1);
      }
      for (int i = 0; i < nchunks; ++i) {
        if (i + 3 < nchunks) {     // into L2, ahead of the loads: from DRAM a stage takes longer than a chunk
          if (v0 == 0) {           // what the slices of a unit share
            for (int x = 0; x < 2 && 64 * x < p.kc; ++x) {
              tma_prefetch_rows(&p.tm_k, 64 * x, hq, first(i + 3));
              tma_prefetch_rows(&p.tm_q, 64 * x, hq, first(i + 3));
            }
            bulk_prefetch(p.TP + tile_of(i + 3) * T_TP, 32768);
          }
          if ((v0 & 63) == 0) tma_prefetch_rows(&p.tm_do, v0, h, first(i + 3));
        }
        if (s.dead) { ok = false; break; }
        if constexpr (BULK) {      // f stands in dO's tile, dv in the scaled dO's
          if (!mbar_wait(&s.oReady, i & 1)) { ok = false; break; }
          bulk_s2g(p.DF + tile_of(i) * T_VN + (v0 / 64) * 8192, s.dO, 8192);
          if (tok_end - first(i) >= C) tma_store_rows(&p.tm_dv, v0, h, first(i), s.Os[0]);
          bulk_commit();
          bulk_wait_read<0>();
        }
        if (i + 1 < nchunks) {
          if (!mbar_wait(&s.freeB, i & 1)) { ok = false; break; }
          loadB(i + 1);
        }
        if (i + 2 < nchunks) {
          if (!mbar_wait(&s.freeA[i & 1], (i >> 1) & 1)) { ok = false; break; }
          loadA(i + 2);
        }
      }
      if (!ok) {
        s.dead = 1;
        atomicOr(p.status, KDA_STATUS_BWD_SCAN_LOAD_WAIT);
      }
      if constexpr (BULK) bulk_wait_read<0>();      // the stores read shared memory that goes with the CTA
    }
    __syncwarp();
  }
  __syncthreads();
  if (tid == 0 && s.dead) {      // somebody gave up: loads and products may still be under way
    uint64_t* const all[] = {&s.fullA[0], &s.fullA[1], &s.fullB, &s.m1, &s.m2, &s.m3};
    for (uint64_t* b : all) mbar_drain(b);
  }
  umma::fence_before_sync();
  __syncthreads();
  if (warp == 0) umma::tmem_dealloc(tb, TM);
}

template <int VC>
static int launch_vc(const RScanParams& p, int units, cudaStream_t st) {
  static DeviceOnce once;
  const int smem = static_cast<int>(sizeof(RSmem<VC>)) + 1024;
  const int rc = once.run([&] { return cudaFuncSetAttribute(delta_bwd_scan_kernel<VC>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem); });
  if (rc != KDA_OK) return rc;
  return static_cast<int>(launch_chained(delta_bwd_scan_kernel<VC>, static_cast<unsigned>(units) * (((p.vc + 63) & ~63) / VC), NT, smem, st, p));
}

int launch_bwd_scan(const RScanParams& p, int units, int slices, cudaStream_t st) {
  // (32 chunks each, us with 1 | 2 | 4 CTAs per unit: 37 units 120 | 112 | 85, 48 120 | 112 | 161, 74 121 | 114 | 165, 96 122 | 219 | 241)
  if (slices == 0) slices = 4 * units <= sm_count() ? 4 : 2 * units <= sm_count() ? 2 : 1;
  return slices == 4 ? launch_vc<32>(p, units, st) : slices == 2 ? launch_vc<64>(p, units, st) : launch_bwd_scan_t(p, units, st);
}

}  // namespace delta
}  // namespace kda
