// Gated delta rule, one decay per token and head: the forward walk over a sequence's chunks (see delta.cuh).
//
// A CTA walks the chunks of one (sequence, head) with VC = 32 or 64 of the value columns, for calls that have fewer units than SMs (delta_scan_t.cu: all
// columns); the recurrence is independent per column.  The state is fp32 in registers (TMEM lane = key row, a thread holds half of a row's columns).  Per
// chunk, three dependent products:
//   1   [K; Q] h             (M = 128: the keys' rows and the queries' in one, K = 128)
//   2   [Tm; Pt] r           (r = beta V - beta exp(G) K h; gives v_new and the chunk's own part of o, K = 64)
//   3   K^T (w v_new)        (added to the state that the registers decay, K = 64)
// h, r and w v_new are bf16 pairs, hi and lo side by side in one operand, so that a product reads A once for both and the epilogue adds the two
// accumulators: the products are bound by reading operands from shared memory, and A is the larger one.
// The warps meet through mbarriers only; warp 8 issues the products, warp 9 the loads.
// With 64 columns v_new and o leave by bulk copies, through operands that are done (v's tile, q's rows).
// Bound by the chain of a chunk: 1 x 32,768 tokens x 32 heads 1,046 us, 2.0 a chunk with 32 columns (3.9 k cycles, of them 1.2 k products), 3.0 with 64.
#include "delta.cuh"

namespace kda {
namespace delta {

namespace {

constexpr int NW = 10, NT = NW * 32, W_ISSUE = 8;

template <int VC>
struct ScanSmem {
  static constexpr int SPANS = VC / 32;                      // 128-byte-wide spans of an operand of VC columns, hi and lo together
  unsigned char KQ[2][2][16384];                             // two stages of [128 rows: k, then q][64 key columns] x 2
  unsigned char TP[2][16384];                                // hi, lo
  unsigned char V[8192];                   // [64 t][64 v]
  unsigned char H[SPANS][16384];                             // [128 keys][64 columns]: hi, then lo (VC = 32: 32 of each in one span)
  unsigned char R[SPANS][8192];                              // [64 t][..] the same of r, then of w v_new
  float vec[2][VEC_COPY / 4];
  uint64_t fullA[2], freeA[2], fullB, freeB;                 // k, q, VEC; TP, v
  uint64_t hReady, rReady, uReady, oReady, m1, m2, m3;
  uint32_t tmem_slot;
  volatile int dead;
};
static_assert(sizeof(ScanSmem<64>) + 1024 <= 227 * 1024, "ScanSmem too large");

}  // namespace

template <int VC, bool TRAIN>
__global__ void __launch_bounds__(NT, 1) delta_scan_kernel(const __grid_constant__ ScanParams p) {
  chain_point();
  using Smem = ScanSmem<VC>;
  constexpr bool BULK = VC == 64;      // tiles and full chunks of o leave by bulk copies
  constexpr int HC = VC / 2, DW = 2 * VC;
  constexpr int D1 = 0, D2 = DW, D3 = 2 * DW;
  constexpr uint32_t TM = 3 * DW <= 256 ? 256 : 512;
  extern __shared__ unsigned char smem_raw[];
  Smem& s = *reinterpret_cast<Smem*>(smem_raw + pad_to_1024(smem_raw));
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, q4 = warp & 3, half = (warp >> 2) & 1;
  const int slices = ((p.vc + 63) & ~63) / VC;               // narrow heads: whole spans of 64 columns, as the tiles have them
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
    mbar_init(&s.rReady, 4);
    mbar_init(&s.uReady, 4);
    mbar_init(&s.oReady, BULK ? 5 : 4);      // (one is the loading warp's: see warp_wait)
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
    // ================= the chain: state, r, v_new, o =================
    const int key = 32 * q4 + lane, col = HC * half;         // state row and first column (of the slice) of this thread
    const int t = 32 * (q4 & 1) + lane;                      // its token: of k's rows (q4 < 2) or of q's
    const bool krow = q4 < 2;
    const size_t sb = ((static_cast<size_t>(seq) * p.H + h) * p.kc + key) * p.vc + v0 + col;
    float S[HC];
#pragma unroll
    for (int e = 0; e < HC; e += 4) {
      const float4 f = p.h0 && key < p.kc && v0 + col + e < p.vc ? *reinterpret_cast<const float4*>(p.h0 + sb + e) : make_float4(0.f, 0.f, 0.f, 0.f);
      S[e] = f.x; S[e + 1] = f.y; S[e + 2] = f.z; S[e + 3] = f.w;
    }
    auto load = [&](int d, int e, float (&x)[16]) {      // hi's and lo's sums
      float y[16];
      umma::tmem_ld16(tq + d + col + e, x);
      umma::tmem_ld16(tq + d + VC + col + e, y);
      umma::tmem_ld_wait();
#pragma unroll
      for (int j = 0; j < 16; ++j) x[j] += y[j];
    };
    bool ok = true;
    for (int i = 0; i < nchunks; ++i) {
      const long long tok0 = tok_begin + static_cast<long long>(i) * C;
      const int len = tok_end - tok0 < C ? static_cast<int>(tok_end - tok0) : C;
      const size_t tile = static_cast<size_t>(c0 + i) * p.H + h;
      if (__any_sync(0xffffffffu, s.dead != 0)) { ok = false; break; }
      // ---- the state as an operand ----
#pragma unroll
      for (int e = 0; e < HC; e += 8) {
        const Split x = split8(&S[e]);
        put<VC>(s.H[0], 128, key, col + e, x);
        if constexpr (TRAIN) leave_state(p.HS + tile * T_STATE, key, v0 + col + e, x.hi);
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
#pragma unroll
      for (int e = 0; e < HC; ++e) S[e] *= last;
      if (krow) {
        if (!(ok = warp_wait(&s.fullB, i & 1))) break;
        if (!(ok = warp_wait(&s.m1, i & 1))) break;
        umma::fence_after_sync();
#pragma unroll
        for (int e = 0; e < HC; e += 16) {
          float x[16], v[16];
          load(D1, e, x);
          const int c = ((VC == 32 ? v0 & 63 : 0) + col + e) >> 3;
          unpack8(*reinterpret_cast<const uint4*>(piece(s.V, t, c)), &v[0]);
          unpack8(*reinterpret_cast<const uint4*>(piece(s.V, t, c + 1)), &v[8]);
#pragma unroll
          for (int j = 0; j < 16; ++j) x[j] = t < len ? fmaf(vb, v[j], -vk * x[j]) : 0.f;
          put<VC>(s.R[0], 64, t, col + e, split8(&x[0]));
          put<VC>(s.R[0], 64, t, col + e + 8, split8(&x[8]));
        }
        fence_proxy_async();
        warp_arrive(&s.rReady, lane);
        if (!(ok = warp_wait(&s.m2, i & 1))) break;
        umma::fence_after_sync();
        uint4 keep[TRAIN && !BULK ? HC / 8 : 1];
#pragma unroll
        for (int e = 0; e < HC; e += 16) {
          float x[16];
          load(D2, e, x);
          if constexpr (TRAIN) {
            const uint4 a = pack8(&x[0]), b = pack8(&x[8]);
            if constexpr (BULK) {      // into v's tile: the same places
              *reinterpret_cast<uint4*>(piece(s.V, t, (col + e) >> 3)) = a;
              *reinterpret_cast<uint4*>(piece(s.V, t, ((col + e) >> 3) + 1)) = b;
            } else {
              keep[e / 8] = a;
              keep[e / 8 + 1] = b;
            }
          }
#pragma unroll
          for (int j = 0; j < 16; ++j) x[j] *= vw;
          put<VC>(s.R[0], 64, t, col + e, split8(&x[0]));
          put<VC>(s.R[0], 64, t, col + e + 8, split8(&x[8]));
        }
        fence_proxy_async();
        warp_arrive(&s.uReady, lane);
        if constexpr (TRAIN && !BULK) {
#pragma unroll
          for (int e = 0; e < HC / 8; ++e) {
            const int v = v0 + col + 8 * e;
            *reinterpret_cast<uint4*>(piece(p.VN + tile * T_VN + (v >> 6) * 8192, t, (v & 63) >> 3)) = keep[e];
          }
        }
      } else {
        if (!(ok = warp_wait(&s.m1, i & 1))) break;
        if (!(ok = warp_wait(&s.m2, i & 1))) break;
        umma::fence_after_sync();
        __nv_bfloat16* const o = p.o + (static_cast<size_t>(tok0 + t) * p.H + h) * p.vc + v0 + col;
#pragma unroll
        for (int e = 0; e < HC; e += 16) {
          float x[16], y[16];
          load(D1, e, x);
          load(D2, e, y);
#pragma unroll
          for (int j = 0; j < 16; ++j) y[j] = fmaf(vq, x[j], y[j]);
          if (BULK && len == C) {      // into q's rows, which product 1 has read
            *reinterpret_cast<uint4*>(piece(s.KQ[i & 1][0] + 8192, t, (col + e) >> 3)) = pack8(&y[0]);
            *reinterpret_cast<uint4*>(piece(s.KQ[i & 1][0] + 8192, t, ((col + e) >> 3) + 1)) = pack8(&y[8]);
            continue;
          }
          if (t < len && v0 + col + e < p.vc) *reinterpret_cast<uint4*>(o + e) = pack8(&y[0]);
          if (t < len && v0 + col + e + 8 < p.vc) *reinterpret_cast<uint4*>(o + e + 8) = pack8(&y[8]);
        }
        if constexpr (BULK) {
          fence_proxy_async();
          warp_arrive(&s.oReady, lane);
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
      if (lane == 0) atomicOr(p.status, KDA_STATUS_SCAN_MMA_WAIT);
    } else if (p.ht && key < p.kc) {
#pragma unroll
      for (int e = 0; e < HC; e += 4)
        if (v0 + col + e < p.vc) *reinterpret_cast<float4*>(p.ht + sb + e) = make_float4(S[e], S[e + 1], S[e + 2], S[e + 3]);
    }
  } else if (warp == W_ISSUE) {
    if (lane == 0) {
      // N of a product with hi and lo side by side (or of one of them), and with hi alone
      constexpr int N = 2 * VC;
      constexpr uint32_t id1 = umma::instr_desc(128, N, false, true), id2l = umma::instr_desc(128, VC, false, true), id3 = umma::instr_desc(128, N, true, true);
      constexpr uint32_t HS_ = 16384, RS_ = 8192;            // strides of the spans
      const uint32_t aH = smem_u32(s.H[0]), aR = smem_u32(s.R[0]), aT = smem_u32(s.TP[0]);
      bool ok = true;
      for (int i = 0; i < nchunks && ok; ++i) {
        const uint32_t aK = smem_u32(s.KQ[i & 1][0]);
        if (s.dead || !mbar_wait(&s.fullA[i & 1], (i >> 1) & 1) || !mbar_wait(&s.hReady, i & 1)) { ok = false; break; }
        umma::fence_after_sync();
#pragma unroll
        for (int b = 0; b < 2; ++b)
          umma::mma4<umma::KSTEP_KMAJOR, umma::KSTEP_MNMAJOR>(tb + D1, umma::desc_kmajor(aK + 16384 * b, 0), umma::desc_mnmajor(aH, 4 * b, HS_), id1, b);
        umma::commit(&s.m1);
        if (!mbar_wait(&s.fullB, i & 1) || !mbar_wait(&s.rReady, i & 1)) { ok = false; break; }
        umma::fence_after_sync();
        umma::mma4<umma::KSTEP_KMAJOR, umma::KSTEP_MNMAJOR>(tb + D2, umma::desc_kmajor(aT, 0), umma::desc_mnmajor(aR, 0, RS_), id1, 0);
        umma::mma4<umma::KSTEP_KMAJOR, umma::KSTEP_MNMAJOR>(tb + D2, umma::desc_kmajor(aT + 16384, 0), umma::desc_mnmajor(aR, 0, RS_), id2l, 1);
        umma::commit(&s.m2);
        umma::commit(&s.freeB);
        if (!mbar_wait(&s.uReady, i & 1)) { ok = false; break; }
        umma::fence_after_sync();
        umma::mma4<umma::KSTEP_MNMAJOR, umma::KSTEP_MNMAJOR>(tb + D3, umma::desc_mnmajor(aK, 0, 16384), umma::desc_mnmajor(aR, 0, RS_), id3, 0);
        umma::commit(&s.m3);
        umma::commit(&s.freeA[i & 1]);
      }
      if (!ok) {
        s.dead = 1;
        atomicOr(p.status, KDA_STATUS_SCAN_MMA_WAIT);
      }
    }
    __syncwarp();
  } else {
    if (lane == 0) {
      const int hq = h / p.grp;
      auto loadA = [&](int i) {
        const int b = i & 1, tok0 = static_cast<int>(tok_begin + static_cast<long long>(i) * C);
        mbar_expect_tx(&s.fullA[b], 4 * 8192 + VEC_COPY);
        for (int x = 0; x < 2; ++x) tma_load_rows(s.KQ[b][x], &p.tm_k, 64 * x, hq, tok0, &s.fullA[b]);
        for (int x = 0; x < 2; ++x) tma_load_rows(s.KQ[b][x] + 8192, &p.tm_q, 64 * x, hq, tok0, &s.fullA[b]);
        bulk_g2s(s.vec[b], p.VEC + (static_cast<size_t>(c0 + i) * p.H + h) * T_VEC, VEC_COPY, &s.fullA[b]);
      };
      auto loadB = [&](int i) {
        const int tok0 = static_cast<int>(tok_begin + static_cast<long long>(i) * C);
        mbar_expect_tx(&s.fullB, 2 * 16384 + 8192);
        tma_load_rows(s.V, &p.tm_v, v0 & ~63, h, tok0, &s.fullB);
        bulk_g2s(s.TP[0], p.TP + (static_cast<size_t>(c0 + i) * p.H + h) * T_TP, 32768, &s.fullB);
      };
      bool ok = true;
      if constexpr (BULK) mbar_arrive(&s.oReady);
      if (nchunks > 0) {
        loadA(0);
        loadB(0);
        if (nchunks > 1) loadA(1);
      }
      for (int i = 0; i < nchunks; ++i) {
        if (i + 3 < nchunks) {                // into L2, ahead of the loads: from DRAM a stage takes longer than a chunk
          const int tok0 = static_cast<int>(tok_begin + static_cast<long long>(i + 3) * C);
          if (v0 == 0) {                      // what the slices of a unit share
            for (int x = 0; x < 2 && 64 * x < p.kc; ++x) {
              tma_prefetch_rows(&p.tm_k, 64 * x, hq, tok0);
              tma_prefetch_rows(&p.tm_q, 64 * x, hq, tok0);
            }
            bulk_prefetch(p.TP + (static_cast<size_t>(c0 + i + 3) * p.H + h) * T_TP, 32768);
          }
          if ((v0 & 63) == 0) tma_prefetch_rows(&p.tm_v, v0, h, tok0);
        }
        if (s.dead) { ok = false; break; }
        if constexpr (TRAIN && BULK) {      // v_new stands in v's tile
          if (!mbar_wait(&s.uReady, i & 1)) { ok = false; break; }
          bulk_s2g(p.VN + (static_cast<size_t>(c0 + i) * p.H + h) * T_VN + (v0 / 64) * 8192, s.V, 8192);
          bulk_commit();
          bulk_wait_read<0>();
        }
        if (i + 1 < nchunks) {
          if (!mbar_wait(&s.freeB, i & 1)) { ok = false; break; }
          loadB(i + 1);
        }
        if constexpr (BULK) {               // o in q's rows
          if (!mbar_wait(&s.oReady, i & 1)) { ok = false; break; }
          mbar_arrive(&s.oReady);
          const long long tok0 = tok_begin + static_cast<long long>(i) * C;
          if (tok_end - tok0 >= C) {
            tma_store_rows(&p.tm_o, v0, h, static_cast<int>(tok0), s.KQ[i & 1][0] + 8192);
            bulk_commit();
            bulk_wait_read<0>();
          }
        }
        if (i + 2 < nchunks) {
          if (!mbar_wait(&s.freeA[i & 1], (i >> 1) & 1)) { ok = false; break; }
          loadA(i + 2);
        }
      }
      if (!ok) {
        s.dead = 1;
        atomicOr(p.status, KDA_STATUS_SCAN_LOAD_WAIT);
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

template <int VC, bool TRAIN>
static int launch_vc(const ScanParams& p, int units, cudaStream_t st) {
  static DeviceOnce once;
  const int smem = static_cast<int>(sizeof(ScanSmem<VC>)) + 1024;
  const int rc = once.run([&] { return cudaFuncSetAttribute(delta_scan_kernel<VC, TRAIN>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem); });
  if (rc != KDA_OK) return rc;
  return static_cast<int>(launch_chained(delta_scan_kernel<VC, TRAIN>, static_cast<unsigned>(units) * (((p.vc + 63) & ~63) / VC), NT, smem, st, p));
}

// Few (sequence, head) units leave SMs idle: their value columns are spread over two or four CTAs, which shortens a chunk's products.
int launch_scan(const ScanParams& p, int units, int slices, cudaStream_t st) {
  // (32 chunks each, us with 1 | 2 | 4 CTAs per unit: 37 units 112 | 96 | 73, 48 113 | 97 | 137, 74 113 | 98 | 140, 96 114 | 181 | 205)
  if (slices == 0) slices = 4 * units <= sm_count() ? 4 : 2 * units <= sm_count() ? 2 : 1;
  const bool train = p.HS != nullptr;
  if (slices == 4) return train ? launch_vc<32, true>(p, units, st) : launch_vc<32, false>(p, units, st);
  if (slices == 2) return train ? launch_vc<64, true>(p, units, st) : launch_vc<64, false>(p, units, st);
  return launch_scan_t(p, units, st);
}

}  // namespace delta
}  // namespace kda
