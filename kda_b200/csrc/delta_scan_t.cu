// Gated delta rule, one decay per token and head: the forward walk with a CTA per (sequence, head) (delta_scan.cu: several).
//
// The transposed form: TMEM lane = value column v, so that every operand the walk produces is the A of its products and stays in tensor memory, and shared
// memory holds nothing but the tiles as they arrive, each a B operand.  Per chunk, three dependent products, A in bf16 pairs:
//   1   h^T [K; Q]^T              (128 v x 128 rows, K = 128 keys)
//   2   r^T [Tm; Pt]^T            (128 v x 128 rows, K = 64 tokens;  r = beta V - beta exp(G) K h)
//   3   (w v_new)^T K             (128 v x 128 keys, K = 64 tokens), added to the state that the registers hold and decay
// A thread has one value column, 32 keys of its state and 16 tokens of a chunk.  v, o and v_new are turned on the way through shared memory, two bytes a
// lane: o in q's rows once product 1 has read them, v_new (for a backward) in v's tile.  Tiles and full chunks of o leave by bulk copies.
// Bound by the chain of a chunk, 3.5 us: the products' 2.3 k cycles and three hand-overs each way.  8 x 4,096 tokens x 32 heads with what a backward needs 465 us
// (two rounds of units; the bytes alone 365), with 96 registers for every thread 504.
#include "delta.cuh"

namespace kda {
namespace delta {

namespace {

constexpr int CW = 16, NT = CREW_THREADS, W_ISSUE = CW;

template <bool TRAIN>
struct TSmem {
  unsigned char KQ[2][2][16384];             // two stages of [128 rows: k, then q][64 key columns] x 2
  unsigned char V[2][2][8192];               // and of [64 t][64 v] x 2
  unsigned char TP[2][16384];                // hi, lo
  unsigned char H[TRAIN ? 2 : 1][TRAIN ? 16384 : 16];      // h as it leaves: [128 v][64 keys] x 2
  alignas(16) float vec[2][VEC_COPY / 4];
  uint64_t fullA[2], freeA[2], fullB, freeB;
  uint64_t hReady, rReady, uReady, oReady, m1, m2, m3;
  uint32_t tmem_slot;
  volatile int dead;
};
static_assert(sizeof(TSmem<true>) + 1024 <= 227 * 1024, "TSmem too large");

// TMEM columns: h hi, lo; r (then w v_new) hi, lo; the three products (3 takes the place of 1)
constexpr int AH = 0, AL = 64, RH = 128, RL = 160, D1 = 192, D2 = 320, D3 = D1;

}  // namespace

template <bool TRAIN>
__global__ void __launch_bounds__(NT, 1) delta_scan_t_kernel(const __grid_constant__ ScanParams p) {
  chain_point();
  extern __shared__ unsigned char smem_raw[];
  TSmem<TRAIN>& s = *reinterpret_cast<TSmem<TRAIN>*>(smem_raw + pad_to_1024(smem_raw));
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
    mbar_init(&s.rReady, CW);
    mbar_init(&s.uReady, CW);
    mbar_init(&s.oReady, CW);
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
    for (int e = 0; e < 32; ++e) S[e] = p.h0 && k0 + e < p.kc && v < p.vc ? p.h0[sb + static_cast<size_t>(k0 + e) * p.vc] : 0.f;
    bool ok = true;
    for (int i = 0; i < nchunks; ++i) {
      const long long tok0 = tok_begin + static_cast<long long>(i) * C;
      const int len = tok_end - tok0 < C ? static_cast<int>(tok_end - tok0) : C;
      if (__any_sync(0xffffffffu, s.dead != 0)) { ok = false; break; }
      // ---- the state as an operand ----
#pragma unroll
      for (int e = 0; e < 32; e += 16) {
        const Split a = split8(&S[e]), b = split8(&S[e + 8]);
        umma::tmem_st8(tq + AH + (k0 + e) / 2, a.hi, b.hi);
        umma::tmem_st8(tq + AL + (k0 + e) / 2, a.lo, b.lo);
        if constexpr (TRAIN) {
          *reinterpret_cast<uint4*>(piece(s.H[g >> 1], v, 4 * (g & 1) + e / 8)) = a.hi;
          *reinterpret_cast<uint4*>(piece(s.H[g >> 1], v, 4 * (g & 1) + e / 8 + 1)) = b.hi;
        }
      }
      umma::tmem_st_wait();
      if (!(ok = warp_wait(&s.fullA[i & 1], (i >> 1) & 1))) break;
      const float* const vec = s.vec[i & 1];
      if (len < C) {
#pragma unroll
        for (int b = 0; b < 4; ++b) clear_rows(s.KQ[i & 1][b >> 1] + (b & 1) * 8192, len, tid, CW * 32);
      }
      if (TRAIN || len < C) fence_proxy_async();
      warp_arrive(&s.hReady, lane);
      const float last = vec[V_LAST];
      // ---- r ----
      const uint32_t at_v = column_at(s.V[i & 1][v >> 6], t0, v & 63), at_o = column_at(s.KQ[i & 1][v >> 6] + 8192, t0, v & 63);
      float r[16], y[16], w[16];
      row16(vec + V_BETA + t0, w);
#pragma unroll
      for (int j = 0; j < 16; ++j) r[j] = __uint_as_float(column_get(at_v, j) << 16) * w[j];
      if (len < C) {      // what stands there belongs to the next sequence
#pragma unroll
        for (int j = 0; j < 16; ++j) r[j] = t0 + j < len ? r[j] : 0.f;
      }
      row16(vec + V_KG + t0, w);
      if (!(ok = warp_wait(&s.m1, i & 1))) break;
      umma::fence_after_sync();
      {
        float x[16];
        umma::tmem_ld16(tq + D1 + t0, x);
        umma::tmem_ld16(tq + D1 + 64 + t0, y);
        umma::tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < 16; ++j) r[j] = fmaf(-w[j], x[j], r[j]);      // (behind a sequence's end k's rows are zero)
        const Split a = split8(&r[0]), b = split8(&r[8]);
        umma::tmem_st8(tq + RH + t0 / 2, a.hi, b.hi);
        umma::tmem_st8(tq + RL + t0 / 2, a.lo, b.lo);
        umma::tmem_st_wait();
      }
      warp_arrive(&s.rReady, lane);
      row16(vec + V_Q + t0, w);
#pragma unroll
      for (int j = 0; j < 16; ++j) y[j] *= w[j];      // o so far
      row16(vec + V_W + t0, w);
      // ---- v_new, o ----
      if (!(ok = warp_wait(&s.m2, i & 1))) break;
      umma::fence_after_sync();
      {
        float z[16];
        umma::tmem_ld16(tq + D2 + t0, r);
        umma::tmem_ld16(tq + D2 + 64 + t0, z);
        umma::tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          w[j] *= r[j];
          y[j] += z[j];
        }
        const Split a = split8(&w[0]), b = split8(&w[8]);
        umma::tmem_st8(tq + RH + t0 / 2, a.hi, b.hi);
        umma::tmem_st8(tq + RL + t0 / 2, a.lo, b.lo);
        umma::tmem_st_wait();
      }
      warp_arrive(&s.uReady, lane);
      if constexpr (TRAIN) {
#pragma unroll
        for (int j = 0; j < 16; ++j) column_put(at_v, j, r[j]);
      }
      if (len == C) {
#pragma unroll
        for (int j = 0; j < 16; ++j) column_put(at_o, j, y[j]);
      } else if (v < p.vc) {
#pragma unroll
        for (int j = 0; j < 16; ++j)
          if (t0 + j < len) p.o[(static_cast<size_t>(tok0 + t0 + j) * p.H + h) * p.vc + v] = __float2bfloat16_rn(y[j]);
      }
      fence_proxy_async();
      warp_arrive(&s.oReady, lane);
      // ---- the state ----
      if (!(ok = warp_wait(&s.m3, i & 1))) break;
      umma::fence_after_sync();
      umma::tmem_ld16(tq + D3 + k0, r);
      umma::tmem_ld16(tq + D3 + k0 + 16, y);
      umma::tmem_ld_wait();
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        S[j] = fmaf(S[j], last, r[j]);
        S[16 + j] = fmaf(S[16 + j], last, y[j]);
      }
      umma::fence_before_sync();
    }
    if (!ok) {
      s.dead = 1;
      if (lane == 0) atomicOr(p.status, KDA_STATUS_SCAN_MMA_WAIT);
    } else if (p.ht && v < p.vc) {
#pragma unroll
      for (int e = 0; e < 32; ++e)
        if (k0 + e < p.kc) p.ht[sb + static_cast<size_t>(k0 + e) * p.vc] = S[e];
    }
  } else {
    helper_registers();
    if (warp == W_ISSUE) {
      if (lane == 0) {
        constexpr uint32_t idK = umma::instr_desc(128, 128, false, false), idM = umma::instr_desc(128, 128, false, true);
        const uint64_t dT = umma::desc_kmajor(smem_u32(s.TP[0]), 0);
        bool ok = true;
        for (int i = 0; i < nchunks && ok; ++i) {
          const uint32_t aK = smem_u32(s.KQ[i & 1][0]);
          const uint64_t dK = umma::desc_kmajor(aK, 0), dKm = umma::desc_mnmajor(aK, 0, 16384);
          if (s.dead || !mbar_wait(&s.fullA[i & 1], (i >> 1) & 1) || !mbar_wait(&s.hReady, i & 1)) { ok = false; break; }
          umma::fence_after_sync();
#pragma unroll
          for (int k = 0; k < 8; ++k) {      // hi and lo with the same rows of B
            const uint64_t b = dK + (k >> 2) * 1024u + (k & 3) * umma::KSTEP_KMAJOR;
            umma::mma_ts(tb + D1, tb + AH + 8 * k, b, idK, k > 0);
            umma::mma_ts(tb + D1, tb + AL + 8 * k, b, idK, 1);
          }
          umma::commit(&s.m1);
          if constexpr (TRAIN) {
#pragma unroll
            for (int x = 0; x < 2; ++x) bulk_s2g(p.HS + (static_cast<size_t>(c0 + i) * p.H + h) * T_STATE + x * 16384, s.H[x], 16384);
            bulk_commit();
          }
          if (!mbar_wait(&s.fullB, i & 1) || !mbar_wait(&s.rReady, i & 1)) { ok = false; break; }
          umma::fence_after_sync();
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const uint64_t b = dT + k * umma::KSTEP_KMAJOR;
            umma::mma_ts(tb + D2, tb + RH + 8 * k, b, idK, k > 0);
            umma::mma_ts(tb + D2, tb + RL + 8 * k, b, idK, 1);
            umma::mma_ts(tb + D2, tb + RH + 8 * k, b + 1024u, idK, 1);
          }
          umma::commit(&s.m2);
          umma::commit(&s.freeB);
          if (!mbar_wait(&s.uReady, i & 1)) { ok = false; break; }
          umma::fence_after_sync();
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const uint64_t b = dKm + k * umma::KSTEP_MNMAJOR;
            umma::mma_ts(tb + D3, tb + RH + 8 * k, b, idM, k > 0);
            umma::mma_ts(tb + D3, tb + RL + 8 * k, b, idM, 1);
          }
          if constexpr (TRAIN) bulk_wait_read<0>();      // m3 also says that h's tile may be overwritten
          umma::commit(&s.m3);
          umma::commit(&s.freeA[i & 1]);
        }
        if (!ok) {
          s.dead = 1;
          atomicOr(p.status, KDA_STATUS_SCAN_MMA_WAIT);
        }
        if constexpr (TRAIN) bulk_wait_read<0>();
      }
      __syncwarp();
    } else if (warp == W_ISSUE + 1) {
      if (lane == 0) {
        const int hq = h / p.grp;
        auto first = [&](int i) { return static_cast<int>(tok_begin + static_cast<long long>(i) * C); };
        auto tile_of = [&](int i) { return static_cast<size_t>(c0 + i) * p.H + h; };
        auto loadA = [&](int i) {
          const int b = i & 1, tok0 = first(i);
          mbar_expect_tx(&s.fullA[b], 6 * 8192 + VEC_COPY);
          for (int x = 0; x < 2; ++x) tma_load_rows(s.KQ[b][x], &p.tm_k, 64 * x, hq, tok0, &s.fullA[b]);
          for (int x = 0; x < 2; ++x) tma_load_rows(s.KQ[b][x] + 8192, &p.tm_q, 64 * x, hq, tok0, &s.fullA[b]);
          for (int x = 0; x < 2; ++x) tma_load_rows(s.V[b][x], &p.tm_v, 64 * x, h, tok0, &s.fullA[b]);
          bulk_g2s(s.vec[b], p.VEC + tile_of(i) * T_VEC, VEC_COPY, &s.fullA[b]);
        };
        auto loadB = [&](int i) {
          mbar_expect_tx(&s.fullB, 2 * 16384);
          bulk_g2s(s.TP[0], p.TP + tile_of(i) * T_TP, 32768, &s.fullB);
        };
        bool ok = true;
        if (nchunks > 0) {
          loadA(0);
          loadB(0);
          if (nchunks > 1) loadA(1);
        }
        for (int i = 0; i < nchunks; ++i) {
          if (i + 2 < nchunks) bulk_prefetch(p.TP + tile_of(i + 2) * T_TP, 32768);      // into L2
          if (s.dead || !mbar_wait(&s.oReady, i & 1)) { ok = false; break; }      // (in front of the next load: see warp_wait)
          if (i + 1 < nchunks) {
            if (!mbar_wait(&s.freeB, i & 1)) { ok = false; break; }
            loadB(i + 1);
          }
          if constexpr (TRAIN) {                 // v_new stands in v's tile
#pragma unroll
            for (int x = 0; x < 2; ++x) bulk_s2g(p.VN + tile_of(i) * T_VN + x * 8192, s.V[i & 1][x], 8192);
          }
          if (tok_end - first(i) >= C) {         // o in q's rows
            for (int x = 0; x < 2 && 64 * x < p.vc; ++x) tma_store_rows(&p.tm_o, 64 * x, h, first(i), s.KQ[i & 1][x] + 8192);
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
          atomicOr(p.status, KDA_STATUS_SCAN_LOAD_WAIT);
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

template <bool TRAIN>
static int launch(const ScanParams& p, int units, cudaStream_t st) {
  static DeviceOnce once;
  const int smem = static_cast<int>(sizeof(TSmem<TRAIN>)) + 1024;
  const int rc = once.run([&] { return crew_ready(delta_scan_t_kernel<TRAIN>, smem); });
  if (rc != KDA_OK) return rc;
  return static_cast<int>(launch_chained(delta_scan_t_kernel<TRAIN>, static_cast<unsigned>(units), NT, smem, st, p));
}

int launch_scan_t(const ScanParams& p, int units, cudaStream_t st) { return p.HS ? launch<true>(p, units, st) : launch<false>(p, units, st); }

}  // namespace delta
}  // namespace kda
