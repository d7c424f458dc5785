// Entry points of the chunked gated delta rule with one decay per token and head: argument checks and launches (the formulas: delta.cuh).
#include "delta.cuh"

namespace kda {
namespace delta {

static int validate(const kda_delta_args& a, bool backward) {
  if (a.tokens < 0 || a.N < 0 || a.H <= 0) return KDA_E_SHAPE;
  if (a.HQ < 0 || (a.HQ > 0 && (a.HQ > a.H || a.H % a.HQ != 0))) return KDA_E_SHAPE;
  if (a.K <= 0 || a.K > KD || a.K % 8 || a.V <= 0 || a.V > VD || a.V % 8) return KDA_E_SHAPE;
  if (a.scan_slices != 0 && a.scan_slices != 1 && a.scan_slices != 2 && a.scan_slices != 4) return KDA_E_SHAPE;
  if (a.io_dtype != KDA_BF16) return KDA_E_DTYPE;
  if ((a.g_dtype != KDA_BF16 && a.g_dtype != KDA_FP32) || (a.beta_dtype != KDA_BF16 && a.beta_dtype != KDA_FP32)) return KDA_E_DTYPE;
  if (a.tokens > 0x7fffffffLL - 64) return KDA_E_SHAPE;                                          // tile coordinates are 32 bits
  if ((a.tokens / C + a.N) * a.H > 0x7fff0000LL || static_cast<int64_t>(a.N) * a.H * 4 > 0x7fffffffLL) return KDA_E_SHAPE;      // so are grids
  if (a.tokens == 0) return KDA_OK;
  if (a.N == 0) return backward ? (!a.dq || !a.dk || !a.dv || !a.dg || !a.dbeta ? KDA_E_NULL : KDA_OK) : (!a.o ? KDA_E_NULL : KDA_OK);      // only written: zeros
  if (!a.q || !a.k || !a.v || !a.g || !a.beta || !a.workspace || (!backward && !a.o)) return KDA_E_NULL;
  if (!a.cu_seqlens && a.tokens % a.N != 0) return KDA_E_SHAPE;
  auto addr = [](const void* p) { return reinterpret_cast<uintptr_t>(p); };
  uintptr_t bits = addr(a.q) | addr(a.k) | addr(a.v) | addr(a.o) | addr(a.h0) | addr(a.ht);
  if (backward) {
    if (!a.d_o || !a.dq || !a.dk || !a.dv || !a.dg || !a.dbeta || !a.bwd_workspace) return KDA_E_NULL;
    bits |= addr(a.d_o) | addr(a.dq) | addr(a.dk) | addr(a.dv) | addr(a.d_ht) | addr(a.dh0);
    if (addr(a.bwd_workspace) & 255u) return KDA_E_ALIGN;
  }
  if ((bits & 15u) || (addr(a.workspace) & 255u)) return KDA_E_ALIGN;
  // the small tensors are read an element at a time
  if (((addr(a.g) | (backward ? addr(a.dg) : 0)) & (a.g_dtype == KDA_BF16 ? 1u : 3u)) || ((addr(a.beta) | (backward ? addr(a.dbeta) : 0)) & (a.beta_dtype == KDA_BF16 ? 1u : 3u)) ||
      (addr(a.cu_seqlens) & 3u))
    return KDA_E_ALIGN;
  return KDA_OK;
}

// Packed calls: rows in front of the first sequence and behind the last one belong to nobody; they come out as zeros, for a gradient that is summed
// over them upstream.  `bytes` per row, a multiple of 2.
struct TailParams {
  const int32_t* cu;
  int N, outs;
  long long tokens;
  void* out[5];
  long long bytes[5];
};
__global__ void __launch_bounds__(256) delta_tail_kernel(const TailParams p) {
  chain_point();
  const auto inside = [&](long long x, long long low) { return x < low ? low : x > p.tokens ? p.tokens : x; };
  const long long a = inside(p.cu[0], 0), b = inside(p.cu[p.N], a);
  for (int o = 0; o < p.outs; ++o) {
    const long long per = p.bytes[o] / 2, front = a * per, n = front + (p.tokens - b) * per;
    for (long long i = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x; i < n; i += static_cast<long long>(gridDim.x) * 256)
      static_cast<unsigned short*>(p.out[o])[i < front ? i : b * per + (i - front)] = 0;
  }
}
// the same where there is no sequence at all: every row
static int clear_rows_of(const TailParams& p, cudaStream_t st) {
  for (int o = 0; o < p.outs; ++o) {
    const cudaError_t e = cudaMemsetAsync(p.out[o], 0, static_cast<size_t>(p.bytes[o]) * static_cast<size_t>(p.tokens), st);
    if (e != cudaSuccess) return static_cast<int>(e);
  }
  return KDA_OK;
}
static int launch_tail(const TailParams& p, cudaStream_t st) { return static_cast<int>(launch_chained(delta_tail_kernel, static_cast<unsigned>(sm_count()), 256, 0, st, p)); }

// Sums dq, dk of a group's value heads: eight columns per thread.  The sum is fp32 and rounded once; its terms arrive as bf16, like the operands that they were made
// from (delta.cuh), so what is lost is 2^-8 of each head's gradient, not of the sum's, should the heads cancel.  As fp32 they would be twice the bytes (8 x 4,096 tokens x 32
// value heads: 0.5 GB more to write and read again), and the gradients of a head would still be good to some 2^-8 of its own.
__global__ void __launch_bounds__(256) delta_group_sum_kernel(const __nv_bfloat16* dqh, const __nv_bfloat16* dkh, __nv_bfloat16* dq, __nv_bfloat16* dk, long long pieces,
                                                              int per_row, int grp) {
  chain_point();
  const long long i = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x;
  if (i >= pieces) return;
  const long long row = i / per_row;
  const size_t src = (static_cast<size_t>(row) * grp * per_row + static_cast<size_t>(i % per_row)) * 8, step = static_cast<size_t>(per_row) * 8;
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    float acc[8] = {};
    for (int j = 0; j < grp; ++j) {
      float x[8];
      unpack8(*reinterpret_cast<const uint4*>((which ? dkh : dqh) + src + j * step), x);
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[e] += x[e];
    }
    *reinterpret_cast<uint4*>((which ? dk : dq) + static_cast<size_t>(i) * 8) = pack8(acc);
  }
}

}  // namespace delta
}  // namespace kda

extern "C" size_t kda_delta_chunk_workspace_bytes(int64_t tokens, int32_t N, int32_t H, int32_t K, int32_t V, int32_t save) {
  (void)V;
  if (tokens < 0 || N < 0 || H <= 0) return 0;
  return kda::delta::carve(nullptr, nullptr, tokens, N, H, K, save != 0, false).fwd_bytes;
}
extern "C" size_t kda_delta_chunk_bwd_workspace_bytes(int64_t tokens, int32_t N, int32_t H, int32_t HQ, int32_t K, int32_t V) {
  (void)V;
  if (tokens < 0 || N < 0 || H <= 0) return 0;
  return kda::delta::carve(nullptr, nullptr, tokens, N, H, K, true, HQ > 0 && HQ < H).bwd_bytes;
}

extern "C" int kda_delta_chunk_fwd(const kda_delta_args* args, void* stream) {
  using namespace kda;
  using namespace kda::delta;
  if (!args) return KDA_E_NULL;
  const kda_delta_args& a = *args;
  int rc = validate(a, false);
  if (rc != KDA_OK) return rc;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const TailParams tail{a.cu_seqlens, a.N, 1, a.tokens, {a.o}, {2LL * a.H * a.V}};
  if (a.N == 0) return a.tokens > 0 ? clear_rows_of(tail, st) : KDA_OK;
  if (a.tokens == 0) {
    if (!a.ht || a.ht == a.h0) return KDA_OK;
    const size_t n = static_cast<size_t>(a.N) * a.H * a.K * a.V * sizeof(float);
    return static_cast<int>(a.h0 ? cudaMemcpyAsync(a.ht, a.h0, n, cudaMemcpyDeviceToDevice, st) : cudaMemsetAsync(a.ht, 0, n, st));
  }
  const Ws w = carve(static_cast<unsigned char*>(a.workspace), nullptr, a.tokens, a.N, a.H, a.K, a.save_for_backward != 0, false);
  if (a.workspace_bytes < w.fwd_bytes) return KDA_E_WORKSPACE;
  const int HQ = a.HQ > 0 ? a.HQ : a.H, most = static_cast<int>(a.tokens / C + a.N);
  ChunkWs cw{};
  cw.seq_chunk_off = w.seq_chunk_off; cw.chunk_seq = w.chunk_seq; cw.seq_order = w.seq_order;
  const ChunkMap map = chunk_map(cw, a.cu_seqlens, a.tokens, a.N);

  PrepParams pp{};
  ScanParams sp{};
  if (make_rows_tmap(&pp.tm_q, a.q, false, a.tokens, HQ, a.K, 64, 64, true) || make_rows_tmap(&pp.tm_k, a.k, false, a.tokens, HQ, a.K, 64, 64, true) ||
      make_rows_tmap(&sp.tm_v, a.v, false, a.tokens, a.H, a.V, 64, 64, true) || make_rows_tmap(&sp.tm_o, a.o, false, a.tokens, a.H, a.V, 64, 64, true))
    return KDA_E_TMAP;
  sp.tm_q = pp.tm_q; sp.tm_k = pp.tm_k;
  ProfCall* const prof = prof_begin(st);
  if (a.cu_seqlens) {
    launch_tables(a.cu_seqlens, a.N, a.tokens, most, w.seq_chunk_off, w.chunk_seq, w.seq_order, w.status, st);
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return static_cast<int>(e);
  }
  prof_mark(prof, KDA_STAGE_TABLES, st);
  pp.map = map; pp.g = a.g; pp.beta = a.beta; pp.g_dtype = a.g_dtype; pp.beta_dtype = a.beta_dtype; pp.TP = w.TP; pp.VEC = w.VEC; pp.status = w.status;
  pp.clear_status = a.cu_seqlens == nullptr; pp.H = a.H; pp.grp = a.H / HQ; pp.use_l2norm = a.use_qk_l2norm; pp.scale = a.scale;
  const long long chunks = map.T > 0 ? static_cast<long long>(a.N) * map.per_seq : most;
  if ((rc = launch_prepare(pp, chunks * a.H, st)) != KDA_OK) return rc;
  prof_mark(prof, KDA_STAGE_PREPARE, st);
  sp.map = map; sp.TP = w.TP; sp.VEC = w.VEC; sp.HS = a.save_for_backward ? w.HS : nullptr; sp.VN = a.save_for_backward ? w.VN : nullptr;
  sp.h0 = a.h0; sp.ht = a.ht; sp.o = static_cast<__nv_bfloat16*>(a.o); sp.status = w.status; sp.H = a.H; sp.grp = pp.grp; sp.kc = a.K; sp.vc = a.V;
  if ((rc = delta::launch_scan(sp, a.N * a.H, a.scan_slices, st)) != KDA_OK) return rc;
  if (a.cu_seqlens && (rc = launch_tail(tail, st)) != KDA_OK) return rc;
  prof_mark(prof, KDA_STAGE_SCAN, st);
  return KDA_OK;
}

extern "C" int kda_delta_chunk_bwd(const kda_delta_args* args, void* stream) {
  using namespace kda;
  using namespace kda::delta;
  if (!args) return KDA_E_NULL;
  const kda_delta_args& a = *args;
  int rc = validate(a, true);
  if (rc != KDA_OK) return rc;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int HQ = a.HQ > 0 ? a.HQ : a.H, grp = a.H / HQ, most = static_cast<int>(a.tokens / C + a.N);
  const long long gb = a.g_dtype == KDA_BF16 ? 2 : 4, bb = a.beta_dtype == KDA_BF16 ? 2 : 4;
  const TailParams tail{a.cu_seqlens, a.N, 5, a.tokens, {a.dq, a.dk, a.dv, a.dg, a.dbeta}, {2LL * HQ * a.K, 2LL * HQ * a.K, 2LL * a.H * a.V, gb * a.H, bb * a.H}};
  if (a.N == 0) return a.tokens > 0 ? clear_rows_of(tail, st) : KDA_OK;
  if (a.tokens == 0) {
    if (!a.dh0 || a.dh0 == a.d_ht) return KDA_OK;
    const size_t n = static_cast<size_t>(a.N) * a.H * a.K * a.V * sizeof(float);
    return static_cast<int>(a.d_ht ? cudaMemcpyAsync(a.dh0, a.d_ht, n, cudaMemcpyDeviceToDevice, st) : cudaMemsetAsync(a.dh0, 0, n, st));
  }
  const Ws w = carve(static_cast<unsigned char*>(a.workspace), static_cast<unsigned char*>(a.bwd_workspace), a.tokens, a.N, a.H, a.K, true, grp > 1);
  if (a.workspace_bytes < w.fwd_bytes || a.bwd_workspace_bytes < w.bwd_bytes) return KDA_E_WORKSPACE;
  ChunkWs cw{};
  cw.seq_chunk_off = w.seq_chunk_off; cw.chunk_seq = w.chunk_seq; cw.seq_order = w.seq_order;
  const ChunkMap map = chunk_map(cw, a.cu_seqlens, a.tokens, a.N);
  RScanParams rp{};
  MainParams mp{};
  mp.dq = grp > 1 ? w.DQH : static_cast<__nv_bfloat16*>(a.dq);
  mp.dk = grp > 1 ? w.DKH : static_cast<__nv_bfloat16*>(a.dk);
  if (make_rows_tmap(&mp.tm_q, a.q, false, a.tokens, HQ, a.K, 64, 64, true) || make_rows_tmap(&mp.tm_k, a.k, false, a.tokens, HQ, a.K, 64, 64, true) ||
      make_rows_tmap(&mp.tm_v, a.v, false, a.tokens, a.H, a.V, 64, 64, true) || make_rows_tmap(&mp.tm_do, a.d_o, false, a.tokens, a.H, a.V, 64, 64, true) ||
      make_rows_tmap(&mp.tm_dq, mp.dq, false, a.tokens, a.H, a.K, 64, 64, true) || make_rows_tmap(&mp.tm_dk, mp.dk, false, a.tokens, a.H, a.K, 64, 64, true) ||
      make_rows_tmap(&rp.tm_dv, a.dv, false, a.tokens, a.H, a.V, 64, 64, true))
    return KDA_E_TMAP;
  rp.tm_q = mp.tm_q; rp.tm_k = mp.tm_k; rp.tm_do = mp.tm_do;
  ProfCall* const prof = prof_begin(st);
  rp.map = map; rp.TP = w.TP; rp.VEC = w.VEC; rp.DH = w.DH; rp.DF = w.DF; rp.d_ht = a.d_ht; rp.dh0 = a.dh0; rp.dv = static_cast<__nv_bfloat16*>(a.dv);
  rp.status = w.status; rp.H = a.H; rp.grp = grp; rp.kc = a.K; rp.vc = a.V;
  if ((rc = delta::launch_bwd_scan(rp, a.N * a.H, a.scan_slices, st)) != KDA_OK) return rc;
  prof_mark(prof, KDA_STAGE_BWD_SCAN, st);
  mp.map = map; mp.VEC = w.VEC; mp.HS = w.HS; mp.VN = w.VN; mp.DH = w.DH; mp.DF = w.DF;
  mp.dg = a.dg; mp.dbeta = a.dbeta; mp.g_dtype = a.g_dtype; mp.beta_dtype = a.beta_dtype; mp.status = w.status; mp.H = a.H; mp.grp = grp; mp.kc = a.K;
  mp.use_l2norm = a.use_qk_l2norm; mp.scale = a.scale;
  const long long chunks = map.T > 0 ? static_cast<long long>(a.N) * map.per_seq : most;
  if ((rc = launch_bwd_main(mp, chunks * a.H, (a.V + 63) / 64, st)) != KDA_OK) return rc;
  if (grp > 1) {
    const int per_row = a.K / 8;
    const long long pieces = static_cast<long long>(a.tokens) * HQ * per_row;
    if ((pieces + 255) / 256 > 0x7fffffffLL) return KDA_E_SHAPE;
    rc = static_cast<int>(launch_chained(delta_group_sum_kernel, static_cast<unsigned>((pieces + 255) / 256), 256, 0, st, w.DQH, w.DKH, static_cast<__nv_bfloat16*>(a.dq),
                                         static_cast<__nv_bfloat16*>(a.dk), pieces, per_row, grp));
    if (rc != KDA_OK) return rc;
  }
  if (a.cu_seqlens && (rc = launch_tail(tail, st)) != KDA_OK) return rc;
  prof_mark(prof, KDA_STAGE_BWD_MAIN, st);
  return KDA_OK;
}
