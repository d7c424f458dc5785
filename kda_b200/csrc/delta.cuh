// The gated delta rule with one decay per (token, head), in chunks of 64 tokens: shared definitions.
//
//     S_t = exp(g_t) (I - beta_t k_t k_t^T) S_{t-1} + beta_t k_t v_t^T,      o_t = scale S_t^T q_t
//
// With one decay per token the decays between two tokens of a chunk are a matrix D_ij = exp(G_i - G_j) (G: sums of g within the chunk) that
// multiplies the products k_i k_j and q_i k_j behind the tensor cores, so that q, k, v and dO are operands as they stand in memory: exact in bf16,
// with no decay-scaled copies.  For a chunk with start state h (K, Q, V: its rows, w_i = exp(G_last - G_i)):
//     A_ij = beta_i D_ij <k_i, k_j>  (j < i),   Tm = (I + A)^-1,   P_ij = scale D_ij <q_i, k_j>  (j <= i),   Pt = P Tm
//     r = beta (V - exp(G) K h),   v_new = Tm r,   o = scale exp(G) Q h + Pt r,   h' = exp(G_last) h + K^T (w v_new)
// and backward, with dh' the gradient of the state behind the chunk:
//     x = w (K dh'),   f = Tm^T x + Pt^T dO  (the gradient of r),   dv = beta f,   dh = exp(G_last) dh' + Q^T (scale exp(G) dO) - K^T (beta exp(G) f)
//     dP_ij = dO_i v_new_j,   dA_ij = -f_i v_new_j
//     dq = scale exp(G) (dO h^T) + (scale D dP) K
//     dk = -beta exp(G) (f h^T) + w (v_new dh'^T) + (beta D dA) K + (beta D dA)^T K + (scale D dP)^T Q
//     dbeta_i = f_i (v_i - exp(G_i) h^T k_i) + sum_j dA_ij D_ij <k_i, k_j>
//     dG_i = q_i dq_i - k_i dk_i, where k's first and third term count with the other sign;  dG_last += exp(G_last) <h, dh'> + sum_i w_i k_i (v_new dh'^T)_i
//     dg = the sum of dG from a token to its chunk's end.
// use_qk_l2norm: rows count as x rsqrt(|x|^2 + 1e-6); these factors travel with the decays, the operands stay what they are.
//
// Precision.  State and gradient of the state are fp32 in registers.  Every operand that is not an input (h, r, v_new, dh', x, f, Tm, Pt) enters the two
// scans as two bf16, hi + lo = 17 bits, with the products hi hi, hi lo and lo hi: final states are good to about 1e-5 of their norm, where one
// bf16 per operand gives 3e-3.  The per-chunk gradients, which end in bf16, take one bf16 per operand; dq and dk of a group's value heads are rounded per head, in front
// of their fp32 sum.
//
// Tiles in the workspace, per (chunk, head), bf16 rows of 128 bytes, swizzled (umma::sw128), each a tcgen05 operand as it lies in memory:
//   TP      [128][64] hi, then lo: rows 0..63 Tm, rows 64..127 Pt
//   VEC     fp32 rows of 64: see the V_ constants; then exp(G_last)
//   HS, DH  [128 v][64 keys] x 2: state in front of the chunk, gradient of the state behind it, both transposed
//   VN, DF  [64 t][64 v] x 2: v_new and f
#pragma once

#include "kda_chunk.cuh"
#include "kda_device.cuh"
#include "kda_tma.cuh"
#include "kda_umma.cuh"

namespace kda {
namespace delta {

constexpr size_t T_TP = 32768, T_STATE = 32768, T_VN = 16384;
constexpr size_t T_VEC = 2304;      // 8 rows of 64 and a word, rounded up to 256
constexpr unsigned VEC_COPY = 2064; // what the scans read of it (a multiple of 16)
// rows of VEC: beta; beta exp(G) / |k|; w / |k|; scale exp(G) / |q|; G as two floats (log2), 1 / |k|, 1 / |q|; VG_LAST: exp(G_last)
constexpr int V_BETA = 0, V_KG = 64, V_W = 128, V_Q = 192, V_GHI = 256, V_GLO = 320, V_RK = 384, V_RQ = 448, V_LAST = 512;

struct Ws {
  unsigned* status;
  int *seq_chunk_off, *chunk_seq, *seq_order;
  unsigned char *TP, *VEC, *HS, *VN;      // HS, VN: for a backward
  unsigned char *DH, *DF;                 // the backward's own
  __nv_bfloat16 *DQH, *DKH;               // [tokens][H][K]: per value head, grouped heads only
  size_t fwd_bytes, bwd_bytes;
};

inline Ws carve(unsigned char* base, unsigned char* bwd, int64_t tokens, int N, int H, int K, bool save, bool grouped) {
  Ws w{};
  const size_t most = static_cast<size_t>(tokens / C + N), tiles = most * static_cast<size_t>(H);
  size_t off = 0;
  auto take = [&](size_t n) { unsigned char* p = base ? base + off : nullptr; off += align_up(n); return p; };
  w.status = reinterpret_cast<unsigned*>(take(16));      // first: kda_chunk_status reads it there
  w.seq_chunk_off = reinterpret_cast<int*>(take(sizeof(int) * (static_cast<size_t>(N) + 1)));
  w.chunk_seq = reinterpret_cast<int*>(take(sizeof(int) * (most + 1)));
  w.seq_order = reinterpret_cast<int*>(take(sizeof(int) * (static_cast<size_t>(N) + 1)));
  w.TP = take(tiles * T_TP);
  w.VEC = take(tiles * T_VEC);
  if (save) {
    w.HS = take(tiles * T_STATE);
    w.VN = take(tiles * T_VN);
  }
  w.fwd_bytes = off;
  off = 0;
  auto takeb = [&](size_t n) { unsigned char* p = bwd ? bwd + off : nullptr; off += align_up(n); return p; };
  w.DH = takeb(tiles * T_STATE);
  w.DF = takeb(tiles * T_VN);
  if (grouped) {
    w.DQH = reinterpret_cast<__nv_bfloat16*>(takeb(static_cast<size_t>(tokens) * H * K * 2));
    w.DKH = reinterpret_cast<__nv_bfloat16*>(takeb(static_cast<size_t>(tokens) * H * K * 2));
  }
  w.bwd_bytes = off;
  return w;
}

// The walks of sixteen compute warps and a warpgroup of helpers (of which two warps work): 20 warps of 96 registers a thread at launch, 61,440 in all.  The helpers
// give 32 of theirs up, and the compute warps have 104: 512 x 104 + 128 x 64 = 61,440.
constexpr int CREW_THREADS = 640, CREW_REGS = 96;
__device__ __forceinline__ void compute_registers() { asm volatile("setmaxnreg.inc.sync.aligned.u32 104;"); }
__device__ __forceinline__ void helper_registers() { asm volatile("setmaxnreg.dec.sync.aligned.u32 64;"); }
// the split draws on what the kernel was launched with: with fewer, the compute warps would wait forever
template <class K>
cudaError_t crew_ready(K kernel, int smem) {
  cudaFuncAttributes f{};
  const cudaError_t e = cudaFuncGetAttributes(&f, kernel);
  if (e != cudaSuccess) return e;
  if ((f.numRegs + 7) / 8 * 8 < CREW_REGS) return cudaErrorLaunchOutOfResources;
  return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
}

struct PrepParams {
  ChunkMap map;
  const void *g, *beta;           // [tokens][H] of g_dtype, beta_dtype
  int g_dtype, beta_dtype;
  unsigned char *TP, *VEC;
  unsigned* status;
  int clear_status, H, grp, use_l2norm;
  float scale;
  alignas(64) CUtensorMap tm_q, tm_k;      // [64][64] boxes, 128-byte swizzle
};
struct ScanParams {
  ChunkMap map;
  const unsigned char *TP, *VEC;
  unsigned char *HS, *VN;         // NULL without a backward
  const float* h0;
  float* ht;
  __nv_bfloat16* o;
  unsigned* status;
  int H, grp, kc, vc;
  alignas(64) CUtensorMap tm_q, tm_k, tm_v, tm_o;
};
struct RScanParams {
  ChunkMap map;
  const unsigned char *TP, *VEC;
  unsigned char *DH, *DF;
  const float* d_ht;
  float* dh0;
  __nv_bfloat16* dv;
  unsigned* status;
  int H, grp, kc, vc;
  alignas(64) CUtensorMap tm_q, tm_k, tm_do, tm_dv;
};
struct MainParams {
  ChunkMap map;
  const unsigned char *VEC, *HS, *VN, *DH, *DF;
  __nv_bfloat16 *dq, *dk;         // [tokens][H or HQ][kc]
  void *dg, *dbeta;               // [tokens][H] of g_dtype, beta_dtype
  int g_dtype, beta_dtype;
  unsigned* status;
  int H, grp, kc, use_l2norm;
  float scale;
  alignas(64) CUtensorMap tm_q, tm_k, tm_v, tm_do, tm_dq, tm_dk;
};

int launch_prepare(const PrepParams& p, long long tiles, cudaStream_t st);
// The walks: `slices` CTAs per (sequence, head) unit (1, 2 or 4; 0: by the number of units and SMs).  The forms with one CTA are in files of their own.
int launch_scan(const ScanParams& p, int units, int slices, cudaStream_t st);
int launch_scan_t(const ScanParams& p, int units, cudaStream_t st);
int launch_bwd_scan(const RScanParams& p, int units, int slices, cudaStream_t st);
int launch_bwd_scan_t(const RScanParams& p, int units, cudaStream_t st);
int launch_bwd_main(const MainParams& p, long long tiles, int spans, cudaStream_t st);   // spans of 64 value columns

// x = hi + lo to 17 bits: eight neighbours at a time, as the two 16-byte pieces of an operand row
struct Split { uint4 hi, lo; };
__device__ __forceinline__ void split2(float a, float b, uint32_t& hi, uint32_t& lo) {
  hi = pack_bf16(a, b);
  const float2 h = unpack_bf16(hi);
  lo = pack_bf16(a - h.x, b - h.y);
}
__device__ __forceinline__ Split split8(const float* v) {
  Split s;
  split2(v[0], v[1], s.hi.x, s.lo.x);
  split2(v[2], v[3], s.hi.y, s.lo.y);
  split2(v[4], v[5], s.hi.z, s.lo.z);
  split2(v[6], v[7], s.hi.w, s.lo.w);
  return s;
}
__device__ __forceinline__ uint4 pack8(const float* v) {
  return make_uint4(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7]));
}
__device__ __forceinline__ void unpack8(const uint4& u, float* v) {
  const float2 a = unpack_bf16(u.x), b = unpack_bf16(u.y), c = unpack_bf16(u.z), d = unpack_bf16(u.w);
  v[0] = a.x; v[1] = a.y; v[2] = b.x; v[3] = b.y; v[4] = c.x; v[5] = c.y; v[6] = d.x; v[7] = d.y;
}
// 16-byte piece `pc` (8 columns) of a row of a tile of 128-byte rows
__device__ __forceinline__ unsigned char* piece(unsigned char* tile, int row, int pc) { return tile + row * 128 + (((pc ^ row) & 7) << 4); }
__device__ __forceinline__ const unsigned char* piece(const unsigned char* tile, int row, int pc) { return tile + row * 128 + (((pc ^ row) & 7) << 4); }
// A wait knows the parity of a phase, not its number: a warp that still waits for phase n when n + 1 is complete waits for good.  Most phases cannot be ahead of whoever
// waits for them, since the next one needs something of that warp: oReady of two walks is waited for in front of the load that the next chunk needs.  Where the load
// has to go out first (oReady of the other two, ready and done of the gradients), the loading warp takes part in the barrier: it arrives for a phase once it has seen the one
// before.  (In delta_scan_t.cu that made the compiler spill: 493 us instead of 463 for the walk of 8 x 4,096 tokens x 32 heads.)
__device__ __forceinline__ bool warp_wait(uint64_t* bar, unsigned parity) { return __all_sync(0xffffffffu, mbar_wait(bar, parity)); }
__device__ __forceinline__ void warp_arrive(uint64_t* bar, int lane) {
  umma::fence_before_sync();
  __syncwarp();
  if (lane == 0) mbar_arrive(bar);
}
// eight columns (col a multiple of 8) of a row of an operand of VC columns as bf16 pairs: 32 + 32 side by side in one tile, 64 in two
template <int VC>
__device__ __forceinline__ void put(unsigned char* tile, int rows, int row, int col, const Split& x) {
  if constexpr (VC == 32) {
    *reinterpret_cast<uint4*>(piece(tile, row, col >> 3)) = x.hi;
    *reinterpret_cast<uint4*>(piece(tile, row, 4 + (col >> 3))) = x.lo;
  } else {
    *reinterpret_cast<uint4*>(piece(tile, row, col >> 3)) = x.hi;
    *reinterpret_cast<uint4*>(piece(tile + rows * 128, row, col >> 3)) = x.lo;
  }
}
// One value column of a [64 t][64 v] tile in shared memory, two bytes a row: `at` from column_at for a first row that is a multiple of eight, `j` rows further.
__device__ __forceinline__ uint32_t column_at(const unsigned char* tile, int row, int v) { return smem_u32(tile) + umma::sw128(row, v); }
__device__ __forceinline__ uint32_t column_get(uint32_t at, int j) {
  unsigned short x;
  asm volatile("ld.shared.u16 %0, [%1];" : "=h"(x) : "r"((at ^ ((j & 7) << 4)) + j * 128) : "memory");
  return x;
}
__device__ __forceinline__ void column_put(uint32_t at, int j, float x) {
  asm volatile("st.shared.b16 [%0], %1;" ::"r"((at ^ ((j & 7) << 4)) + j * 128), "h"(__bfloat16_as_ushort(__float2bfloat16_rn(x))) : "memory");
}
// sixteen neighbours of VEC
__device__ __forceinline__ void row16(const float* p, float (&x)[16]) {
#pragma unroll
  for (int e = 0; e < 16; e += 4) *reinterpret_cast<float4*>(&x[e]) = *reinterpret_cast<const float4*>(p + e);
}
// eight value columns of a state's row `key`, as bf16, into a [128 v][64 keys] x 2 tile in global memory: the lanes of a warp are neighbouring keys
__device__ __forceinline__ void leave_state(unsigned char* tile, int key, int v, const uint4& x) {
  const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
  for (int j = 0; j < 8; ++j)
    *reinterpret_cast<uint16_t*>(tile + (key >> 6) * 16384 + umma::sw128(v + j, key & 63)) = static_cast<uint16_t>(j & 1 ? w[j / 2] >> 16 : w[j / 2]);
}
// rows len..63 of the [64][64] boxes at `tile` and `tile + stride` (a sequence's last chunk): what a load found there belongs to the next sequence
__device__ __forceinline__ void clear_rows(unsigned char* tile, int len, int tid, int nthreads) {
  for (int e = tid; e < (C - len) * 8; e += nthreads) *reinterpret_cast<uint4*>(tile + (len + (e >> 3)) * 128 + (e & 7) * 16) = make_uint4(0, 0, 0, 0);
}

}  // namespace delta
}  // namespace kda
