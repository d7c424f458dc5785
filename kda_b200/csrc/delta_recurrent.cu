// Gated delta rule, one decay per token and head, token by token: decode and scans (kda_delta_recurrent_fwd).
//
// The kernels of kda_recurrent.cu with that decay: a warp per (sequence, head, slice of the value columns), its state in registers.  They are kernels of their own: as
// variants of the same templates both sides were compiled differently (with a decay per column one token of one sequence took 4.1 instead of 3.6 us, 48 sequences from
// raw gates 36.8 instead of 33.5).  What else differs: a slot outside the pool or an accepted count that names no column is not followed (HeadArgs), and in packed
// calls offsets are cut to the call's tokens, and rows of no sequence become zeros.
#include "kda_recurrent.cuh"

namespace kda {

namespace {

// Packed calls: rows of o in front of the first sequence and behind the last one become zeros.  All sequences' warps share them, so that a server's padded
// buffer costs no more than its bytes.  Asked for in front of the tokens, used behind them; cut to the call's tokens.
struct RowsOfNone {
  long long first, last;
  template <bool CLEAR>
  __device__ __forceinline__ static RowsOfNone of(const HeadArgs& a) {
    if constexpr (CLEAR) return {a.cu_seqlens[0], a.cu_seqlens[a.N]};
    else return {0, 0};
  }
  // a warp's part: four columns from `col` on in every RG-th row, rg the lane's first
  template <typename IO, int RG>
  __device__ __forceinline__ void clear(const HeadArgs& a, long long n, int h, int col, int rg) const {
    const size_t row = static_cast<size_t>(a.H) * a.V, step = static_cast<size_t>(a.N) * RG * row;
    auto zeros = [&](long long from, long long to) {
      long long t = from + n * RG + rg;
      IO* p = static_cast<IO*>(a.o) + static_cast<size_t>(t) * row + static_cast<size_t>(h) * a.V + col;
#pragma unroll 4
      for (; t < to; t += static_cast<long long>(a.N) * RG, p += step) IoTraits<IO>::st4(p, make_float4(0.f, 0.f, 0.f, 0.f));
    };
    zeros(0, first < a.tokens ? first : a.tokens);
    const long long from = last > 0 ? last : 0;
    zeros(first > from ? first : from, a.tokens);
  }
};

// A token's vectors are fetched while the token before is worked on: with one warp per slice there is nobody else to hide
// their latency (one sequence of four draft tokens: 14.2 us when each token fetched its own, 8.0 us so).
// CLEAR: packed, so that there may be rows of no sequence (a variant of its own: with the rows' few instructions in it one token of one sequence takes 4.1 us, 3.6 without).
template <typename IO, int K, int VS, bool CLEAR>
__global__ void __launch_bounds__(REC_WARPS * 32) delta_recurrent_kernel(const HeadArgs a) {
  chain_point();
  constexpr int CL = VS / 4;      // lanes across the V slice (4 columns each)
  constexpr int RG = 32 / CL;     // row groups
  constexpr int R = K / RG;       // state rows per lane
  constexpr int E = K / 32;       // q/k elements staged per lane
  constexpr bool IO16 = sizeof(IO) == 2;
  static_assert(K % RG == 0 && K % 32 == 0, "unsupported K");

  __shared__ float s_k[REC_WARPS][K], s_q[REC_WARPS][K];

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int nvs = a.V / VS;
  const long long wid = static_cast<long long>(blockIdx.x) * REC_WARPS + warp;
  const long long total = static_cast<long long>(a.N) * a.H * nvs;
  if (wid >= total) return;   // whole warps leave; only __syncwarp is used below
  const int vs = static_cast<int>(wid % nvs);
  const int h = static_cast<int>((wid / nvs) % a.H);
  const int n = static_cast<int>(wid / (static_cast<long long>(nvs) * a.H));
  const int HQ = a.HQ > 0 ? a.HQ : a.H, grp = a.H / HQ;      // grouped value heads
  const int cg = lane % CL, rg = lane / CL;
  const int col = vs * VS + cg * 4;

  long long bos, eos;
  if (a.cu_seqlens) {
    bos = a.cu_seqlens[n];
    eos = a.cu_seqlens[n + 1];
    bos = bos < 0 ? 0 : bos;      // (offsets outside the call's tokens are not followed either)
    eos = eos < a.tokens ? eos : a.tokens;
  } else {
    bos = static_cast<long long>(n) * a.T;
    eos = bos + a.T;
  }
  const bool g16 = a.g_raw_dtype == KDA_BF16, b16 = a.beta_raw_dtype == KDA_BF16;
  struct Token {
    RowBits<E> q, k;
    RowBits<4> v;
    RowBits<1> g, b;
  };
  auto fetch = [&](long long t, Token& x) {
    const size_t rowq = (static_cast<size_t>(t) * HQ + h / grp) * K + lane * E;   // q, k row (their own head count)
    const size_t row = static_cast<size_t>(t) * a.H + h;
    x.q.load(a.q, rowq, IO16);
    x.k.load(a.k, rowq, IO16);
    x.g.load(a.g, row, g16);
    x.b.load(a.beta, row, b16);
    x.v.load(a.v, row * a.V + col, IO16);
  };
  // continuous batching: the sequence's row of slot numbers; it starts from the slot of the last accepted token
  const int32_t* slots = a.state_indices ? a.state_indices + static_cast<size_t>(n) * a.state_indices_stride : nullptr;
  [[maybe_unused]] const RowsOfNone none = RowsOfNone::of<CLEAR>(a);
  long long slot = n;
  if (slots && !a.holds(slot = a.start_slot(n))) {
    if (rg == 0)
      for (long long t = bos; t < eos; ++t) IoTraits<IO>::st4(static_cast<IO*>(a.o) + (static_cast<size_t>(t) * a.H + h) * a.V + col, make_float4(0.f, 0.f, 0.f, 0.f));
    if constexpr (CLEAR) none.clear<IO, RG>(a, n, h, col, rg);
    return;
  }
  Token cur, nxt;
  if (bos < eos) fetch(bos, cur);
  const float bias = a.dt_bias ? a.dt_bias[h] : 0.f, A_log = a.A_log ? a.A_log[h] : 0.f;
  const size_t sbase = (static_cast<size_t>(slot) * a.H + h) * K * a.V + col;

  float4 S[R];
  if (a.h0) {
#pragma unroll
    for (int i = 0; i < R; ++i)
      S[i] = __ldcs(reinterpret_cast<const float4*>(a.h0 + sbase + static_cast<size_t>(rg + RG * i) * a.V));
  } else {
#pragma unroll
    for (int i = 0; i < R; ++i) S[i] = make_float4(0.f, 0.f, 0.f, 0.f);
  }
  IO* op = static_cast<IO*>(a.o);

  for (long long t = bos; t < eos; ++t) {
    if (t + 1 < eos) fetch(t + 1, nxt);
    float qf[E], kf[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
      qf[e] = cur.q.get(e, IO16);
      kf[e] = cur.k.get(e, IO16);
    }
    float g = cur.g.get(0, g16);
    if (a.A_log) g = head_gate(g + bias, A_log, a);
    const float decay = exp_full(g);
    float qs = a.scale;
    if (a.use_qk_l2norm) {
      float sq = 0.f, sk = 0.f;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        sq += qf[e] * qf[e];
        sk += kf[e] * kf[e];
      }
      sq = warp_sum(sq);
      sk = warp_sum(sk);
      qs *= rsqrtf(sq + L2NORM_EPS);
      const float ks = rsqrtf(sk + L2NORM_EPS);
#pragma unroll
      for (int e = 0; e < E; ++e) kf[e] *= ks;
    }
#pragma unroll
    for (int e = 0; e < E; ++e) {
      s_k[warp][lane * E + e] = kf[e];
      s_q[warp][lane * E + e] = qf[e] * qs;
    }
    float beta = cur.b.get(0, b16);
    if (a.beta_sigmoid) beta = sigmoid_full(beta);
    const float4 vt = make_float4(cur.v.get(0, IO16), cur.v.get(1, IO16), cur.v.get(2, IO16), cur.v.get(3, IO16));
    __syncwarp();

    float4 hk = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const int r = rg + RG * i;
      const float kk = s_k[warp][r];
      S[i].x *= decay; S[i].y *= decay; S[i].z *= decay; S[i].w *= decay;
      hk.x += kk * S[i].x; hk.y += kk * S[i].y; hk.z += kk * S[i].z; hk.w += kk * S[i].w;
    }
#pragma unroll
    for (int off = CL; off < 32; off <<= 1) {
      hk.x += __shfl_xor_sync(0xffffffffu, hk.x, off);
      hk.y += __shfl_xor_sync(0xffffffffu, hk.y, off);
      hk.z += __shfl_xor_sync(0xffffffffu, hk.z, off);
      hk.w += __shfl_xor_sync(0xffffffffu, hk.w, off);
    }
    const float4 dv = make_float4(beta * (vt.x - hk.x), beta * (vt.y - hk.y), beta * (vt.z - hk.z), beta * (vt.w - hk.w));
    float4 oa = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const int r = rg + RG * i;
      const float kk = s_k[warp][r], qq = s_q[warp][r];
      S[i].x += kk * dv.x; S[i].y += kk * dv.y; S[i].z += kk * dv.z; S[i].w += kk * dv.w;
      oa.x += qq * S[i].x; oa.y += qq * S[i].y; oa.z += qq * S[i].z; oa.w += qq * S[i].w;
    }
#pragma unroll
    for (int off = CL; off < 32; off <<= 1) {
      oa.x += __shfl_xor_sync(0xffffffffu, oa.x, off);
      oa.y += __shfl_xor_sync(0xffffffffu, oa.y, off);
      oa.z += __shfl_xor_sync(0xffffffffu, oa.z, off);
      oa.w += __shfl_xor_sync(0xffffffffu, oa.w, off);
    }
    if (rg == 0) IoTraits<IO>::st4(op + (static_cast<size_t>(t) * a.H + h) * a.V + col, oa);
    if (slots && a.ht && a.keeps(slots, t - bos)) {      // the state after every token goes to that token's slot
      const size_t tb = (static_cast<size_t>(slots[t - bos]) * a.H + h) * K * a.V + col;
#pragma unroll
      for (int i = 0; i < R; ++i) __stcs(reinterpret_cast<float4*>(a.ht + tb + static_cast<size_t>(rg + RG * i) * a.V), S[i]);
    }
    cur = nxt;
    __syncwarp();
  }

  if (a.ht && !slots) {
#pragma unroll
    for (int i = 0; i < R; ++i)
      __stcs(reinterpret_cast<float4*>(a.ht + sbase + static_cast<size_t>(rg + RG * i) * a.V), S[i]);
  }
  if constexpr (CLEAR) none.clear<IO, RG>(a, n, h, col, rg);
}

// ---- transposed state layout [slots, H, V, K] (K contiguous) ------------------------------------------------------
// One warp owns (sequence, head, 32 value rows); a lane holds the 32 x (K / 32) slice of key columns
// lane*(K/32) .. of those rows, so every state access is again contiguous over the warp.  The two reductions over K
// are per-lane partial dot products summed over the lanes 32 values at a time by a butterfly (lane L ends up with
// the total of value row L); the delta-rule update needs every row's dv in every lane: one shuffle per row.
template <typename IO, int K, bool CLEAR>
__global__ void __launch_bounds__(REC_WARPS * 32) delta_recurrent_t_kernel(const HeadArgs a) {
  constexpr int E = K / 32;       // key columns per lane
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int nvs = a.V / 32;
  const long long wid = static_cast<long long>(blockIdx.x) * REC_WARPS + warp;
  const long long total = static_cast<long long>(a.N) * a.H * nvs;
  if (wid >= total) return;
  const int vs = static_cast<int>(wid % nvs);
  const int h = static_cast<int>((wid / nvs) % a.H);
  const int n = static_cast<int>(wid / (static_cast<long long>(nvs) * a.H));
  const int HQ = a.HQ > 0 ? a.HQ : a.H, grp = a.H / HQ;      // grouped value heads
  long long bos, eos;
  if (a.cu_seqlens) {
    bos = a.cu_seqlens[n];
    eos = a.cu_seqlens[n + 1];
    bos = bos < 0 ? 0 : bos;      // (offsets outside the call's tokens are not followed either)
    eos = eos < a.tokens ? eos : a.tokens;
  } else {
    bos = static_cast<long long>(n) * a.T;
    eos = bos + a.T;
  }
  const int32_t* slots = a.state_indices ? a.state_indices + static_cast<size_t>(n) * a.state_indices_stride : nullptr;
  [[maybe_unused]] const RowsOfNone none = RowsOfNone::of<CLEAR>(a);
  long long slot = n;
  if (slots && !a.holds(slot = a.start_slot(n))) {
    for (long long t = bos; t < eos; ++t) static_cast<IO*>(a.o)[(static_cast<size_t>(t) * a.H + h) * a.V + vs * 32 + lane] = IO(0.f);
    if constexpr (CLEAR) none.clear<IO, 4>(a, n, h, vs * 32 + 4 * (lane & 7), lane >> 3);
    return;
  }
  auto state_ptr = [&](const float* base, long long sl) {
    return base + ((static_cast<size_t>(sl) * a.H + h) * a.V + vs * 32) * K + lane * E;
  };
  float S[32][E];
  if (a.h0) {
    const float* p0 = state_ptr(a.h0, slot);
#pragma unroll
    for (int r = 0; r < 32; ++r) ld_row<E>(S[r], p0 + static_cast<size_t>(r) * K);
  } else {
#pragma unroll
    for (int r = 0; r < 32; ++r)
#pragma unroll
      for (int e = 0; e < E; ++e) S[r][e] = 0.f;
  }
  const IO* qp = static_cast<const IO*>(a.q);
  const IO* kp = static_cast<const IO*>(a.k);
  const IO* vp = static_cast<const IO*>(a.v);
  IO* op = static_cast<IO*>(a.o);
  for (long long t = bos; t < eos; ++t) {
    const size_t rowq = (static_cast<size_t>(t) * HQ + h / grp) * K + lane * E;   // q, k row (their own head count)
    float qf[E], kf[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
      qf[e] = IoTraits<IO>::ld(qp + rowq + e);
      kf[e] = IoTraits<IO>::ld(kp + rowq + e);
    }
    const float decay = exp_full(recurrent_head_decay(a, static_cast<size_t>(t) * a.H + h, h));
    float qs = a.scale;
    if (a.use_qk_l2norm) {
      float sq = 0.f, sk = 0.f;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        sq += qf[e] * qf[e];
        sk += kf[e] * kf[e];
      }
      sq = warp_sum(sq);
      sk = warp_sum(sk);
      qs *= rsqrtf(sq + L2NORM_EPS);
      const float ks = rsqrtf(sk + L2NORM_EPS);
#pragma unroll
      for (int e = 0; e < E; ++e) kf[e] *= ks;
    }
#pragma unroll
    for (int e = 0; e < E; ++e) qf[e] *= qs;
    const float beta = recurrent_head_beta(a, static_cast<size_t>(t) * a.H + h);
    const float vt = IoTraits<IO>::ld(vp + (static_cast<size_t>(t) * a.H + h) * a.V + vs * 32 + lane);      // value row `lane`
    float part[32];
#pragma unroll
    for (int r = 0; r < 32; ++r) {
      float acc = 0.f;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        S[r][e] *= decay;
        acc = fmaf(kf[e], S[r][e], acc);
      }
      part[r] = acc;
    }
    const float hk = butterfly_sum32(part, lane);            // S^T k for value row `lane`
    const float dv = beta * (vt - hk);
#pragma unroll
    for (int r = 0; r < 32; ++r) {
      const float dvr = __shfl_sync(0xffffffffu, dv, r);
      float acc = 0.f;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        S[r][e] = fmaf(kf[e], dvr, S[r][e]);
        acc = fmaf(qf[e], S[r][e], acc);
      }
      part[r] = acc;
    }
    const float o = butterfly_sum32(part, lane);
    if (sizeof(IO) == 2) reinterpret_cast<__nv_bfloat16*>(op)[(static_cast<size_t>(t) * a.H + h) * a.V + vs * 32 + lane] = __float2bfloat16_rn(o);
    else reinterpret_cast<float*>(op)[(static_cast<size_t>(t) * a.H + h) * a.V + vs * 32 + lane] = o;
    if (slots && a.ht && a.keeps(slots, t - bos)) {
      float* pt = const_cast<float*>(state_ptr(a.ht, slots[t - bos]));
#pragma unroll
      for (int r = 0; r < 32; ++r) st_row<E>(pt + static_cast<size_t>(r) * K, S[r]);
    }
  }
  if (a.ht && !slots) {
    float* pt = const_cast<float*>(state_ptr(a.ht, slot));
#pragma unroll
    for (int r = 0; r < 32; ++r) st_row<E>(pt + static_cast<size_t>(r) * K, S[r]);
  }
  if constexpr (CLEAR) none.clear<IO, 4>(a, n, h, vs * 32 + 4 * (lane & 7), lane >> 3);
}

template <typename IO, int K>
int launch_rec_t(const HeadArgs& a, cudaStream_t st) {
  const long long total = static_cast<long long>(a.N) * a.H * (a.V / 32);
  const long long blocks = (total + REC_WARPS - 1) / REC_WARPS;
  if (blocks <= 0) return KDA_OK;
  if (blocks > 0x7fffffffLL) return KDA_E_SHAPE;
  if (a.cu_seqlens) delta_recurrent_t_kernel<IO, K, true><<<static_cast<unsigned>(blocks), REC_WARPS * 32, 0, st>>>(a);
  else delta_recurrent_t_kernel<IO, K, false><<<static_cast<unsigned>(blocks), REC_WARPS * 32, 0, st>>>(a);
  return static_cast<int>(cudaGetLastError());
}

template <typename IO, int K, int VS>
int launch_rec(const HeadArgs& a, cudaStream_t st) {
  const long long total = static_cast<long long>(a.N) * a.H * (a.V / VS);
  const long long blocks = (total + REC_WARPS - 1) / REC_WARPS;
  if (blocks <= 0) return KDA_OK;
  if (blocks > 0x7fffffffLL) return KDA_E_SHAPE;
  if (a.cu_seqlens) return static_cast<int>(launch_chained(delta_recurrent_kernel<IO, K, VS, true>, static_cast<unsigned>(blocks), REC_WARPS * 32, 0, st, a));
  return static_cast<int>(launch_chained(delta_recurrent_kernel<IO, K, VS, false>, static_cast<unsigned>(blocks), REC_WARPS * 32, 0, st, a));
}

template <typename IO>
int dispatch_rec(const HeadArgs& a, cudaStream_t st) {
  if (a.transpose_state) {
    switch (a.K) {
      case 64: return launch_rec_t<IO, 64>(a, st);
      case 128: return launch_rec_t<IO, 128>(a, st);
      default: return KDA_E_SHAPE;
    }
  }
  switch (a.K) {
    case 32: return launch_rec<IO, 32, 32>(a, st);
    case 64: return launch_rec<IO, 64, 32>(a, st);
    // one or two sequences leave most SMs idle: twice as many warps with half the columns each (one sequence x 32 heads, one token: 3.4
    // instead of 4.3 us; from half a state per SM on the wider slices win: 96 states 4.3 against 4.5 us)
    case 128: return 2LL * a.N * a.H <= sm_count() ? launch_rec<IO, 128, 16>(a, st) : launch_rec<IO, 128, 32>(a, st);
    case 256: return (a.V % 32 == 0) ? launch_rec<IO, 256, 16>(a, st) : KDA_E_SHAPE;
    default: return KDA_E_SHAPE;
  }
}

}  // namespace

int recurrent_head_launch(const HeadArgs& a, cudaStream_t st) {
  if (a.io_dtype == KDA_BF16) return dispatch_rec<__nv_bfloat16>(a, st);
  if (a.io_dtype == KDA_FP32) return dispatch_rec<float>(a, st);
  return KDA_E_DTYPE;
}

}  // namespace kda
