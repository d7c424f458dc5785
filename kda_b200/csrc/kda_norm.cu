// The norms around a block, each one pass over its rows, forward and backward:
//
//   gated      y = n w act(z),  n = x / rms(x),  act: sigmoid or z sigmoid(z)                     (behind the operator, before the output projection)
//              dn = dy w act,  dx = (dn - n mean(dn n)) / rms(x),  dz = dy n w act'(z),  dw = sum over rows of dy n act
//   residual   b = x, or n1 wp with n1 = x / rms(x);  r = residual + s b;  y = n w,  n = r / rms(r)        (between two blocks)
//              t = dr + (dy w - n mean(dy w n)) / rms(r):  the gradient of the residual;  db = s t;  dx = db, or (db wp - n1 mean(db wp n1)) / rms(x)
//              dw = sum of dy n;  with A the sum of t n1 (n1 = x without a norm of its own):  dwp = s A,  ds = wp A
//   rms(x) = sqrt(mean x^2 + eps).  All sums are fp32; every tensor may be bf16 or fp32 on its own.
//
// Bound by HBM: each tensor crosses it once.  A thread holds eight neighbouring columns (16 or 32 bytes) of a row; up to 256 columns a row belongs to
// 2^n lanes of a warp (a warp has several rows in flight and no barrier), beyond that to a CTA.  The backward recomputes the norms from the inputs, which it
// reads anyway, so the forward keeps nothing.  Sums over rows stay in registers while a CTA walks its rows; its partial sums are added in a second kernel in a
// fixed order, so that gradients have the same bits on every run.  Columns that are no multiple of eight, or rows at odd addresses, are read one by one.
// Calls with many rows take kda_norm_ring.cu's kernels, where rows travel through shared memory; these here serve the others (a decode step's 48 rows: no
// ring to set up: 2.6 us a call against 5.3) and odd rows that are too wide for it.
#include <algorithm>

#include "kda_norm.cuh"

namespace kda {

namespace {

constexpr int NORM_CTA = 256;           // threads of a CTA of the kernels for narrow rows
constexpr int NARROW = 256;             // columns up to which a row stays inside a warp

// The sum over a row's threads of one value, in all of them.  Wide: through shared memory, in turns of two so that one barrier is enough.
template <bool WIDE>
struct RowSum {
  float (*part)[32];      // [2][32]
  int lanes, turn = 0;
  __device__ __forceinline__ float operator()(float x) {
    if constexpr (!WIDE) {
      for (int o = lanes >> 1; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
      return x;
    } else {
      x = warp_sum(x);
      const int warps = blockDim.x >> 5;
      if ((threadIdx.x & 31) == 0) part[turn][threadIdx.x >> 5] = x;
      __syncthreads();
      x = 0.f;
      for (int w = 0; w < warps; ++w) x += part[turn][w];
      turn ^= 1;
      return x;
    }
  }
};

struct NormParams {
  kda_norm_args a;
  float* partial;         // [CTAs][sums][cols]
  int lanes;              // threads of a row (narrow)
};

// a CTA's sums over its rows -> partial[CTA][which][column]
template <bool VEC, int NV, bool WIDE, int SUMS>
__device__ __forceinline__ void leave_sums(const NormParams& p, const Cols<VEC>& c, float (&acc)[SUMS][NV][8]) {
  float* const out = p.partial + static_cast<size_t>(blockIdx.x) * SUMS * c.cols;
  if constexpr (WIDE) {
#pragma unroll
    for (int s = 0; s < SUMS; ++s)
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (c.any(i) && c.has(i, j)) out[s * c.cols + c.at(i, j)] = acc[s][i][j];
  } else {      // several rows at a time: their threads' sums in the order of the threads
    __shared__ float m[NORM_CTA * 8];
    const int rows = NORM_CTA / c.lanes;
#pragma unroll
    for (int s = 0; s < SUMS; ++s) {
      __syncthreads();
#pragma unroll
      for (int j = 0; j < 8; ++j) m[threadIdx.x * 8 + j] = acc[s][0][j];
      __syncthreads();
      for (int e = threadIdx.x; e < c.lanes * 8; e += NORM_CTA) {
        const Cols<VEC> d{e >> 3, c.lanes, c.cols};
        float x = 0.f;
        for (int r = 0; r < rows; ++r) x += m[r * c.lanes * 8 + e];
        if (d.any(0) && d.has(0, e & 7)) out[s * c.cols + d.at(0, e & 7)] = x;
      }
    }
  }
}

template <bool VEC, int NV, bool WIDE>
__device__ __forceinline__ Cols<VEC> my_cols(const NormParams& p) {
  return WIDE ? Cols<VEC>{static_cast<int>(threadIdx.x), static_cast<int>(blockDim.x), p.a.cols} : Cols<VEC>{static_cast<int>(threadIdx.x) & (p.lanes - 1), p.lanes, p.a.cols};
}
// first row of a thread and the step to its next; narrow: every lane of a warp takes part in the sums, so rows beyond the end are walked without loads
template <bool WIDE>
__device__ __forceinline__ void my_rows(const NormParams& p, long long& row, long long& step, long long& last) {
  const int per = WIDE ? 1 : NORM_CTA / p.lanes;
  row = static_cast<long long>(blockIdx.x) * per + (WIDE ? 0 : static_cast<int>(threadIdx.x) / p.lanes);
  step = static_cast<long long>(gridDim.x) * per;
  last = (p.a.rows + per - 1) / per * per;      // the same number of turns for a CTA's threads
}

__device__ __forceinline__ void act_as(bool exact, float z, int activation, float& act, float& slope) {
  if (exact) act_of<true>(z, activation, act, slope);
  else act_of<false>(z, activation, act, slope);
}

// ---- gated -----------------------------------------------------------------------------------------------------------------------------------
template <bool VEC, int NV, bool WIDE>
__global__ void gated_fwd_kernel(const __grid_constant__ NormParams p) {
  __shared__ float part[2][32];
  const kda_norm_args& a = p.a;
  const Cols<VEC> c = my_cols<VEC, NV, WIDE>(p);
  RowSum<WIDE> sum{part, p.lanes};
  const float inv = 1.f / a.cols;
  const bool exact = a.io_dtype == KDA_FP32;
  long long row, step, last;
  my_rows<WIDE>(p, row, step, last);
  float w[NV][8];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    if (a.weight) load8<VEC>(a.weight, 0, a.weight_dtype, c, i, w[i]);
    else
#pragma unroll
      for (int j = 0; j < 8; ++j) w[i][j] = 1.f;
  }
  for (; row < last; row += step) {
    const bool there = row < a.rows;
    Bits bx[NV], bz[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      bx[i] = bz[i] = Bits{};
      if (there) {
        bx[i] = fetch<VEC>(a.x, row, a.io_dtype, c, i);
        bz[i] = fetch<VEC>(a.gate, row, a.gate_dtype, c, i);
      }
    }
    float x[NV][8], ss = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      values(bx[i], a.io_dtype, x[i]);
#pragma unroll
      for (int j = 0; j < 8; ++j) ss = fmaf(x[i][j], x[i][j], ss);
    }
    const float rstd = rsqrtf(fmaf(sum(ss), inv, a.eps));
    if (!there) continue;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float z[8];
      values(bz[i], a.gate_dtype, z);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        float act, slope;
        act_as(exact, z[j], a.activation, act, slope);
        z[j] = x[i][j] * rstd * w[i][j] * act;
      }
      store8<VEC>(a.y, row, a.io_dtype, c, i, z);
    }
  }
}

template <bool VEC, int NV, bool WIDE>
__global__ void __launch_bounds__(WIDE ? 512 : NORM_CTA) gated_bwd_kernel(const __grid_constant__ NormParams p) {
  __shared__ float part[2][32];
  const kda_norm_args& a = p.a;
  const Cols<VEC> c = my_cols<VEC, NV, WIDE>(p);
  RowSum<WIDE> sum{part, p.lanes};
  const float inv = 1.f / a.cols;
  const bool exact = a.io_dtype == KDA_FP32;
  long long row, step, last;
  my_rows<WIDE>(p, row, step, last);
  float w[NV][8], acc[1][NV][8] = {};
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    if (a.weight) load8<VEC>(a.weight, 0, a.weight_dtype, c, i, w[i]);
    else
#pragma unroll
      for (int j = 0; j < 8; ++j) w[i][j] = 1.f;
  }
  for (; row < last; row += step) {
    const bool there = row < a.rows;
    Bits bx[NV], bz[NV], bd[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      bx[i] = bz[i] = bd[i] = Bits{};
      if (there) {
        bx[i] = fetch<VEC>(a.x, row, a.io_dtype, c, i);
        bz[i] = fetch<VEC>(a.gate, row, a.gate_dtype, c, i);
        bd[i] = fetch<VEC>(a.dy, row, a.io_dtype, c, i);
      }
    }
    float x[NV][8], ss = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      values(bx[i], a.io_dtype, x[i]);
#pragma unroll
      for (int j = 0; j < 8; ++j) ss = fmaf(x[i][j], x[i][j], ss);
    }
    const float rstd = rsqrtf(fmaf(sum(ss), inv, a.eps));
    float dn[NV][8], dz[NV][8], dot = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float d[8];
      values(bd[i], a.io_dtype, d);
      values(bz[i], a.gate_dtype, dz[i]);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        float act, slope;
        act_as(exact, dz[i][j], a.activation, act, slope);
        x[i][j] *= rstd;
        acc[0][i][j] = there ? fmaf(d[j] * x[i][j], act, acc[0][i][j]) : acc[0][i][j];
        dn[i][j] = d[j] * w[i][j] * act;
        dz[i][j] = d[j] * w[i][j] * x[i][j] * slope;
        dot = fmaf(dn[i][j], x[i][j], dot);
      }
    }
    dot = sum(dot) * inv;
    if (!there) continue;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
#pragma unroll
      for (int j = 0; j < 8; ++j) dn[i][j] = rstd * fmaf(-dot, x[i][j], dn[i][j]);
      store8<VEC>(a.dx, row, a.io_dtype, c, i, dn[i]);
      store8<VEC>(a.dgate, row, a.gate_dtype, c, i, dz[i]);
    }
  }
  if (p.partial) leave_sums<VEC, NV, WIDE, 1>(p, c, acc);
}

// ---- residual ----------------------------------------------------------------------------------------------------------------------------------
template <bool VEC, int NV, bool WIDE>
__global__ void residual_fwd_kernel(const __grid_constant__ NormParams p) {
  __shared__ float part[2][32];
  const kda_norm_args& a = p.a;
  const Cols<VEC> c = my_cols<VEC, NV, WIDE>(p);
  RowSum<WIDE> sum{part, p.lanes};
  const float inv = 1.f / a.cols;
  long long row, step, last;
  my_rows<WIDE>(p, row, step, last);
  for (; row < last; row += step) {
    const bool there = row < a.rows;
    Bits bx[NV], br[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      bx[i] = br[i] = Bits{};
      if (there) {
        bx[i] = fetch<VEC>(a.x, row, a.io_dtype, c, i);
        br[i] = fetch<VEC>(a.residual, row, a.residual_dtype, c, i);
      }
    }
    float rstd1 = 1.f;
    if (a.post_weight) {
      float ss = 0.f;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        float x[8];
        values(bx[i], a.io_dtype, x);
#pragma unroll
        for (int j = 0; j < 8; ++j) ss = fmaf(x[j], x[j], ss);
      }
      rstd1 = rsqrtf(fmaf(sum(ss), inv, a.eps));
    }
    float r[NV][8], ss = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float x[8], wp[8], s[8];
      values(bx[i], a.io_dtype, x);
      values(br[i], a.residual_dtype, r[i]);
      param8<VEC>(a.post_weight, a.post_dtype, 1.f, c, i, wp);
      param8<VEC>(a.scale, a.scale_dtype, a.scale_value, c, i, s);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        r[i][j] = fmaf(s[j], x[j] * rstd1 * wp[j], r[i][j]);
        if (!(c.any(i) && c.has(i, j))) r[i][j] = 0.f;
        ss = fmaf(r[i][j], r[i][j], ss);
      }
    }
    const float rstd = rsqrtf(fmaf(sum(ss), inv, a.eps));
    if (!there) continue;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float w[8];
      store8<VEC>(a.r, row, a.residual_dtype, c, i, r[i]);
      param8<VEC>(a.weight, a.weight_dtype, 1.f, c, i, w);
#pragma unroll
      for (int j = 0; j < 8; ++j) w[j] *= r[i][j] * rstd;
      store8<VEC>(a.y, row, a.io_dtype, c, i, w);
    }
  }
}

template <bool VEC, int NV, bool WIDE>
__global__ void __launch_bounds__(WIDE ? 512 : NORM_CTA) residual_bwd_kernel(const __grid_constant__ NormParams p) {
  __shared__ float part[2][32];
  const kda_norm_args& a = p.a;
  const Cols<VEC> c = my_cols<VEC, NV, WIDE>(p);
  RowSum<WIDE> sum{part, p.lanes};
  const float inv = 1.f / a.cols;
  long long row, step, last;
  my_rows<WIDE>(p, row, step, last);
  float acc[2][NV][8] = {};      // dw, A
  for (; row < last; row += step) {
    const bool there = row < a.rows;
    Bits bx[NV], br[NV], bdy[NV], bdr[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      bx[i] = br[i] = bdy[i] = bdr[i] = Bits{};
      if (there) {
        bx[i] = fetch<VEC>(a.x, row, a.io_dtype, c, i);
        br[i] = fetch<VEC>(a.residual, row, a.residual_dtype, c, i);
        if (a.dy) bdy[i] = fetch<VEC>(a.dy, row, a.io_dtype, c, i);
        if (a.dr) bdr[i] = fetch<VEC>(a.dr, row, a.residual_dtype, c, i);
      }
    }
    float rstd1 = 1.f;
    if (a.post_weight) {
      float ss = 0.f;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        float x[8];
        values(bx[i], a.io_dtype, x);
#pragma unroll
        for (int j = 0; j < 8; ++j) ss = fmaf(x[j], x[j], ss);
      }
      rstd1 = rsqrtf(fmaf(sum(ss), inv, a.eps));
    }
    float r[NV][8], ss = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float x[8], wp[8], s[8];
      values(bx[i], a.io_dtype, x);
      values(br[i], a.residual_dtype, r[i]);
      param8<VEC>(a.post_weight, a.post_dtype, 1.f, c, i, wp);
      param8<VEC>(a.scale, a.scale_dtype, a.scale_value, c, i, s);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        r[i][j] = fmaf(s[j], x[j] * rstd1 * wp[j], r[i][j]);
        if (!(c.any(i) && c.has(i, j))) r[i][j] = 0.f;
        ss = fmaf(r[i][j], r[i][j], ss);
      }
    }
    const float rstd = rsqrtf(fmaf(sum(ss), inv, a.eps));
    float t[NV][8], dot = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float w[8];
      values(bdy[i], a.io_dtype, t[i]);
      param8<VEC>(a.weight, a.weight_dtype, 1.f, c, i, w);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        r[i][j] *= rstd;
        acc[0][i][j] = there ? fmaf(t[i][j], r[i][j], acc[0][i][j]) : acc[0][i][j];
        t[i][j] *= w[j];
        dot = fmaf(t[i][j], r[i][j], dot);
      }
    }
    dot = sum(dot) * inv;
    float dn[NV][8], dot1 = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float x[8], wp[8], s[8], dr[8];
      values(bdr[i], a.residual_dtype, dr);
      values(bx[i], a.io_dtype, x);
      param8<VEC>(a.post_weight, a.post_dtype, 1.f, c, i, wp);
      param8<VEC>(a.scale, a.scale_dtype, a.scale_value, c, i, s);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        t[i][j] = fmaf(rstd, fmaf(-dot, r[i][j], t[i][j]), dr[j]);
        const float n1 = x[j] * rstd1, db = s[j] * t[i][j];
        acc[1][i][j] = there ? fmaf(t[i][j], n1, acc[1][i][j]) : acc[1][i][j];
        dn[i][j] = db * wp[j];
        dot1 = fmaf(dn[i][j], n1, dot1);
      }
      if (there && a.dresidual) store8<VEC>(a.dresidual, row, a.residual_dtype, c, i, t[i]);
    }
    if (a.post_weight) {
      dot1 = sum(dot1) * inv;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        float x[8];
        values(bx[i], a.io_dtype, x);
#pragma unroll
        for (int j = 0; j < 8; ++j) dn[i][j] = rstd1 * fmaf(-dot1, x[j] * rstd1, dn[i][j]);
      }
    }
    if (!there) continue;
#pragma unroll
    for (int i = 0; i < NV; ++i) store8<VEC>(a.dx, row, a.io_dtype, c, i, dn[i]);
  }
  if (p.partial) leave_sums<VEC, NV, WIDE, 2>(p, c, acc);
}

// ---- the CTAs' partial sums, in their order: 32 columns and 32 runs of CTAs per block --------------------------------------------------------------
struct SumParams {
  kda_norm_args a;
  const float* partial;
  int ctas, sums;
};
__global__ void __launch_bounds__(1024) norm_sums_kernel(const __grid_constant__ SumParams p) {
  __shared__ float m[32][33];
  const kda_norm_args& a = p.a;
  const int s = blockIdx.y, lane = threadIdx.x & 31, run = threadIdx.x >> 5, col = blockIdx.x * 32 + lane;
  float x = 0.f;
  if (col < a.cols)
    for (int b = run; b < p.ctas; b += 32) x += p.partial[(static_cast<size_t>(b) * p.sums + s) * a.cols + col];
  m[run][lane] = x;
  __syncthreads();
  if (run != 0 || col >= a.cols) return;
  x = 0.f;
  for (int r = 0; r < 32; ++r) x += m[r][lane];
  auto leave = [&](void* out, int dtype, float y) {
    if (!out) return;
    if (dtype == KDA_BF16) static_cast<__nv_bfloat16*>(out)[col] = __float2bfloat16_rn(y);
    else static_cast<float*>(out)[col] = y;
  };
  if (s == 0) leave(a.dweight, a.weight_dtype, x);
  else {
    leave(a.dpost_weight, a.post_dtype, x * (a.scale ? load_raw(a.scale, col, a.scale_dtype) : a.scale_value));
    leave(a.dscale, a.scale_dtype, x * (a.post_weight ? load_raw(a.post_weight, col, a.post_dtype) : 1.f));
  }
}

// ---- launches ------------------------------------------------------------------------------------------------------------------------------------
struct Shape { int nv, threads, lanes, per; bool wide; };      // vectors per thread, threads and rows of a CTA
Shape shape_of(int cols) {
  Shape s{};
  s.wide = cols > NARROW;
  if (s.wide) {
    s.nv = cols <= 4096 ? 1 : 2;
    s.threads = ((cols + 8 * s.nv - 1) / (8 * s.nv) + 31) / 32 * 32;
    s.per = 1;
  } else {
    s.nv = 1;
    s.threads = NORM_CTA;
    for (s.lanes = 1; s.lanes * 8 < cols; s.lanes *= 2) {}
    s.per = NORM_CTA / s.lanes;
  }
  return s;
}
// CTAs of a backward: as many as the device holds at a time (their number is part of the order of the sums, so it depends on the sizes alone)
int bwd_ctas(int64_t rows, const Shape& s) { return static_cast<int>(std::min<int64_t>((rows + s.per - 1) / s.per, static_cast<int64_t>(sm_count()) * std::max(1, 1024 / s.threads))); }

template <class F>
int with_shape(const Shape& s, bool vec, F&& f) {
#define KDA_NORM(V, N, W) return f(std::integral_constant<bool, V>{}, std::integral_constant<int, N>{}, std::integral_constant<bool, W>{})
  if (vec) {
    if (!s.wide) KDA_NORM(true, 1, false);
    if (s.nv == 1) KDA_NORM(true, 1, true);
    KDA_NORM(true, 2, true);
  }
  if (!s.wide) KDA_NORM(false, 1, false);
  if (s.nv == 1) KDA_NORM(false, 1, true);
  KDA_NORM(false, 2, true);
#undef KDA_NORM
}

bool known(int dtype) { return dtype == KDA_BF16 || dtype == KDA_FP32; }
DeviceOnce g_norm_once;

int check_norm(const kda_norm_args& a, bool gated, bool backward) {
  if (a.rows < 0 || a.cols <= 0 || a.rows > (1LL << 40)) return KDA_E_SHAPE;
  if (a.cols > NORM_MOST) return KDA_E_LIMIT;
  if (!known(a.io_dtype) || !known(gated ? a.gate_dtype : a.residual_dtype) || (a.weight && !known(a.weight_dtype)) || (a.post_weight && !known(a.post_dtype)) ||
      (a.scale && !known(a.scale_dtype)))
    return KDA_E_DTYPE;
  if (gated && a.activation != KDA_ACT_SIGMOID && a.activation != KDA_ACT_SILU) return KDA_E_SHAPE;
  if (a.rows == 0) return KDA_OK;
  if (!a.x || (gated ? !a.gate : (!a.residual || !a.weight))) return KDA_E_NULL;
  if (!backward && (!a.y || (!gated && !a.r))) return KDA_E_NULL;
  if (backward && (!a.dx || (gated ? (!a.dy || !a.dgate) : (!a.dy && !a.dr)))) return KDA_E_NULL;
  // elements at their natural boundary at least (16 bytes: the wide forms)
  uintptr_t bf = 0, fp = 0;
  for (const auto& [p, dtype] : {std::pair<const void*, int>{a.x, a.io_dtype}, {a.y, a.io_dtype}, {a.dy, a.io_dtype}, {a.dx, a.io_dtype}, {a.gate, a.gate_dtype}, {a.dgate, a.gate_dtype},
                                 {a.residual, a.residual_dtype}, {a.r, a.residual_dtype}, {a.dr, a.residual_dtype}, {a.dresidual, a.residual_dtype}, {a.weight, a.weight_dtype},
                                 {a.dweight, a.weight_dtype}, {a.post_weight, a.post_dtype}, {a.dpost_weight, a.post_dtype}, {a.scale, a.scale_dtype}, {a.dscale, a.scale_dtype}})
    (dtype == KDA_BF16 ? bf : fp) |= reinterpret_cast<uintptr_t>(p);
  if ((bf & 1u) || (fp & 3u)) return KDA_E_ALIGN;
  if (backward && (a.dweight || a.dpost_weight || a.dscale)) {
    if (!a.workspace) return KDA_E_NULL;
    if (reinterpret_cast<uintptr_t>(a.workspace) & 15u) return KDA_E_ALIGN;
    if (a.workspace_bytes < kda_norm_bwd_workspace_bytes(a.rows, a.cols, gated ? 1 : 2)) return KDA_E_WORKSPACE;
  }
  return KDA_OK;
}
int run_norm(const kda_norm_args& a, bool gated, bool backward, cudaStream_t st) {
  int rc = check_norm(a, gated, backward);
  if (rc != KDA_OK) return rc;
  if ((rc = g_norm_once.run([] { return cudaSuccess; })) != KDA_OK) return rc;
  const bool sums = backward && (a.dweight || a.dpost_weight || a.dscale);
  const Shape s = shape_of(a.cols);
  NormParams p{};
  p.a = a;
  p.lanes = s.lanes;
  p.partial = sums ? static_cast<float*>(a.workspace) : nullptr;
  int ctas = 0;
  if (a.rows > 0) {
    if (norm_ring_covers(a, gated, backward)) {
      if ((rc = norm_ring(a, gated, backward, p.partial, &ctas, st)) != KDA_OK) return rc;
    } else {
      const bool vec = a.cols % 8 == 0 && norm_aligned(a);
      ctas = backward ? bwd_ctas(a.rows, s) : static_cast<int>(std::min<int64_t>((a.rows + s.per - 1) / s.per, static_cast<int64_t>(sm_count()) * 64));
      rc = with_shape(s, vec, [&](auto V, auto N, auto W) {
        if (gated) {
          if (backward) gated_bwd_kernel<V.value, N.value, W.value><<<ctas, s.threads, 0, st>>>(p);
          else gated_fwd_kernel<V.value, N.value, W.value><<<ctas, s.threads, 0, st>>>(p);
        } else {
          if (backward) residual_bwd_kernel<V.value, N.value, W.value><<<ctas, s.threads, 0, st>>>(p);
          else residual_fwd_kernel<V.value, N.value, W.value><<<ctas, s.threads, 0, st>>>(p);
        }
        return static_cast<int>(cudaGetLastError());
      });
      if (rc != KDA_OK) return rc;
    }
  }
  if (!sums) return KDA_OK;
  const SumParams q{a, p.partial, ctas, gated ? 1 : 2};
  norm_sums_kernel<<<dim3((a.cols + 31) / 32, q.sums), 1024, 0, st>>>(q);
  return static_cast<int>(cudaGetLastError());
}

}  // namespace
}  // namespace kda

extern "C" size_t kda_norm_bwd_workspace_bytes(int64_t rows, int32_t cols, int32_t sums) {
  if (rows < 0 || cols <= 0 || cols > kda::NORM_MOST || sums < 1 || sums > 2) return 0;
  return std::max<size_t>(std::max(1, kda::bwd_ctas(rows, kda::shape_of(cols))), kda::norm_ring_partials()) * sums * cols * sizeof(float);
}
extern "C" int kda_norm_status(uint32_t* host_out) { return kda::norm_ring_status(host_out); }
extern "C" int kda_gated_norm_fwd(const kda_norm_args* a, void* st) { return a ? kda::run_norm(*a, true, false, static_cast<cudaStream_t>(st)) : KDA_E_NULL; }
extern "C" int kda_gated_norm_bwd(const kda_norm_args* a, void* st) { return a ? kda::run_norm(*a, true, true, static_cast<cudaStream_t>(st)) : KDA_E_NULL; }
extern "C" int kda_residual_norm_fwd(const kda_norm_args* a, void* st) { return a ? kda::run_norm(*a, false, false, static_cast<cudaStream_t>(st)) : KDA_E_NULL; }
extern "C" int kda_residual_norm_bwd(const kda_norm_args* a, void* st) { return a ? kda::run_norm(*a, false, true, static_cast<cudaStream_t>(st)) : KDA_E_NULL; }
