// The norms of kda_norm.cu for calls with many rows: whole rows travel through a ring of shared-memory stages by bulk copies, and the results leave from the
// places of the inputs that they replace (y and dx from x's, dgate from the gate's, r and dresidual from the residual's).
//
// Bound by HBM.  A thread that loads its columns, waits for the row's sums and stores keeps too few bytes under way: 32,768 x 4096 backward 904 us, 1,048,576 x 128
// backward 389, with half of HBM's rate.  Here one warp keeps 100 to 200 KB per SM coming and going whatever the others wait for.  Rows are copied as runs
// of bytes, so columns need not be a multiple of anything: a stage holds as many rows as make 16 bytes even.
#include <algorithm>

#include "kda_norm.cuh"

namespace kda {

namespace {

// Bit 0: a bounded wait on a stage gave up (the call's results are incomplete).
__device__ unsigned g_norm_status = 0;

constexpr int RING_MOST = 200 * 1024, STAGES_MOST = 4;

// The sum over a row's threads, in all of them.  More than a warp: through shared memory, in turns of two so that one barrier is enough.
struct GroupSum {
  float* part;      // [2][16] of this group
  int lanes, bar, turn = 0;
  __device__ __forceinline__ float operator()(float x) {
    if (lanes <= 32) {
      for (int o = lanes >> 1; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
      return x;
    }
    x = warp_sum(x);
    const int warps = lanes >> 5, warp = (threadIdx.x >> 5) % warps;
    if ((threadIdx.x & 31) == 0) part[16 * turn + warp] = x;
    asm volatile("bar.sync %0, %1;" ::"r"(bar), "r"(lanes) : "memory");
    x = 0.f;
    for (int w = 0; w < warps; ++w) x += part[16 * turn + w];
    turn ^= 1;
    return x;
  }
};

// vector i of a thread's columns in a row in shared memory
template <bool VEC>
__device__ __forceinline__ void get8(const unsigned char* row, int dtype, const Cols<VEC>& c, int i, float (&v)[8]) {
  if constexpr (VEC) {
    if (!c.any(i)) {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = 0.f;
      return;
    }
    Bits b;
    if (dtype == KDA_BF16) b.a = *reinterpret_cast<const uint4*>(row + 2 * c.at(i, 0));
    else {
      b.a = *reinterpret_cast<const uint4*>(row + 4 * c.at(i, 0));
      b.b = *reinterpret_cast<const uint4*>(row + 4 * c.at(i, 0) + 16);
    }
    values(b, dtype, v);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      v[j] = !c.has(i, j) ? 0.f : dtype == KDA_BF16 ? __bfloat162float(*reinterpret_cast<const __nv_bfloat16*>(row + 2 * c.at(i, j))) : *reinterpret_cast<const float*>(row + 4 * c.at(i, j));
  }
}
template <bool VEC>
__device__ __forceinline__ void put8(unsigned char* row, int dtype, const Cols<VEC>& c, int i, const float (&v)[8]) {
  if constexpr (VEC) {
    if (!c.any(i)) return;
    if (dtype == KDA_BF16) {
      *reinterpret_cast<uint4*>(row + 2 * c.at(i, 0)) = make_uint4(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7]));
    } else {
      *reinterpret_cast<float4*>(row + 4 * c.at(i, 0)) = make_float4(v[0], v[1], v[2], v[3]);
      *reinterpret_cast<float4*>(row + 4 * c.at(i, 0) + 16) = make_float4(v[4], v[5], v[6], v[7]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (c.has(i, j)) {
        if (dtype == KDA_BF16) *reinterpret_cast<__nv_bfloat16*>(row + 2 * c.at(i, j)) = __float2bfloat16_rn(v[j]);
        else *reinterpret_cast<float*>(row + 4 * c.at(i, j)) = v[j];
      }
  }
}

// A row of the gated norm.  x, z, d: the row of x, of the gate, of dy; results over x and z.
template <bool VEC, int NV, bool BWD>
__device__ __forceinline__ void gated_row(const kda_norm_args& a, const Cols<VEC>& c, GroupSum& sum, bool there, unsigned char* x_, unsigned char* z_, const unsigned char* d_,
                                          float (&acc)[3][NV][8]) {
  const float inv = 1.f / a.cols;
  float x[NV][8], ss = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    get8<VEC>(x_, a.io_dtype, c, i, x[i]);
#pragma unroll
    for (int j = 0; j < 8; ++j) ss = fmaf(x[i][j], x[i][j], ss);
  }
  const float rstd = rsqrtf(fmaf(sum(ss), inv, a.eps));
  if constexpr (!BWD) {
    if (!there) return;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float z[8], w[8];
      get8<VEC>(z_, a.gate_dtype, c, i, z);
      param8<VEC>(a.weight, a.weight_dtype, 1.f, c, i, w);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        float act, slope;
        act_of(z[j], a.activation, act, slope);
        z[j] = x[i][j] * rstd * w[j] * act;
      }
      put8<VEC>(x_, a.io_dtype, c, i, z);
    }
  } else {
    float dn[NV][8], dot = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float z[8], d[8], w[8];
      get8<VEC>(z_, a.gate_dtype, c, i, z);
      get8<VEC>(d_, a.io_dtype, c, i, d);
      param8<VEC>(a.weight, a.weight_dtype, 1.f, c, i, w);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        float act, slope;
        act_of(z[j], a.activation, act, slope);
        x[i][j] *= rstd;
        if (there) acc[0][i][j] = fmaf(d[j] * x[i][j], act, acc[0][i][j]);
        dn[i][j] = d[j] * w[j] * act;
        z[j] = d[j] * w[j] * x[i][j] * slope;
        dot = fmaf(dn[i][j], x[i][j], dot);
      }
      if (there) put8<VEC>(z_, a.gate_dtype, c, i, z);
    }
    dot = sum(dot) * inv;
    if (!there) return;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
#pragma unroll
      for (int j = 0; j < 8; ++j) dn[i][j] = rstd * fmaf(-dot, x[i][j], dn[i][j]);
      put8<VEC>(x_, a.io_dtype, c, i, dn[i]);
    }
  }
}

// A row of the residual norm.  x, r, dy, dr: the row of x, of the residual, of their gradients (or NULL); results over x and r.
template <bool VEC, int NV, bool BWD>
__device__ __forceinline__ void residual_row(const kda_norm_args& a, const Cols<VEC>& c, GroupSum& sum, bool there, unsigned char* x_, unsigned char* r_, const unsigned char* dy_,
                                             const unsigned char* dr_, float (&acc)[3][NV][8]) {
  const float inv = 1.f / a.cols;
  float x[NV][8], rstd1 = 1.f, ss = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i) get8<VEC>(x_, a.io_dtype, c, i, x[i]);
  if (a.post_weight) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) ss = fmaf(x[i][j], x[i][j], ss);
    rstd1 = rsqrtf(fmaf(sum(ss), inv, a.eps));
  }
  float r[NV][8];
  ss = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    float wp[8], s[8];
    get8<VEC>(r_, a.residual_dtype, c, i, r[i]);
    param8<VEC>(a.post_weight, a.post_dtype, 1.f, c, i, wp);
    param8<VEC>(a.scale, a.scale_dtype, a.scale_value, c, i, s);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      x[i][j] *= rstd1;
      r[i][j] = fmaf(s[j], x[i][j] * wp[j], r[i][j]);      // (columns that are not there: x and the residual read as zero)
      ss = fmaf(r[i][j], r[i][j], ss);
    }
  }
  const float rstd = rsqrtf(fmaf(sum(ss), inv, a.eps));
  if constexpr (!BWD) {
    if (!there) return;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float w[8];
      put8<VEC>(r_, a.residual_dtype, c, i, r[i]);
      param8<VEC>(a.weight, a.weight_dtype, 1.f, c, i, w);
#pragma unroll
      for (int j = 0; j < 8; ++j) w[j] *= r[i][j] * rstd;
      put8<VEC>(x_, a.io_dtype, c, i, w);
    }
  } else {
    float t[NV][8], dot = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float w[8];
      if (dy_) get8<VEC>(dy_, a.io_dtype, c, i, t[i]);
      else
#pragma unroll
        for (int j = 0; j < 8; ++j) t[i][j] = 0.f;
      param8<VEC>(a.weight, a.weight_dtype, 1.f, c, i, w);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        r[i][j] *= rstd;
        if (there) acc[0][i][j] = fmaf(t[i][j], r[i][j], acc[0][i][j]);
        t[i][j] *= w[j];
        dot = fmaf(t[i][j], r[i][j], dot);
      }
    }
    dot = sum(dot) * inv;
    float dot1 = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float wp[8], s[8], dr[8];
      if (dr_) get8<VEC>(dr_, a.residual_dtype, c, i, dr);
      else
#pragma unroll
        for (int j = 0; j < 8; ++j) dr[j] = 0.f;
      param8<VEC>(a.post_weight, a.post_dtype, 1.f, c, i, wp);
      param8<VEC>(a.scale, a.scale_dtype, a.scale_value, c, i, s);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        t[i][j] = fmaf(rstd, fmaf(-dot, r[i][j], t[i][j]), dr[j]);
        const float db = s[j] * t[i][j];
        if (there) {
          acc[1][i][j] = fmaf(db, x[i][j], acc[1][i][j]);
          acc[2][i][j] = fmaf(t[i][j], x[i][j] * wp[j], acc[2][i][j]);
        }
        r[i][j] = db * wp[j];      // (now the gradient of n1)
        dot1 = fmaf(r[i][j], x[i][j], dot1);
      }
      if (there) put8<VEC>(r_, a.residual_dtype, c, i, t[i]);
    }
    if (a.post_weight) {
      dot1 = sum(dot1) * inv;
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) r[i][j] = rstd1 * fmaf(-dot1, x[i][j], r[i][j]);
    }
    if (!there) return;
#pragma unroll
    for (int i = 0; i < NV; ++i) put8<VEC>(x_, a.io_dtype, c, i, r[i]);
  }
}

struct RingParams {
  kda_norm_args a;
  float* partial;                 // [CTAs * groups][sums][cols] or NULL
  int lanes, groups;              // threads of a row, rows at a time
  int rows, stages, stage_bytes;  // rows of a stage
  long long chunks;
  int n;                          // tensors that are read: x, gate or residual, dy, dr
  const void* in[4];
  void* out[2];                   // over the first and the second one
  int size[4], off[4];            // bytes of an element; where a stage has it
};

}  // namespace

template <bool GATED, bool VEC, int NV, bool BWD>
__global__ void __launch_bounds__(544, 1) norm_ring_kernel(const __grid_constant__ RingParams p) {
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ uint64_t full[STAGES_MOST], done[STAGES_MOST];
  __shared__ float part[16][32];
  const kda_norm_args& a = p.a;
  const int warps = (blockDim.x >> 5) - 1, warp = threadIdx.x >> 5;
  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES_MOST; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&done[s], warps);
    }
    fence_mbar_init();
  }
  __syncthreads();
  if (warp == warps) {
    // ================= copies =================
    if ((threadIdx.x & 31) == 0) {
      auto rows_of = [&](long long c) { return static_cast<int>(min(static_cast<long long>(p.rows), a.rows - c * p.rows)); };
      auto load = [&](long long c, int s) {
        unsigned char* const st = smem + s * p.stage_bytes;
        const int rows = rows_of(c);
        unsigned tx = 0;
        for (int i = 0; i < p.n; ++i) {
          const int bytes = rows * a.cols * p.size[i];
          const unsigned char* const src = static_cast<const unsigned char*>(p.in[i]) + static_cast<size_t>(c) * p.rows * a.cols * p.size[i];
          for (int b = bytes & ~15; b < bytes; b += 2)      // the end of the last rows: what is no 16 bytes
            *reinterpret_cast<unsigned short*>(st + p.off[i] + b) = *reinterpret_cast<const unsigned short*>(src + b);
          tx += bytes & ~15;
        }
        mbar_expect_tx(&full[s], tx);
        for (int i = 0; i < p.n; ++i) {
          const int bytes = rows * a.cols * p.size[i] & ~15;
          if (bytes) bulk_g2s(st + p.off[i], static_cast<const unsigned char*>(p.in[i]) + static_cast<size_t>(c) * p.rows * a.cols * p.size[i], bytes, &full[s]);
        }
      };
      auto store = [&](long long c, int s) {
        const unsigned char* const st = smem + s * p.stage_bytes;
        const int rows = rows_of(c);
        for (int i = 0; i < 2; ++i) {
          if (!p.out[i]) continue;
          const int bytes = rows * a.cols * p.size[i];
          unsigned char* const dst = static_cast<unsigned char*>(p.out[i]) + static_cast<size_t>(c) * p.rows * a.cols * p.size[i];
          if (bytes & ~15) bulk_s2g(dst, st + p.off[i], bytes & ~15);
          for (int b = bytes & ~15; b < bytes; b += 2) *reinterpret_cast<unsigned short*>(dst + b) = *reinterpret_cast<const unsigned short*>(st + p.off[i] + b);
        }
        bulk_commit();
      };
      // chunk k of this CTA is chunk blockIdx.x + k * gridDim.x, in stage k % stages
      const long long mine = blockIdx.x < p.chunks ? (p.chunks - blockIdx.x + gridDim.x - 1) / gridDim.x : 0;
      bool alive = true;
      for (long long k = 0; k < mine + p.stages; ++k) {
        const int s = static_cast<int>(k % p.stages);
        if (k >= p.stages && k - p.stages < mine) {
          if (!(alive = mbar_wait(&done[s], static_cast<unsigned>((k / p.stages - 1) & 1)))) break;
          store(blockIdx.x + (k - p.stages) * gridDim.x, s);
          if (k < mine) bulk_wait_read<0>();
        }
        if (k < mine) load(blockIdx.x + k * gridDim.x, s);
      }
      if (!alive) {      // loads may still be under way into this CTA's memory
        atomicOr(&g_norm_status, 1u);
        for (int s = 0; s < p.stages; ++s) mbar_drain(&full[s]);
      }
      bulk_wait_read<0>();
    }
    return;
  }
  const int group = threadIdx.x / p.lanes;
  const Cols<VEC> c{static_cast<int>(threadIdx.x) % p.lanes, p.lanes, a.cols};
  GroupSum sum{part[group & 15], p.lanes, 1 + (group & 15)};
  float acc[3][NV][8] = {};
  int k = 0;
  bool ok = true;
  for (long long ch = blockIdx.x; ch < p.chunks; ch += gridDim.x, ++k) {
    const int s = k % p.stages;
    if (!(ok = __all_sync(0xffffffffu, mbar_wait(&full[s], (k / p.stages) & 1)))) break;
    unsigned char* const st = smem + s * p.stage_bytes;
    const long long left = a.rows - ch * p.rows;
    for (int r = group; r < p.rows; r += p.groups) {      // the same number of turns for all of a warp
      const bool there = r < left;
      const int at = there ? r * a.cols : 0;
      if constexpr (GATED)
        gated_row<VEC, NV, BWD>(a, c, sum, there, st + p.off[0] + at * p.size[0], st + p.off[1] + at * p.size[1], BWD ? st + p.off[2] + at * p.size[2] : nullptr, acc);
      else
        residual_row<VEC, NV, BWD>(a, c, sum, there, st + p.off[0] + at * p.size[0], st + p.off[1] + at * p.size[1], BWD && a.dy ? st + p.off[2] + at * p.size[2] : nullptr,
                                   BWD && a.dr ? st + p.off[a.dy ? 3 : 2] + at * p.size[a.dy ? 3 : 2] : nullptr, acc);
    }
    fence_proxy_async();
    __syncwarp();
    if ((threadIdx.x & 31) == 0) mbar_arrive(&done[s]);
  }
  if (!ok && (threadIdx.x & 31) == 0) atomicOr(&g_norm_status, 1u);
  if (BWD && p.partial && ok) {
    constexpr int SUMS = GATED ? 1 : 3;
    float* const out = p.partial + static_cast<size_t>(blockIdx.x * p.groups + group) * SUMS * a.cols;
#pragma unroll
    for (int i = 0; i < SUMS; ++i)
#pragma unroll
      for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (c.any(v) && c.has(v, j)) out[i * a.cols + c.at(v, j)] = acc[i][v][j];
  }
}

int norm_ring_status(uint32_t* host_out) {
  if (!host_out) return KDA_E_NULL;
  unsigned v = 0, zero = 0;
  cudaError_t e = cudaMemcpyFromSymbol(&v, g_norm_status, sizeof(v));
  if (e == cudaSuccess && v) e = cudaMemcpyToSymbol(g_norm_status, &zero, sizeof(zero));
  *host_out = v;
  return static_cast<int>(e);
}

// How a call goes through the ring: false where its rows are too wide for two stages.
static bool plan(const kda_norm_args& a, bool gated, bool backward, RingParams& p) {
  auto size = [](int dtype) { return dtype == KDA_BF16 ? 2 : 4; };
  p.n = 0;
  auto add = [&](const void* t, int dtype) {
    p.in[p.n] = t;
    p.size[p.n++] = size(dtype);
  };
  add(a.x, a.io_dtype);
  add(gated ? a.gate : a.residual, gated ? a.gate_dtype : a.residual_dtype);
  if (backward && a.dy) add(a.dy, a.io_dtype);
  if (backward && !gated && a.dr) add(a.dr, a.residual_dtype);
  p.out[0] = backward ? a.dx : a.y;
  p.out[1] = backward ? (gated ? a.dgate : a.dresidual) : (gated ? nullptr : a.r);
  int per_row = 0, narrow = 4;
  for (int i = 0; i < p.n; ++i) {
    per_row += p.size[i] * a.cols;
    narrow = std::min(narrow, p.size[i]);
  }
  const int nv = a.cols <= 4096 ? 1 : 2, need = (a.cols + 8 * nv - 1) / (8 * nv);
  if (need <= 32) {
    for (p.lanes = 1; p.lanes < need; p.lanes *= 2) {}
    p.groups = 512 / p.lanes;
  } else {
    p.lanes = (need + 31) / 32 * 32;
    p.groups = 512 / p.lanes;
  }
  int even = 1;      // rows that make 16 bytes even
  while (even * a.cols * narrow % 16) even *= 2;
  const int step = std::max(even, p.groups);      // (both are powers of two, or groups is one of 1, 2, 3, 5 with even <= 8)
  const int unit = step % even ? step * even : step;
  p.rows = unit;
  while (p.rows * per_row < 24 * 1024 && (p.rows + unit) * per_row <= RING_MOST / 4) p.rows += unit;
  p.stage_bytes = 0;
  for (int i = 0; i < p.n; ++i) {
    p.off[i] = p.stage_bytes;
    p.stage_bytes += (p.rows * a.cols * p.size[i] + 127) / 128 * 128;
  }
  p.stages = std::min(STAGES_MOST, RING_MOST / p.stage_bytes);
  p.chunks = (a.rows + p.rows - 1) / p.rows;
  return p.stages >= 2;
}

static unsigned ring_ctas(const RingParams& p) { return static_cast<unsigned>(std::min<long long>(p.chunks, sm_count())); }

bool norm_ring_covers(const kda_norm_args& a, bool gated, bool backward) {
  if (a.rows * a.cols < NORM_RING_MIN || !norm_aligned(a)) return false;
  RingParams p{};
  return plan(a, gated, backward, p);
}
// the most partial sums of a call: groups never exceed 512, CTAs the SMs
size_t norm_ring_partials(int cols) {
  kda_norm_args a{};
  a.cols = cols;
  RingParams p{};
  plan(a, true, false, p);
  return static_cast<size_t>(sm_count()) * p.groups;
}

template <bool GATED, bool VEC, int NV, bool BWD>
static int launch_ring(const RingParams& p, cudaStream_t st) {
  static DeviceOnce once;
  const int rc = once.run([] { return cudaFuncSetAttribute(norm_ring_kernel<GATED, VEC, NV, BWD>, cudaFuncAttributeMaxDynamicSharedMemorySize, RING_MOST); });
  if (rc != KDA_OK) return rc;
  norm_ring_kernel<GATED, VEC, NV, BWD><<<ring_ctas(p), p.lanes * p.groups + 32, p.stages * p.stage_bytes, st>>>(p);
  return static_cast<int>(cudaGetLastError());
}

int norm_ring(const kda_norm_args& a, bool gated, bool backward, float* partial, int* partials, cudaStream_t st) {
  RingParams p{};
  if (!plan(a, gated, backward, p)) return KDA_E_SHAPE;
  p.a = a;
  p.partial = partial;
  *partials = static_cast<int>(ring_ctas(p)) * p.groups;
  const int which = (gated ? 8 : 0) + (a.cols % 8 == 0 ? 4 : 0) + (a.cols > 4096 ? 2 : 0) + (backward ? 1 : 0);
  switch (which) {
    case 0: return launch_ring<false, false, 1, false>(p, st);
    case 1: return launch_ring<false, false, 1, true>(p, st);
    case 2: return launch_ring<false, false, 2, false>(p, st);
    case 3: return launch_ring<false, false, 2, true>(p, st);
    case 4: return launch_ring<false, true, 1, false>(p, st);
    case 5: return launch_ring<false, true, 1, true>(p, st);
    case 6: return launch_ring<false, true, 2, false>(p, st);
    case 7: return launch_ring<false, true, 2, true>(p, st);
    case 8: return launch_ring<true, false, 1, false>(p, st);
    case 9: return launch_ring<true, false, 1, true>(p, st);
    case 10: return launch_ring<true, false, 2, false>(p, st);
    case 11: return launch_ring<true, false, 2, true>(p, st);
    case 12: return launch_ring<true, true, 1, false>(p, st);
    case 13: return launch_ring<true, true, 1, true>(p, st);
    case 14: return launch_ring<true, true, 2, false>(p, st);
    default: return launch_ring<true, true, 2, true>(p, st);
  }
}

}  // namespace kda
