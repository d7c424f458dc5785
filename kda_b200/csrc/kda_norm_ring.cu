// The norms of kda_norm.cu for calls with many rows: whole rows travel through a ring of shared-memory stages by bulk copies, and the results leave from the
// places of the inputs that they replace (y and dx from x's, dgate from the gate's, r and dresidual from the residual's).
//
// Bound by HBM.  A thread that loads its columns, waits for the row's sums and stores keeps too few bytes under way: 32,768 x 4096 backward 904 us, 1,048,576 x 128
// backward 389, with half of HBM's rate.  Here one warp keeps 100 to 200 KB per SM coming and going whatever the others wait for.  Rows are copied as runs
// of bytes, so columns need not be a multiple of anything: a stage holds as many rows as make 16 bytes even.
//   us, forward + backward: gated 1,048,576 x 128 124 + 207 (6.4 TB/s); residual 32,768 x 4096 with an fp32 residual and post weight 248 + 470 (6.5, 5.1 TB/s: the
//   backward's copies alone take 392, and the four sums of a row one after the other are not quite hidden behind them)
#include <algorithm>

#include "kda_norm.cuh"

#ifndef KDA_RING_VERDICT      // what a wait of the compute warps says; csrc/debug/kda_norm_ring_test.cu builds the kernel with waits that give up
#define KDA_RING_VERDICT(ok) (ok)
#define KDA_RING_ENTRY 1
#endif

namespace kda {

namespace {

// Bit 0: a bounded wait on a stage gave up (the call's results are incomplete).
__device__ unsigned g_norm_status = 0;

constexpr int RING_MOST = 224 * 1024, RING_STAGE = 32 * 1024, STAGES_LEAST = 4, STAGES_MOST = 6;

// The sum over a row's threads, in all of them.  More than a warp: through shared memory, in turns of two so that one barrier is enough.
struct GroupSum {
  float* part;      // [2][16] of this group
  int lanes, bar, warp, turn = 0;      // warp: of the row's
  __device__ __forceinline__ float operator()(float x) {
    if (lanes <= 32) {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1)
        if (lanes > o) x += __shfl_xor_sync(0xffffffffu, x, o);
      return x;
    }
    x = warp_sum(x);
    float* const p = part + 16 * turn;      // (places of warps that there are not hold zeros)
    if ((threadIdx.x & 31) == 0) p[warp] = x;
    asm volatile("bar.sync %0, %1;" ::"r"(bar), "r"(lanes) : "memory");
    const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
    x = (a.x + a.y) + (a.z + a.w) + ((b.x + b.y) + (b.z + b.w));
    if (lanes > 256) {
      const float4 c = *reinterpret_cast<const float4*>(p + 8), d = *reinterpret_cast<const float4*>(p + 12);
      x += (c.x + c.y) + (c.z + c.w) + ((d.x + d.y) + (d.z + d.w));
    }
    turn ^= 1;
    return x;
  }
};

// vector i of a thread's columns in a row in shared memory, of type T (KDA_BF16 or KDA_FP32)
template <int T, bool VEC>
__device__ __forceinline__ void get8(const unsigned char* row, const Cols<VEC>& c, int i, float (&v)[8]) {
  if constexpr (VEC) {
    Bits b{make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
    if (c.any(i)) {
      if constexpr (T == KDA_BF16) b.a = *reinterpret_cast<const uint4*>(row + 2 * c.at(i, 0));
      else {
        b.a = *reinterpret_cast<const uint4*>(row + 4 * c.at(i, 0));
        b.b = *reinterpret_cast<const uint4*>(row + 4 * c.at(i, 0) + 16);
      }
    }
    values(b, T, v);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      v[j] = 0.f;
      if (c.has(i, j)) {
        if constexpr (T == KDA_BF16) v[j] = __bfloat162float(*reinterpret_cast<const __nv_bfloat16*>(row + 2 * c.at(i, j)));
        else v[j] = *reinterpret_cast<const float*>(row + 4 * c.at(i, j));
      }
    }
  }
}
template <int T, bool VEC>
__device__ __forceinline__ void put8(unsigned char* row, const Cols<VEC>& c, int i, const float (&v)[8]) {
  if constexpr (VEC) {
    if (!c.any(i)) return;
    if constexpr (T == KDA_BF16) {
      *reinterpret_cast<uint4*>(row + 2 * c.at(i, 0)) = make_uint4(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7]));
    } else {
      *reinterpret_cast<float4*>(row + 4 * c.at(i, 0)) = make_float4(v[0], v[1], v[2], v[3]);
      *reinterpret_cast<float4*>(row + 4 * c.at(i, 0) + 16) = make_float4(v[4], v[5], v[6], v[7]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (c.has(i, j)) {
        if constexpr (T == KDA_BF16) *reinterpret_cast<__nv_bfloat16*>(row + 2 * c.at(i, j)) = __float2bfloat16_rn(v[j]);
        else *reinterpret_cast<float*>(row + 4 * c.at(i, j)) = v[j];
      }
  }
}
// A parameter in shared memory, as fp32.  VEC: the first four of every eight columns, then the others, so that neighbours read neighbouring 16 bytes.
template <bool VEC>
__device__ __forceinline__ int param_at(int col, int cols) { return VEC ? ((col & 4) ? cols / 2 : 0) + (col >> 3) * 4 + (col & 3) : col; }
template <bool VEC>
__device__ __forceinline__ void get_param(const float* p, const Cols<VEC>& c, int i, float (&v)[8]) {
  if constexpr (VEC) {
    const float* const q = p + (c.any(i) ? c.at(i, 0) / 2 : 0);
    const float4 a = *reinterpret_cast<const float4*>(q), b = *reinterpret_cast<const float4*>(q + c.cols / 2);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = c.has(i, j) ? p[c.at(i, j)] : 0.f;
  }
}

// A row of the gated norm.  x, z, d: the row of x, of the gate, of dy; results over x and z.
template <int XT, int ZT, bool VEC, bool BWD, int NV>
__device__ __forceinline__ void gated_row(const kda_norm_args& a, const float* w_, const Cols<VEC>& c, GroupSum& sum, bool there, unsigned char* x_, unsigned char* z_,
                                          const unsigned char* d_, float (&acc)[2][NV][8]) {
  const float inv = 1.f / a.cols;
  float x[NV][8], ss = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    get8<XT, VEC>(x_, c, i, x[i]);
#pragma unroll
    for (int j = 0; j < 8; ++j) ss = fmaf(x[i][j], x[i][j], ss);
  }
  const float rstd = rsqrtf(fmaf(sum(ss), inv, a.eps));
  if constexpr (!BWD) {
    if (!there) return;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float z[8], w[8];
      get8<ZT, VEC>(z_, c, i, z);
      get_param<VEC>(w_, c, i, w);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        float act, slope;
        act_of<XT == KDA_FP32>(z[j], a.activation, act, slope);
        z[j] = x[i][j] * rstd * w[j] * act;
      }
      put8<XT, VEC>(x_, c, i, z);
    }
  } else {
    float dn[NV][8], dot = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float z[8], d[8], w[8];
      get8<ZT, VEC>(z_, c, i, z);
      get8<XT, VEC>(d_, c, i, d);
      get_param<VEC>(w_, c, i, w);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        float act, slope;
        act_of<XT == KDA_FP32>(z[j], a.activation, act, slope);
        x[i][j] *= rstd;
        const float da = d[j] * act, dx = d[j] * x[i][j] * w[j];
        if (there) acc[0][i][j] = fmaf(da, x[i][j], acc[0][i][j]);
        dn[i][j] = da * w[j];
        dot = fmaf(dn[i][j], x[i][j], dot);
        z[j] = dx * slope;
      }
      if (there) put8<ZT, VEC>(z_, c, i, z);
    }
    dot = sum(dot) * inv;
    if (!there) return;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
#pragma unroll
      for (int j = 0; j < 8; ++j) dn[i][j] = rstd * fmaf(-dot, x[i][j], dn[i][j]);
      put8<XT, VEC>(x_, c, i, dn[i]);
    }
  }
}

// A row of the residual norm.  x, r, dy, dr: the row of x, of the residual, of their gradients (or NULL); results over x and r.  sw: scale times post_weight.
template <int XT, int RT, bool VEC, bool BWD, int NV, bool ROOMY>
__device__ __forceinline__ void residual_row(const kda_norm_args& a, const float* w_, const float* sw_, const Cols<VEC>& c, GroupSum& sum, bool there, unsigned char* x_,
                                             unsigned char* r_, const unsigned char* dy_, const unsigned char* dr_, float (&acc)[2][NV][8], const float (&wr)[ROOMY ? NV : 1][8],
                                             const float (&swr)[ROOMY ? NV : 1][8]) {
  const float inv = 1.f / a.cols;
  float rstd1 = 1.f, ss = 0.f;
  // ROOMY: x and the parameters stay in registers.  Elsewhere x is read from shared memory wherever it is needed: with it, r, t and the sums over rows in
  // registers the backward spilled, into an L1 that the ring leaves little of (32,768 x 4096: 596 us)
  float xs[ROOMY ? NV : 1][8];
  if constexpr (ROOMY) {
#pragma unroll
    for (int i = 0; i < NV; ++i) get8<XT, VEC>(x_, c, i, xs[i]);
  }
  auto raw = [&](int i, float (&x)[8]) {
    if constexpr (ROOMY) {
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = xs[i][j];
    } else get8<XT, VEC>(x_, c, i, x);
  };
  auto n1 = [&](int i, float (&x)[8]) {
    raw(i, x);
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] *= rstd1;
  };
  auto param = [&](const float* p, const float (&kept)[ROOMY ? NV : 1][8], int i, float (&v)[8]) {
    if constexpr (ROOMY) {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = kept[i][j];
    } else get_param<VEC>(p, c, i, v);
  };
  if (a.post_weight) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float x[8];
      raw(i, x);
#pragma unroll
      for (int j = 0; j < 8; ++j) ss = fmaf(x[j], x[j], ss);
    }
    rstd1 = rsqrtf(fmaf(sum(ss), inv, a.eps));
  }
  float r[NV][8];
  ss = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    float x[8], sw[8];
    n1(i, x);
    get8<RT, VEC>(r_, c, i, r[i]);
    param(sw_, swr, i, sw);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      r[i][j] = fmaf(sw[j], x[j], r[i][j]);      // (columns that are not there: x and the residual read as zero)
      ss = fmaf(r[i][j], r[i][j], ss);
    }
  }
  const float rstd = rsqrtf(fmaf(sum(ss), inv, a.eps));
  if constexpr (!BWD) {
    if (!there) return;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float w[8];
      put8<RT, VEC>(r_, c, i, r[i]);
      param(w_, wr, i, w);
#pragma unroll
      for (int j = 0; j < 8; ++j) w[j] *= r[i][j] * rstd;
      put8<XT, VEC>(x_, c, i, w);
    }
  } else {
    float t[NV][8], dot = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float w[8];
      if (dy_) get8<XT, VEC>(dy_, c, i, t[i]);
      else
#pragma unroll
        for (int j = 0; j < 8; ++j) t[i][j] = 0.f;
      param(w_, wr, i, w);
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
      float x[8], sw[8], dr[8];
      n1(i, x);
      if (dr_) get8<RT, VEC>(dr_, c, i, dr);
      else
#pragma unroll
        for (int j = 0; j < 8; ++j) dr[j] = 0.f;
      param(sw_, swr, i, sw);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        t[i][j] = fmaf(rstd, fmaf(-dot, r[i][j], t[i][j]), dr[j]);
        if (there) acc[1][i][j] = fmaf(t[i][j], x[j], acc[1][i][j]);
        r[i][j] = sw[j] * t[i][j];      // (now the gradient of n1)
        dot1 = fmaf(r[i][j], x[j], dot1);
      }
      if (there) put8<RT, VEC>(r_, c, i, t[i]);
    }
    if (a.post_weight) {
      dot1 = sum(dot1) * inv;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        float x[8];
        n1(i, x);
#pragma unroll
        for (int j = 0; j < 8; ++j) r[i][j] = rstd1 * fmaf(-dot1, x[j], r[i][j]);
      }
    }
    if (!there) return;
#pragma unroll
    for (int i = 0; i < NV; ++i) put8<XT, VEC>(x_, c, i, r[i]);
  }
}

struct RingParams {
  kda_norm_args a;
  float* partial;                 // [CTAs][sums][cols] or NULL
  int lanes, groups;              // threads of a row, rows at a time
  int params;                     // bytes of the parameters in front of the stages
  int rows, stages, stage_bytes;  // rows of a stage
  long long chunks;
  const void* in[4];              // x; gate or residual; dy; dr (NULL: not read)
  void* out[2];                   // over the first and the second one
  int size[4], off[4];            // bytes of an element; where a stage has it
};

}  // namespace

// A wait gave up in chunk `ch`: this warp frees no stage any more, so that the copies and the other warps' waits come to their end too.  Until then, and beyond, the other warps
// of its row meet it in the row's barriers: it goes on taking part in them, once for every sum of every row that is left.  (Not inlined: the rows' code has no register to spare;
// inlined, 1,048,576 x 128 took 127.5 + 209 us instead of 124 + 206.5.)
__device__ __noinline__ void meet_others(const RingParams& p, long long ch, int next, int bar, int sums) {
  for (; ch < p.chunks; ch += gridDim.x) {
    int r = next;
    for (; r < p.rows; r += p.groups)
      for (int i = 0; i < sums; ++i) asm volatile("bar.sync %0, %1;" ::"r"(bar), "r"(p.lanes) : "memory");
    next = r - p.rows;
  }
}

// ROOMY (the residual norm's backward): half the threads, with registers for all of a row that they need more than once.
template <bool GATED, int XT, int ZT, bool VEC, bool BWD, int NV, bool ROOMY>
__global__ void __launch_bounds__(ROOMY ? 288 : 544, 1) norm_ring_kernel(const __grid_constant__ RingParams p) {
  extern __shared__ __align__(128) unsigned char smem_raw[];
  __shared__ uint64_t full[STAGES_MOST], done[STAGES_MOST];
  __shared__ __align__(16) float part[16][32];
  const kda_norm_args& a = p.a;
  const int warps = (blockDim.x >> 5) - 1, warp = threadIdx.x >> 5;
  float* const w_ = reinterpret_cast<float*>(smem_raw);
  float* const sw_ = w_ + a.cols;
  unsigned char* const smem = smem_raw + p.params;
  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES_MOST; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&done[s], warps);
    }
    fence_mbar_init();
  }
  for (int e = threadIdx.x; e < 16 * 32; e += blockDim.x) part[e / 32][e % 32] = 0.f;
  for (int e = threadIdx.x; e < a.cols; e += blockDim.x) {
    w_[param_at<VEC>(e, a.cols)] = a.weight ? load_raw(a.weight, e, a.weight_dtype) : 1.f;
    if constexpr (!GATED)
      sw_[param_at<VEC>(e, a.cols)] = (a.scale ? load_raw(a.scale, e, a.scale_dtype) : a.scale_value) * (a.post_weight ? load_raw(a.post_weight, e, a.post_dtype) : 1.f);
  }
  __syncthreads();
  if (warp == warps) {
    // ================= copies =================
    if ((threadIdx.x & 31) == 0) {
      // one chunk per stage and turn, some hundred cycles each: sizes of whole chunks are known ahead, and the last one takes its own way
      unsigned whole[4], tx = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        whole[i] = p.in[i] ? static_cast<unsigned>(p.rows * a.cols * p.size[i]) : 0;
        tx += whole[i];
      }
      const int last_rows = static_cast<int>(a.rows - (p.chunks - 1) * p.rows);
      auto load = [&](long long c, int s) {
        unsigned char* const st = smem + s * p.stage_bytes;
        if (c + 1 < p.chunks) {
          mbar_expect_tx(&full[s], tx);
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (p.in[i]) bulk_g2s(st + p.off[i], static_cast<const unsigned char*>(p.in[i]) + static_cast<size_t>(c) * whole[i], whole[i], &full[s]);
          return;
        }
        unsigned even = 0;
        for (int i = 0; i < 4; ++i) {
          if (!p.in[i]) continue;
          const int bytes = last_rows * a.cols * p.size[i];
          const unsigned char* const src = static_cast<const unsigned char*>(p.in[i]) + static_cast<size_t>(c) * whole[i];
          for (int b = bytes & ~15; b < bytes; b += 2)      // the end of the last rows: what is no 16 bytes
            *reinterpret_cast<unsigned short*>(st + p.off[i] + b) = *reinterpret_cast<const unsigned short*>(src + b);
          even += bytes & ~15;
        }
        mbar_expect_tx(&full[s], even);
        for (int i = 0; i < 4; ++i) {
          const int bytes = last_rows * a.cols * p.size[i] & ~15;
          if (p.in[i] && bytes) bulk_g2s(st + p.off[i], static_cast<const unsigned char*>(p.in[i]) + static_cast<size_t>(c) * whole[i], bytes, &full[s]);
        }
      };
      auto store = [&](long long c, int s) {
        const unsigned char* const st = smem + s * p.stage_bytes;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          if (!p.out[i]) continue;
          const int bytes = c + 1 < p.chunks ? static_cast<int>(whole[i]) : last_rows * a.cols * p.size[i];
          unsigned char* const dst = static_cast<unsigned char*>(p.out[i]) + static_cast<size_t>(c) * whole[i];
          if (bytes & ~15) bulk_s2g(dst, st + p.off[i], bytes & ~15);
          for (int b = bytes & ~15; b < bytes; b += 2) *reinterpret_cast<unsigned short*>(dst + b) = *reinterpret_cast<const unsigned short*>(st + p.off[i] + b);
        }
        bulk_commit();
      };
      // the CTA's chunks are blockIdx.x, blockIdx.x + gridDim.x, ..; they take the stages in turn
      bool alive = true;
      long long ahead = blockIdx.x;
      for (int s = 0; s < p.stages && ahead < p.chunks; ++s, ahead += gridDim.x) load(ahead, s);
      int s = 0;
      unsigned turn = 0;
      for (long long c = blockIdx.x; c < p.chunks; c += gridDim.x) {
        if (!(alive = mbar_wait(&done[s], turn))) break;
        store(c, s);
        if (c != blockIdx.x && ahead < p.chunks) {      // into the stage before, whose store has had a turn's time to read it
          bulk_wait_read<1>();
          load(ahead, s == 0 ? p.stages - 1 : s - 1);
          ahead += gridDim.x;
        }
        if (++s == p.stages) {
          s = 0;
          turn ^= 1u;
        }
      }
      if (!alive) {      // loads may still be under way into this CTA's memory
        atomicOr(&g_norm_status, 1u);
        for (int i = 0; i < p.stages; ++i) mbar_drain(&full[i]);
      }
      bulk_wait_read<0>();
    }
    __syncwarp();
    if (BWD && p.partial && p.groups > 1) asm volatile("bar.arrive 15, %0;" ::"r"(blockDim.x) : "memory");      // the stages are free
    return;
  }
  const int group = threadIdx.x / p.lanes;
  const Cols<VEC> c{static_cast<int>(threadIdx.x) % p.lanes, p.lanes, a.cols};
  GroupSum sum{part[group & 15], p.lanes, 1 + (group & 15), c.lane >> 5};
  float acc[2][NV][8] = {}, wr[ROOMY ? NV : 1][8], swr[ROOMY ? NV : 1][8];
  if constexpr (ROOMY) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      get_param<VEC>(w_, c, i, wr[i]);
      get_param<VEC>(sw_, c, i, swr[i]);
    }
  }
  constexpr int XS = XT == KDA_BF16 ? 2 : 4, ZS = ZT == KDA_BF16 ? 2 : 4;
  int k = 0, s = 0, next = group;      // next: this group's next row of the stage
  bool ok = true;
  long long ch = blockIdx.x;
  for (; ch < p.chunks; ch += gridDim.x) {
    if (!(ok = __all_sync(0xffffffffu, KDA_RING_VERDICT(mbar_wait(&full[s], k & 1))))) break;
    unsigned char* const st = smem + s * p.stage_bytes;
    const long long left = a.rows - ch * p.rows;
    int r = next;
    for (; r < p.rows; r += p.groups) {      // (groups that share a warp take the same number of turns)
      const bool there = r < left;
      const int at = there ? r * a.cols : 0;
      if constexpr (GATED)
        gated_row<XT, ZT, VEC, BWD, NV>(a, w_, c, sum, there, st + p.off[0] + at * XS, st + p.off[1] + at * ZS, st + p.off[2] + at * XS, acc);
      else
        residual_row<XT, ZT, VEC, BWD, NV, ROOMY>(a, w_, sw_, c, sum, there, st + p.off[0] + at * XS, st + p.off[1] + at * ZS, a.dy ? st + p.off[2] + at * XS : nullptr,
                                       a.dr ? st + p.off[3] + at * ZS : nullptr, acc, wr, swr);
    }
    next = r - p.rows;
    fence_proxy_async();
    __syncwarp();
    if ((threadIdx.x & 31) == 0) mbar_arrive(&done[s]);
    if (++s == p.stages) {
      s = 0;
      ++k;
    }
  }
  if (!ok) {
    if ((threadIdx.x & 31) == 0) atomicOr(&g_norm_status, 1u);
    if (p.lanes > 32) meet_others(p, ch, next, sum.bar, (BWD ? 2 : 1) * (!GATED && a.post_weight ? 2 : 1));
  }
  if (BWD && p.partial) {
    constexpr int SUMS = GATED ? 1 : 2;
    float* const out = p.partial + static_cast<size_t>(blockIdx.x) * SUMS * a.cols;
    // the groups' sums meet in the stages' place (a partial sum per group: 1,048,576 x 128 has 4,736 of them, and joining those took 30 us)
    float* const mine = p.groups > 1 ? reinterpret_cast<float*>(smem) + group * SUMS * a.cols : out;
    if (p.groups > 1) asm volatile("bar.sync 15, %0;" ::"r"(blockDim.x) : "memory");
#pragma unroll
    for (int i = 0; i < SUMS; ++i)
#pragma unroll
      for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (c.any(v) && c.has(v, j)) mine[i * a.cols + c.at(v, j)] = acc[i][v][j];
    if (p.groups > 1) {
      const int threads = blockDim.x - 32;
      asm volatile("bar.sync 14, %0;" ::"r"(threads) : "memory");
      for (int e = threadIdx.x; e < SUMS * a.cols; e += threads) {
        float x = 0.f;
        for (int g = 0; g < p.groups; ++g) x += reinterpret_cast<const float*>(smem)[g * SUMS * a.cols + e];
        out[e] = x;
      }
    }
  }
}

int norm_ring_status(uint32_t* host_out) {
  if (!host_out) return KDA_E_NULL;
  unsigned v = 0, zero = 0;
  cudaError_t e = cudaDeviceSynchronize();      // (a copy alone waits for the default stream, not for those of torch)
  if (e == cudaSuccess) e = cudaMemcpyFromSymbol(&v, g_norm_status, sizeof(v));
  if (e == cudaSuccess && v) e = cudaMemcpyToSymbol(g_norm_status, &zero, sizeof(zero));
  *host_out = v;
  return static_cast<int>(e);
}

// threads of a row and rows at a time
static void split(int cols, int nv, int threads, int& lanes, int& groups) {
  const int need = (cols + 8 * nv - 1) / (8 * nv);
  for (lanes = 1; lanes < need && lanes < 32; lanes *= 2) {}
  if (need > 32) lanes = (need + 31) / 32 * 32;
  groups = threads / lanes;
}
// Vectors of eight columns per thread.  Two: what a thread does once a row (sums over it, addresses) it does for sixteen columns.  The residual norm's backward has
// sums over rows, r and t in registers besides: one, where a row's threads allow it; or, with a norm of x to go back through and whole vectors, two with half the
// threads (ROOMY), if these come to 200.  us, 2^26 elements with an fp32 residual, one | ROOMY: 128 columns 214 | 203, 512 261 | 221, 1,024 258 | 242, 4,096 279 | 253; with
// two and 512 threads 4,096 took 300, spilling into an L1 that the ring leaves little of.  On the other side, without post_weight (bf16): 1,024 173 | 178; columns one by
// one: 1,001 456 | 501; 160 threads: 2,500 474 | 610.
struct Form { int nv; bool roomy; };
static Form form(const kda_norm_args& a, bool gated, bool backward) {
  if (gated || !backward || a.cols > 4096) return {2, false};
  int lanes, groups;
  split(a.cols, 2, 256, lanes, groups);
  return a.post_weight && a.cols % 8 == 0 && lanes * groups >= 200 ? Form{2, true} : Form{1, false};
}

// How a call goes through the ring: false where its rows are too wide for two stages.
static bool plan(const kda_norm_args& a, bool gated, bool backward, RingParams& p) {
  const int other = gated ? a.gate_dtype : a.residual_dtype;
  p.in[0] = a.x;
  p.in[1] = gated ? a.gate : a.residual;
  p.in[2] = backward ? a.dy : nullptr;
  p.in[3] = backward && !gated ? a.dr : nullptr;
  p.size[0] = p.size[2] = a.io_dtype == KDA_BF16 ? 2 : 4;
  p.size[1] = p.size[3] = other == KDA_BF16 ? 2 : 4;
  p.out[0] = backward ? a.dx : a.y;
  p.out[1] = backward ? (gated ? a.dgate : a.dresidual) : (gated ? nullptr : a.r);
  const Form f = form(a, gated, backward);
  split(a.cols, f.nv, f.roomy ? 256 : 512, p.lanes, p.groups);
  int per_row = 0;
  for (int i = 0; i < 4; ++i)
    if (p.in[i]) per_row += p.size[i] * a.cols;
  int even = 1;      // rows that make 16 bytes even
  while (even * a.cols * std::min(p.size[0], p.size[1]) % 16) even *= 2;
  p.params = (a.cols * (gated ? 4 : 8) + 127) / 128 * 128;
  // Bytes under way.  The gated norm: all that fit (1,048,576 x 128 forward, stages of 32 KB: four 131.6 us, five 126.5, six 124.4).  The residual norm, whose
  // forward writes as much as it reads: about 128 KB (32,768 x 4096 forward, fp32 residual: 120 KB 248 us, 144 276, 192 282; bf16 residual: 128 KB
  // 170, 160 KB 197).
  const int room = RING_MOST - p.params, most = gated ? room : std::min(room, 128 * 1024);
  // a row for every group in each stage; it has to be so where groups share a warp, elsewhere if all stages fit
  int unit = even;
  while (unit % p.groups) unit += even;
  if (p.lanes > 32 && static_cast<long long>(STAGES_LEAST) * unit * per_row > most) unit = even;
  p.rows = unit;
  while (p.rows * per_row < RING_STAGE && (p.rows + unit) * per_row <= most / STAGES_LEAST) p.rows += unit;
  p.stage_bytes = 0;
  for (int i = 0; i < 4; ++i) {
    p.off[i] = p.stage_bytes;
    if (p.in[i]) p.stage_bytes += (p.rows * a.cols * p.size[i] + 127) / 128 * 128;
  }
  p.stages = std::min({STAGES_MOST, room / std::max(1, p.stage_bytes), std::max(STAGES_LEAST, most / std::max(1, p.stage_bytes))});
  p.chunks = (a.rows + p.rows - 1) / p.rows;
  return p.stages >= 2 && (!backward || p.groups == 1 || p.groups * (gated ? 1 : 2) * a.cols * 4 <= p.stages * p.stage_bytes);
}

static unsigned ring_ctas(const RingParams& p) { return static_cast<unsigned>(std::min<long long>(p.chunks, sm_count())); }

// Float32 x with a bf16 gate goes straight from memory (us, 2^26 elements of 128 columns, ring | direct: forward 114 | 105, backward 274 | 176); with a bf16 residual it does not
// (4,096 columns: forward 138 | 179, backward with post_weight 254 | 448; 1,024: 140 | 136, 242 | 350).
bool norm_ring_covers(const kda_norm_args& a, bool gated, bool backward) {
  if (a.rows * a.cols < ring_min(backward) || !norm_aligned(a) || (gated && a.io_dtype == KDA_FP32 && a.gate_dtype == KDA_BF16)) return false;
  RingParams p{};
  return plan(a, gated, backward, p);
}
// the most partial sums of a call
size_t norm_ring_partials() { return static_cast<size_t>(sm_count()); }

template <bool GATED, int XT, int ZT, bool VEC, bool BWD, int NV, bool ROOMY>
static int launch_ring_nv(const RingParams& p, cudaStream_t st) {
  static DeviceOnce once;
  const int rc = once.run([] { return cudaFuncSetAttribute(norm_ring_kernel<GATED, XT, ZT, VEC, BWD, NV, ROOMY>, cudaFuncAttributeMaxDynamicSharedMemorySize, RING_MOST); });
  if (rc != KDA_OK) return rc;
  norm_ring_kernel<GATED, XT, ZT, VEC, BWD, NV, ROOMY><<<ring_ctas(p), p.lanes * p.groups + 32, p.params + p.stages * p.stage_bytes, st>>>(p);
  return static_cast<int>(cudaGetLastError());
}
template <bool GATED, int XT, int ZT, bool VEC, bool BWD>
static int launch_ring(const RingParams& p, cudaStream_t st) {
  if constexpr (BWD && !GATED) {
    const Form f = form(p.a, GATED, BWD);
    if constexpr (VEC) {
      if (f.roomy) return launch_ring_nv<GATED, XT, ZT, VEC, BWD, 2, true>(p, st);
    }
    if (f.nv == 1) return launch_ring_nv<GATED, XT, ZT, VEC, BWD, 1, false>(p, st);
  }
  return launch_ring_nv<GATED, XT, ZT, VEC, BWD, 2, false>(p, st);
}
#ifdef KDA_RING_ENTRY
template <bool GATED, int XT, int ZT>
static int launch_types(const RingParams& p, bool backward, cudaStream_t st) {
  if (p.a.cols % 8 == 0) return backward ? launch_ring<GATED, XT, ZT, true, true>(p, st) : launch_ring<GATED, XT, ZT, true, false>(p, st);
  return backward ? launch_ring<GATED, XT, ZT, false, true>(p, st) : launch_ring<GATED, XT, ZT, false, false>(p, st);
}
template <bool GATED>
static int launch_norm(const RingParams& p, bool backward, cudaStream_t st) {
  if constexpr (!GATED) {
    if (p.a.io_dtype == KDA_FP32 && p.a.residual_dtype == KDA_BF16) return launch_types<GATED, KDA_FP32, KDA_BF16>(p, backward, st);
  }
  if (p.a.io_dtype == KDA_FP32) return launch_types<GATED, KDA_FP32, KDA_FP32>(p, backward, st);
  return (GATED ? p.a.gate_dtype : p.a.residual_dtype) == KDA_BF16 ? launch_types<GATED, KDA_BF16, KDA_BF16>(p, backward, st)
                                                                     : launch_types<GATED, KDA_BF16, KDA_FP32>(p, backward, st);
}

int norm_ring(const kda_norm_args& a, bool gated, bool backward, float* partial, int* partials, cudaStream_t st) {
  RingParams p{};
  if (!plan(a, gated, backward, p)) return KDA_E_SHAPE;
  p.a = a;
  p.partial = partial;
  *partials = static_cast<int>(ring_ctas(p));
  return gated ? launch_norm<true>(p, backward, st) : launch_norm<false>(p, backward, st);
}
#endif

}  // namespace kda
