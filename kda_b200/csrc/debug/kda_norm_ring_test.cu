// Development check of the norms' kernel for many rows when waits for a stage give up (built into libkda_b200_debug.so, not into the product library): the kernel itself, with a
// verdict that says so to one warp of one CTA, in a given round through the stages.  That warp frees no stage any more, so the CTA's other bounded waits run out as well (a second
// or two); the rows that are left stay unwritten, the status word says so, and every warp comes to the kernel's end.
namespace kda {
__device__ int g_lose[3];      // CTA, warp (-1: none), first round through the stages
}  // namespace kda
#define KDA_RING_VERDICT(ok) ((ok) && !(blockIdx.x == g_lose[0] && warp == g_lose[1] && k == g_lose[2]))
#include "../kda_norm_ring.cu"

// gated norm in bf16, backward when args->dy is there, without sums over rows; status: of these kernels, cleared by the read
extern "C" __attribute__((visibility("default"))) int kda_b200_debug_ring_lost(const kda_norm_args* args, int cta, int warp, int round, float* partial, uint32_t* status, void* stream) {
  using namespace kda;
  if (!args || !status) return KDA_E_NULL;
  const bool backward = args->dy != nullptr;
  RingParams p{};
  if (args->io_dtype != KDA_BF16 || args->gate_dtype != KDA_BF16 || args->cols % 8 || !norm_aligned(*args) || !plan(*args, true, backward, p)) return KDA_E_SHAPE;
  p.a = *args;
  p.partial = partial;
  const int lose[3] = {cta, warp, round};
  cudaError_t e = cudaMemcpyToSymbol(g_lose, lose, sizeof(lose));
  if (e != cudaSuccess) return static_cast<int>(e);
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int rc = backward ? launch_ring<true, KDA_BF16, KDA_BF16, true, true>(p, st) : launch_ring<true, KDA_BF16, KDA_BF16, true, false>(p, st);
  if (rc != KDA_OK) return rc;
  if ((e = cudaStreamSynchronize(st)) != cudaSuccess) return static_cast<int>(e);
  return norm_ring_status(status);
}
