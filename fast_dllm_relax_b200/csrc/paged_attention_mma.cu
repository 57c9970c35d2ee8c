// Attention over a paged 8-bit KV cache on the 5th-generation tensor cores (fdllm_paged_attention, bf16, head_dim
// 128): one launch for the items of all classes, a CTA an item.  Tiles of up to 48 query rows have the keys on the
// MMA's M side (paged_attention_tc.cuh), larger ones the rows (paged_attention_wide.cuh).
//
// A class is a range of the grid, so a CTA sets its barriers and tensor memory up before the plan may be read.  The
// classes' CTAs run side by side: 4 requests of 1 to 8 rows over a few keys, tiles of three classes, take 9.3 us,
// with a launch a class they took 21.8 (8 prompts of 2 to 221 rows: 10.9 instead of 27.0).
#include "paged_attention_tc.cuh"
#include "paged_attention_wide.cuh"

namespace fdllm {

namespace {

template <typename... T>
constexpr size_t largest() {
  size_t m = 0;
  ((m = sizeof(T) > m ? sizeof(T) : m), ...);
  return m;
}
constexpr int most(int a, int b) { return a > b ? a : b; }
constexpr size_t kBars = largest<paged_tc::Bars<16>, paged_tc::Bars<32>, paged_tc::Bars<48>, paged_wide::Bars>();
constexpr int kBytes = most(most(paged_tc::Cfg<16>::kBytes, paged_tc::Cfg<32>::kBytes),
                            most(paged_tc::Cfg<48>::kBytes, paged_wide::kBytes));
static_assert(2 * (kBytes + static_cast<int>(kBars) + 1024) <= 228 * 1024, "two CTAs per SM, with the system's 1 KB each");

}  // namespace

__global__ void __launch_bounds__(kThreads, 2)
    paged_attn_mma_kernel(const PagedAttnArgs a, const __grid_constant__ CUtensorMap tm_k,
                          const __grid_constant__ CUtensorMap tm_v) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ alignas(16) uint8_t bars[kBars];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int i = blockIdx.x;
  if (i < a.class_end[kPagedWide]) paged_wide::run(a, tm_k, tm_v, smem, *reinterpret_cast<paged_wide::Bars*>(bars));
  else if (i < a.class_end[2]) paged_tc::run<48>(a, tm_k, tm_v, smem, *reinterpret_cast<paged_tc::Bars<48>*>(bars));
  else if (i < a.class_end[1]) paged_tc::run<32>(a, tm_k, tm_v, smem, *reinterpret_cast<paged_tc::Bars<32>*>(bars));
  else paged_tc::run<16>(a, tm_k, tm_v, smem, *reinterpret_cast<paged_tc::Bars<16>*>(bars));
}

// The register splits only ever ask for what the launch brought: checked here, not by waiting for more.
int init_paged_attention_mma_attributes() {
  cudaFuncAttributes f;
  cudaError_t e = cudaFuncGetAttributes(&f, paged_attn_mma_kernel);
  if (e == cudaSuccess && f.numRegs < kRegsLaunch) e = cudaErrorInvalidKernelImage;
  return e != cudaSuccess ? e : cudaFuncSetAttribute(paged_attn_mma_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kBytes);
}

int launch_paged_attention_mma(const PagedAttnArgs& a, const CUtensorMap& k, const CUtensorMap& v, cudaStream_t s) {
  return launch_k(paged_attn_mma_kernel, dim3(a.class_end[0]), dim3(kThreads), kBytes, s, a, k, v);
}

}  // namespace fdllm
