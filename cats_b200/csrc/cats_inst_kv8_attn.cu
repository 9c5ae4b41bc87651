// The attention kernels of the paged 8-bit cache for ONE element type; compiled once per type with
// -DCATS_ELEM_ID=0|1|2 (float, __half, __nv_bfloat16).
#include "cats_kv8_attn.cuh"
#include "cats_kv8_run.cuh"

namespace cats {

template <typename T, int HD, int NQ>
static cudaError_t run_attend(const cats_kv8& c, const KvAttnArgs<T>& A, cudaStream_t st) {
  using S = AttnShape<NQ>;
  // (the attribute stays with the kernel: once per device; two threads at once set the same value)
  static bool ready[64];
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !ready[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(reinterpret_cast<const void*>(k_kv8_attend<T, HD, NQ>),
                                               cudaFuncAttributeMaxDynamicSharedMemorySize, (int)attn_smem<NQ>());
    if (e != cudaSuccess) return e;
    if (dev >= 0 && dev < 64) ready[dev] = true;
  }
  return launch_ready(k_kv8_attend<T, HD, NQ>, dim3(A.ctas), dim3(S::kThreads), attn_smem<NQ>(), st, c, A);
}

template <typename T, int HD>
static cudaError_t run_attend(const cats_kv8& c, const KvAttnArgs<T>& A, cudaStream_t st) {
  // rows of a key head: (new tokens) x (query heads per key head), on average over the sequences
  const long long rows = ((long long)A.tokens + c.n_seqs - 1) / c.n_seqs * (A.nh / c.n_kv_heads);
  if (rows <= 8) return run_attend<T, HD, 1>(c, A, st);
  if constexpr (sizeof(T) == 2) {                       // (fp32 queries are two halves: no room)
    if (rows > 16) return run_attend<T, HD, 4>(c, A, st);
  }
  return run_attend<T, HD, 2>(c, A, st);
}

template <typename T>
cudaError_t inst_kv8_attend(const cats_kv8& c, const KvAttnArgs<T>& A, cudaStream_t st) {
  switch (c.head_dim) {
    case 32: return run_attend<T, 32>(c, A, st);
    case 64: return run_attend<T, 64>(c, A, st);
    case 96: return run_attend<T, 96>(c, A, st);
    default: return run_attend<T, 128>(c, A, st);
  }
}

#if CATS_ELEM_ID == 0
template cudaError_t inst_kv8_attend<float>(const cats_kv8&, const KvAttnArgs<float>&, cudaStream_t);
#elif CATS_ELEM_ID == 1
template cudaError_t inst_kv8_attend<__half>(const cats_kv8&, const KvAttnArgs<__half>&, cudaStream_t);
#else
template cudaError_t inst_kv8_attend<__nv_bfloat16>(const cats_kv8&, const KvAttnArgs<__nv_bfloat16>&, cudaStream_t);
#endif

}  // namespace cats
