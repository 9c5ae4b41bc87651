// The attention kernels of the paged 8-bit cache for ONE element type; compiled once per type with
// -DCATS_ELEM_ID=0|1|2 (float, __half, __nv_bfloat16).
#include "cats_kv8_attn.cuh"
#include "cats_kv8_run.cuh"

namespace cats {

template <typename T, int HD>
static cudaError_t run_attend(const cats_kv8& c, const KvAttnArgs<T>& A, cudaStream_t st) {
  cudaError_t e = launch(k_kv8_attend<T, HD>, dim3(A.ctas), dim3(kAttnThreads), attn_smem(HD), st, c, A);
  if (e != cudaSuccess) return e;
  const long long rows = ((long long)A.tokens * A.nh + kAttnWarps - 1) / kAttnWarps, most = 8LL * dev_info().sms;
  return launch(k_kv8_attend_join<T, HD>, dim3((unsigned)(rows < most ? rows : most)), dim3(kAttnThreads), 0, st, c, A);
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
