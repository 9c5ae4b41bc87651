// The attention kernels of the paged 8-bit cache for ONE element type; compiled once per type with
// -DCATS_ELEM_ID=0|1|2 (float, __half, __nv_bfloat16).
#include "cats_kv8_attn_tc.cuh"
#include "cats_kv8_run.cuh"

namespace cats {

template <typename T>
static cudaError_t run(void (*kernel)(cats_kv8, KvAttnArgs<T>), int threads, size_t smem, const cats_kv8& c,
                       const KvAttnArgs<T>& A, cudaStream_t st) {
  return launch(kernel, dim3(A.ctas), dim3(threads), smem, st, c, A);
}

template <typename T, int HD, int NQ>
static cudaError_t run_attend(const cats_kv8& c, const KvAttnArgs<T>& A, cudaStream_t st) {
  return run<T>(k_kv8_attend<T, HD, NQ>, AttnShape<NQ>::kThreads, attn_smem<NQ>(), c, A, st);
}

// Up to 8 rows and up to 16 the tiles of cats_kv8_attn.cuh, bound by the codes' bytes; beyond that the
// products count.  (Rows of a key head, on average over all sequences of the cache: idle ones count too, so that a
// long span among many of them gets small tiles, right but slower.)  A CTA takes 128 positions of 32 rows in 1.9 us
// with those tiles, and of up to 128 rows in 3.3 us on tcgen05 (2 x 256 tokens x 4 heads per key head: 217 and 128 us
// at head_dim 128, 162 and 101 us at 64): 16-bit
// queries with more than 32 rows go there, but for head_dim 32 and 96, which do not fill a 128-byte
// swizzle row.  fp32 queries are split in two halves, which leaves registers for 16 rows.
template <typename T, int HD>
static cudaError_t run_attend(const cats_kv8& c, const KvAttnArgs<T>& A, cudaStream_t st) {
  const long long rows = attn_rows(c, A.tokens, A.nh);
  if (rows <= 8) return run_attend<T, HD, 1>(c, A, st);
  if constexpr (sizeof(T) == 2) {
    if (rows > kAttnFewRows) {
      if constexpr (HD % 64 == 0) {
        if (rows > kAttnSomeRows) return run<T>(k_kv8_attend_tc<T, HD>, kTcThreads, attn_tc_smem(HD), c, A, st);
      }
      return run_attend<T, HD, 4>(c, A, st);
    }
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
