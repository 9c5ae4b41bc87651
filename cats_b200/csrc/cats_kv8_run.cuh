// Launcher of the attention kernels (one translation unit per element type, cats_inst_kv8_attn.cu).
#pragma once

#include "cats_kv8_attn.cuh"
#include "cats_run.cuh"

namespace cats {

template <typename T>
cudaError_t inst_kv8_attend(const cats_kv8& c, const KvAttnArgs<T>& A, cudaStream_t st);
extern template cudaError_t inst_kv8_attend<float>(const cats_kv8&, const KvAttnArgs<float>&, cudaStream_t);
extern template cudaError_t inst_kv8_attend<__half>(const cats_kv8&, const KvAttnArgs<__half>&, cudaStream_t);
extern template cudaError_t inst_kv8_attend<__nv_bfloat16>(const cats_kv8&, const KvAttnArgs<__nv_bfloat16>&,
                                                           cudaStream_t);

}  // namespace cats
