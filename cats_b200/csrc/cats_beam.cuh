// Beam selection: the k best continuations over the beams of a batch item and the vocabulary.
//
//   c[w, v] = score[w] + (logit[w, v] - logsumexp(logit[w, :]));  ended beam: c[w, eos] = score[w],
//   -inf elsewhere; a beam whose score or logsumexp is not finite: -inf everywhere.
// The k largest c in descending order, ties to the lowest (w, v).  Within a beam the order of c is
// the order of the logits, so a pass over the logits only has to bring back the k largest of every
// beam and the running maximum and sum of the softmax.
#pragma once

#include <math_constants.h>

#include "cats_common.cuh"

namespace cats {

constexpr int kBeamThreads = 256;
constexpr int kBeamMaxK = 32;
constexpr int kBeamMaxBeams = 32;

// fp32 -> unsigned whose order is the order of the floats; NaN as -inf
__device__ __forceinline__ uint32_t beam_order(float x) {
  if (x != x) x = -CUDART_INF_F;
  if (x == 0.f) x = 0.f;                               // -0 == +0
  const uint32_t b = __float_as_uint(x);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float beam_value(uint32_t o) {
  return __uint_as_float((o & 0x80000000u) ? (o & 0x7fffffffu) : ~o);
}
// larger key = earlier place: value, then lower index
__device__ __forceinline__ unsigned long long beam_key(float x, int idx) {
  return ((unsigned long long)beam_order(x) << 32) | (0xffffffffu - (uint32_t)idx);
}

struct BeamPart {                                      // of one row (or part of a row)
  float max;                                           // largest logit (not a NaN)
  float sum;                                           // sum of exp(logit - max); NaN if a logit is
};

struct BeamArgs {
  const void* logits;                                  // [n, beams, vocab], rows ld elements apart
  long long ld;
  const float* scores;                                 // [n, beams]
  const uint8_t* done;                                 // [n, beams] or nullptr
  int n, beams, vocab, k, eos, splits;
  BeamPart* parts;                                     // [rows, splits]
  unsigned long long* keys;                            // [rows, splits, k], 0 where there are fewer
  float* out_scores;                                   // [n, k]
  int* out_rows;                                       // [n, k]
  long long* out_tokens;                               // [n, k]
  uint8_t* out_done;                                   // [n, k] or nullptr
};

__device__ __forceinline__ unsigned long long beam_block_max(unsigned long long v, unsigned long long* s) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const unsigned long long u = __shfl_xor_sync(0xffffffffu, v, o);
    v = u > v ? u : v;
  }
  __syncthreads();
  if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
  __syncthreads();
  for (int w = 0; w < kBeamThreads / 32; ++w) v = s[w] > v ? s[w] : v;
  return v;
}

// One CTA per row: k passes that each find the largest key below the last one found.
template <typename T>
__global__ void __launch_bounds__(kBeamThreads) k_beam_rows_simple(const BeamArgs A) {
  pdl_wait();
  __shared__ unsigned long long s_key[kBeamThreads / 32];
  __shared__ float s_sum[kBeamThreads / 32];
  const int row = blockIdx.x;
  const T* x = static_cast<const T*>(A.logits) + (size_t)row * A.ld;
  unsigned long long last = ~0ull;
  float top = 0.f;
  for (int k = 0; k < A.k; ++k) {
    unsigned long long best = 0;
    for (int i = threadIdx.x; i < A.vocab; i += kBeamThreads) {
      const unsigned long long key = beam_key(VecT<T>::to_f(x[i]), i);
      if (key < last && key > best) best = key;
    }
    last = beam_block_max(best, s_key);
    if (k == 0) top = beam_value((uint32_t)(last >> 32));
    if (threadIdx.x == 0) A.keys[(size_t)row * A.k + k] = last;
  }
  float sum = 0.f;
  for (int i = threadIdx.x; i < A.vocab; i += kBeamThreads) sum += expf(VecT<T>::to_f(x[i]) - top);
  sum = warp_sum(sum);
  if ((threadIdx.x & 31) == 0) s_sum[threadIdx.x >> 5] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    double t = 0;
    for (int w = 0; w < kBeamThreads / 32; ++w) t += s_sum[w];
    A.parts[row] = {top, (float)t};
  }
}

// One CTA per batch item: the rows' parts and keys into the k best of the item.  Every candidate
// counts the candidates before it; its rank is its place.
__global__ void __launch_bounds__(kBeamThreads) k_beam_join(const BeamArgs A) {
  pdl_wait();
  extern __shared__ __align__(16) unsigned char smem[];
  const int per_row = A.splits * A.k, rows = A.beams;
  double* s_c = reinterpret_cast<double*>(smem);                       // [rows * k]
  unsigned long long* s_key = reinterpret_cast<unsigned long long*>(s_c + rows * A.k);  // [rows * per_row]
  double* s_lse = reinterpret_cast<double*>(s_key + (size_t)rows * per_row);            // [rows]
  int* s_tok = reinterpret_cast<int*>(s_lse + rows);                   // [rows * k]
  const int item = blockIdx.x, row0 = item * A.beams;
  for (int i = threadIdx.x; i < rows * per_row; i += blockDim.x)
    s_key[i] = A.keys[(size_t)row0 * per_row + i];
  for (int i = threadIdx.x; i < rows * A.k; i += blockDim.x) s_tok[i] = -1;
  for (int r = threadIdx.x; r < rows; r += blockDim.x) {
    const BeamPart* p = A.parts + (size_t)(row0 + r) * A.splits;
    float top = -CUDART_INF_F;
    for (int s = 0; s < A.splits; ++s) top = fmaxf(top, p[s].max);
    double sum = 0;
    for (int s = 0; s < A.splits; ++s)
      if (!(p[s].max == -CUDART_INF_F && p[s].sum == 0.f)) sum += (double)p[s].sum * exp((double)p[s].max - (double)top);
    s_lse[r] = (double)top + log(sum);
  }
  __syncthreads();
  // the k largest logits of each row, in order
  for (int i = threadIdx.x; i < rows * per_row; i += blockDim.x) {
    const int r = i / per_row;
    const unsigned long long key = s_key[i];
    if (key == 0) continue;
    int rank = 0;
    for (int j = 0; j < per_row; ++j) rank += s_key[r * per_row + j] > key;
    if (rank >= A.k) continue;
    const bool done = A.done && A.done[row0 + r];
    const float score = A.scores[row0 + r];
    const double lse = s_lse[r];
    double v = (double)score + ((double)beam_value((uint32_t)(key >> 32)) - lse);
    int tok = (int)(0xffffffffu - (uint32_t)key);
    // a row without usable values takes part with its first tokens at -inf; an ended one with eos
    // and then its first other tokens
    if (done) {
      tok = rank == 0 ? A.eos : rank - 1 < A.eos ? rank - 1 : rank;
      v = rank == 0 ? (double)score : -CUDART_INF;
      if (!isfinite(score)) {
        tok = rank;
        v = -CUDART_INF;
      }
    } else if (!isfinite(score) || !isfinite(lse)) {
      tok = rank;
      v = -CUDART_INF;
    }
    s_c[r * A.k + rank] = v;
    s_tok[r * A.k + rank] = tok;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < rows * A.k; i += blockDim.x) {
    const int tok = s_tok[i], r = i / A.k;
    if (tok < 0) continue;                             // fewer than k tokens in the vocabulary
    const double v = s_c[i];
    int rank = 0;
    for (int j = 0; j < rows * A.k; ++j) {
      if (s_tok[j] < 0) continue;
      const int q = j / A.k;
      rank += s_c[j] > v || (s_c[j] == v && (q < r || (q == r && s_tok[j] < tok)));
    }
    if (rank >= A.k) continue;
    const size_t o = (size_t)item * A.k + rank;
    A.out_scores[o] = (float)v;
    A.out_rows[o] = row0 + r;
    A.out_tokens[o] = tok;
    if (A.out_done) A.out_done[o] = (A.done && A.done[row0 + r]) || tok == A.eos;
  }
}

}  // namespace cats
