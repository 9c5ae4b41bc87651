// Beam selection: the k best continuations over the beams of a batch item and the vocabulary.
//
//   c[w, v] = score[w] + (logit[w, v] - logsumexp(logit[w, :]));  ended beam: c[w, eos] = score[w],
//   -inf elsewhere; a beam whose score or logsumexp is not finite: -inf everywhere.
// The k largest c in descending order, ties to the lowest (w, v).  Within a beam the order of c is
// the order of the logits, so a pass over the logits only has to bring back the k largest of every
// beam and the running maximum and sum of the softmax.
// Measured: 256 rows of 129283 bf16 logits 33.7 us, 2.0 TB/s, the same rows in fp32 39.5 us, 3.3 TB/s; 4 rows of 32000
// 8.0 us (two launches).  Neither DRAM (27 %) nor the issue slots (59 %, some 15 instructions a value) are full: the
// largest stall is at the barriers around the threshold, and 512 CTAs on 592 places leave some SMs a fourth, some not.
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
  float sum;                                           // sum of exp(logit - max); NaN if one is NaN or +inf
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

constexpr int kBeamPer = 16;                           // values of a thread and tile
constexpr int kBeamTile = kBeamThreads * kBeamPer;
// A thread adds up this many tiles (512 values) in fp32, the rest in fp64: at most 48 roundings in a row, 2^-18 of
// the sum.
constexpr int kBeamFold = 32;
constexpr int kBeamCap = 1024;                         // candidates that a CTA can hold

// Up to kFar a reference ref = rn(m log2e) is off from m log2e by at most 2^-4 (half a step of fp32), so that
// 2^(x log2e - ref) is at most 2^(1/16) and its sum can be put right at the end; beyond it the steps grow to where
// that exponential is infinite or 0 at x = m, and the difference x - m is taken first.
constexpr float kLog2e = 1.4426950408889634f, kFar = 1048576.f;
__device__ __forceinline__ float beam_exp2(float d) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(d));
  return r;
}
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

// One CTA per part of a row, one pass over its logits (bound: HBM; 16 values a thread in registers,
// 16-byte loads whatever the row's alignment): the softmax's running maximum and sum, and the k
// largest.  For those, the first tile gives a threshold that at least k of its values reach: the k-th
// largest of the maxima of 32 groups of 128 values.  From there on a value costs one comparison; the
// few that reach the threshold (k or a few more of the first tile, about k / 4096 of the others) are
// put aside and ranked at the end; the threshold follows them after 2, 4, 8 ... tiles.  Rows with more than kBeamCap of them (many equal or nothing but
// -inf, values in rising order) take k more passes, each for the largest key below the last.
template <typename T>
__global__ void __launch_bounds__(kBeamThreads, 4) k_beam_rows(const BeamArgs A) {
  constexpr int N = VecT<T>::N, NV = kBeamPer / N;
  __shared__ unsigned long long s_keys[kBeamCap];
  __shared__ unsigned long long s_group[32];
  __shared__ float s_max[kBeamThreads / 32];
  __shared__ double s_sum[kBeamThreads / 32];
  __shared__ int s_count;
  __shared__ unsigned long long s_tau;
  pdl_wait();
  pdl_launch_dependents();
  const int row = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const T* x = static_cast<const T*>(A.logits) + (size_t)row * A.ld;
  // vectors of the row counted from the 16-byte boundary at or before its first value
  const int skip = (int)((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T));
  const int vecs = (int)(((long long)skip + A.vocab + N - 1) / N);
  const int v0 = (int)((long long)vecs * blockIdx.x / A.splits), v1 = (int)((long long)vecs * (blockIdx.x + 1) / A.splits);
  const int i0 = max(v0 * N - skip, 0), i1 = min(v1 * N - skip, A.vocab);    // its values
  if (threadIdx.x == 0) s_count = 0;

  // the vectors of the next tile are on their way while this one is worked on; the ones at the row's
  // ends, which reach over it, are read value by value when it is their turn
  const int whole0 = max(v0, skip ? 1 : 0);            // vectors that lie inside the row
  const unsigned wholes = (unsigned)max(min(v1, (int)(((long long)skip + A.vocab) / N)) - whole0, 0);
  auto whole = [&](int v) { return (unsigned)(v - whole0) < wholes; };
  uint4 next[NV];
  const uint4* from = reinterpret_cast<const uint4*>(x - skip) + v0 + threadIdx.x;   // (never read before the row)
  auto fetch = [&](int base) {
#pragma unroll
    for (int k = 0; k < NV; ++k)
      if (whole(base + k * kBeamThreads + (int)threadIdx.x)) next[k] = ldg_stream(from + k * kBeamThreads);
    from += kBeamThreads * NV;
  };
  fetch(v0);
  float m = -CUDART_INF_F, ref = 0.f, sum = 0.f, tau = -CUDART_INF_F;
  float whole_m = -CUDART_INF_F;                       // of the tiles before the last few (kBeamFold): their maximum
  double whole_sum = 0;                                // and their sum relative to it
  // Sum relative to m instead of 2^ref: both products are with the same constant, so what is left of
  // its error is a factor of (x - m)
  auto fold = [&]() {
    if (m > -CUDART_INF_F && fabsf(ref) <= kFar) sum *= beam_exp2(-fmaf(m, kLog2e, -ref));
    if (whole_m < m) whole_sum *= beam_exp2((whole_m - m) * kLog2e);   // (nothing yet: 0 times 0, or a NaN that stays)
    whole_m = m;
    whole_sum += sum;
    sum = 0.f;
  };
  for (int base = v0; base < v1; base += kBeamThreads * NV) {
    float f[NV][N];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int v = base + k * kBeamThreads + threadIdx.x, e0 = v * N - skip;
      VecT<T>::unpack(next[k], f[k]);
      if (!whole(v)) {
#pragma unroll
        for (int i = 0; i < N; ++i) f[k][i] = v < v1 && e0 + i >= 0 && e0 + i < A.vocab ? VecT<T>::to_f(x[e0 + i]) : -CUDART_INF_F;
      }
    }
    fetch(base + kBeamThreads * NV);
    float top = -CUDART_INF_F;
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
      for (int i = 0; i < N; ++i) top = fmaxf(top, f[k][i]);     // (drops NaN)
    if (top > m) {
      const float to = top * kLog2e;
      // (while nothing has been summed there is no m to come from: the sum is 0, or NaN after a NaN)
      if (m > -CUDART_INF_F) {
        const bool was = fabsf(ref) <= kFar, is = fabsf(to) <= kFar;
        float by = was && is ? ref - to : (m - top) * kLog2e;
        if (was != is) by += was ? -fmaf(m, kLog2e, -ref) : fmaf(top, kLog2e, -to);   // relative to 2^ref on one side only
        sum *= beam_exp2(by);
      }
      m = top;
      ref = to;
    }
    // 2^(x log2e - ref), one rounding: ref is only near m log2e, which the end of the kernel makes up
    // for.  Far from zero (masks of large negative numbers) the difference comes first.
    float part = 0.f;
    if (fabsf(ref) <= kFar) {
#pragma unroll
      for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int i = 0; i < N; ++i) part += beam_exp2(fmaf(f[k][i], kLog2e, -ref));   // a NaN makes it NaN
    } else {                                           // m = +inf: NaN
#pragma unroll
      for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int i = 0; i < N; ++i) part += beam_exp2((f[k][i] - m) * kLog2e);
    }
    sum += part;
    // bit k N + i: the value is this row's and reaches the threshold (a NaN counts as -inf)
    auto reaching = [&](float t) {
      uint32_t bits = 0;
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        const int v = base + k * kBeamThreads + threadIdx.x;
#pragma unroll
        for (int i = 0; i < N; ++i) {
          if (t == -CUDART_INF_F ? !(f[k][i] > t) || f[k][i] > t : f[k][i] >= t) bits |= 1u << (k * N + i);
        }
        if (!whole(v)) {
#pragma unroll
          for (int i = 0; i < N; ++i) {
            const int e = v * N - skip + i;
            if (v >= v1 || e < 0 || e >= A.vocab) bits &= ~(1u << (k * N + i));
          }
        }
      }
      return bits;
    };
    auto index = [&](int bit) { return (base + (bit / N) * kBeamThreads + (int)threadIdx.x) * N - skip + bit % N; };
    if (base == v0) {
      const uint32_t bits = reaching(top);             // the first of the thread's largest
      unsigned long long best = bits ? beam_key(top, index(__ffs(bits) - 1)) : 0;
#pragma unroll
      for (int o = 1; o < 8; o <<= 1) {
        const unsigned long long u = __shfl_xor_sync(0xffffffffu, best, o);
        best = u > best ? u : best;
      }
      if ((lane & 7) == 0) s_group[threadIdx.x >> 3] = best;
      __syncthreads();
      if (warp == 0) {
        const unsigned long long mine = s_group[lane];
        int rank = 0;
#pragma unroll 8
        for (int j = 0; j < 32; ++j) rank += s_group[j] > mine || (s_group[j] == mine && j < lane);
        if (rank == A.k - 1) s_tau = mine;             // 0 where fewer than k groups hold a value
      }
      __syncthreads();
      const unsigned long long t = s_tau;
      tau = t == 0 ? -CUDART_INF_F : beam_value((uint32_t)(t >> 32));
    }
    if (top >= tau) {
      for (uint32_t bits = reaching(tau); bits; bits &= bits - 1) {
        const int e = index(__ffs(bits) - 1), at = atomicAdd(&s_count, 1);
        if (at < kBeamCap) s_keys[at] = beam_key(VecT<T>::to_f(x[e]), e);
      }
    }
    const int tiles = (base - v0) / (kBeamThreads * NV) + 1;
    if (tiles % kBeamFold == 0) fold();
    // after 2, 4, 8 ... tiles: the k-th largest so far is the threshold of the next
    if (tiles > 1 && (tiles & (tiles - 1)) == 0 && base + kBeamThreads * NV < v1) {
      __syncthreads();
      const int n = s_count;
      if (n <= kBeamThreads && (int)threadIdx.x < n) {
        const unsigned long long mine = s_keys[threadIdx.x];
        int rank = 0;
        for (int j = 0; j < n; ++j) rank += s_keys[j] > mine;
        if (rank == A.k - 1) s_tau = mine;
      }
      __syncthreads();
      const unsigned long long t = s_tau;
      tau = t == 0 ? -CUDART_INF_F : beam_value((uint32_t)(t >> 32));
    }
  }
  fold();
  // maximum and sum of the part
  float top = m;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  double all = top == -CUDART_INF_F ? (whole_sum == whole_sum ? 0.0 : whole_sum) : whole_sum * beam_exp2((m - top) * kLog2e);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) all += __shfl_xor_sync(0xffffffffu, all, o);
  if (lane == 0) {
    s_max[warp] = top;
    s_sum[warp] = all;
  }
  __syncthreads();
  const size_t part = (size_t)row * A.splits + blockIdx.x;
  if (threadIdx.x == 0) {
    float t = -CUDART_INF_F;
    for (int w = 0; w < kBeamThreads / 32; ++w) t = fmaxf(t, s_max[w]);
    double total = 0;
    for (int w = 0; w < kBeamThreads / 32; ++w)
      total += s_max[w] == -CUDART_INF_F ? s_sum[w] : s_sum[w] * (double)expf(s_max[w] - t);
    A.parts[part] = {t, (float)total};
  }
  unsigned long long* out = A.keys + part * A.k;
  const int n = s_count;
  if (n <= kBeamCap) {
    for (int i = threadIdx.x; i < n; i += kBeamThreads) {
      const unsigned long long mine = s_keys[i];
      int rank = 0;
      for (int j = 0; j < n; ++j) rank += s_keys[j] > mine;
      if (rank < A.k) out[rank] = mine;
    }
    for (int i = n + threadIdx.x; i < A.k; i += kBeamThreads) out[i] = 0;
    return;
  }
  unsigned long long last = ~0ull;
  for (int k = 0; k < A.k; ++k) {
    unsigned long long best = 0;
    for (int i = i0 + threadIdx.x; i < i1; i += kBeamThreads) {
      const unsigned long long key = beam_key(VecT<T>::to_f(x[i]), i);
      if (key < last && key > best) best = key;
    }
    last = beam_block_max(best, s_keys);
    if (threadIdx.x == 0) out[k] = last;
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
  long long* s_flat = reinterpret_cast<long long*>(s_lse + rows);      // [rows * k] beam * vocab + token, -1: none
  const int item = blockIdx.x, row0 = item * A.beams;
  for (int i = threadIdx.x; i < rows * per_row; i += blockDim.x)
    s_key[i] = A.keys[(size_t)row0 * per_row + i];
  for (int i = threadIdx.x; i < rows * A.k; i += blockDim.x) s_flat[i] = -1;
  for (int r = threadIdx.x >> 5; r < rows; r += kBeamThreads / 32) {     // a warp per row
    const BeamPart* p = A.parts + (size_t)(row0 + r) * A.splits;
    const int lane = threadIdx.x & 31;
    float top = -CUDART_INF_F;
    for (int s = lane; s < A.splits; s += 32) top = fmaxf(top, p[s].max);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    double sum = 0;
    for (int s = lane; s < A.splits; s += 32)
      if (!(p[s].max == -CUDART_INF_F && p[s].sum == 0.f)) sum += (double)p[s].sum * (double)expf(p[s].max - top);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) s_lse[r] = (double)top + log(sum);
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
    s_flat[r * A.k + rank] = (long long)r * A.vocab + tok;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < rows * A.k; i += blockDim.x) {
    const long long flat = s_flat[i];
    if (flat < 0) continue;                            // fewer than k tokens in the vocabulary
    const double v = s_c[i];
    int rank = 0;
#pragma unroll 4
    for (int j = 0; j < rows * A.k; ++j)
      rank += s_flat[j] >= 0 && (s_c[j] > v || (s_c[j] == v && s_flat[j] < flat));
    if (rank >= A.k) continue;
    const size_t o = (size_t)item * A.k + rank;
    const int r = i / A.k, tok = (int)(flat - (long long)r * A.vocab);
    A.out_scores[o] = (float)v;
    A.out_rows[o] = row0 + r;
    A.out_tokens[o] = tok;
    if (A.out_done) A.out_done[o] = (A.done && A.done[row0 + r]) || tok == A.eos;
  }
}

}  // namespace cats
