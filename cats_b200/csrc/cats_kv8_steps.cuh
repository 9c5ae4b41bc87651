// Paged key/value cache in 8 bits (cats_kv8.cuh): the writer (rotary embedding + quantisation) and
// the page bookkeeping (grow, reorder, compact).
#pragma once

#include "cats_kv8.cuh"

namespace cats {

// ---------------------------------------------------------------------------------------------
// append: rotary embedding + quantising write
// ---------------------------------------------------------------------------------------------
// One CTA per (sequence, touched page) and some of its blocks of rows (keys or values, head), one after
// the other: a scale belongs to a block, so the CTA that takes the rows' largest magnitude is the one that writes them, and the new
// rows are read once and stay in registers between the two (at most RPT rows of a thread).  hd / 16
// threads share a row; a thread holds eight values of the row's first half and the eight that the
// rotation pairs them with.  Further CTAs of the same launch rotate the queries: a thread keeps its
// token's cosines and sines and goes through the heads, four of them on their way.
// Rounding: products and sums of the rotation are each rounded to fp32 (no contraction), the query
// once more to its type; keys and values go from fp32 straight to e4m3.  Infinities are stored as
// NaN (e4m3 has none) and neither sets a scale.
// Measured: a decode step of eight sequences 2.9 us, all of it the launch and three dependent loads
// (length, page, row); four prompts of 700 .. 4096 tokens, 32 + 2 x 32 heads of 128, bf16, 346 MB: 73 us,
// 4.7 TB/s (the queries alone 28 us, 5 TB/s; keys and values, 256-byte pieces of far rows, 66 us); with one
// block of rows per CTA and no loads under way it was 130 us.  Two CTAs of 256 threads an SM: with three,
// 80 registers each, values are spilled (80 us; 8000 fp32 tokens of 32 + 2 x 8 heads: 92 us, 65 with two).
template <typename T>
struct KvAppendArgs {
  const T* qkv;
  long long ld;           // elements between two tokens
  const T* cosv;          // [rope_len, hd] or nullptr
  const T* sinv;
  T* q_out;               // [tokens, nh, hd] or nullptr
  const int* cu;
  int uniform, tokens, nh, layer, kv_blocks;
  int kv_heads, q_heads;  // blocks of rows (keys' and values' heads) and query heads of a CTA
};

// sixteen values as they lie in memory: columns col .. col + 8 and col + half .. col + half + 8
template <typename T>
struct Raw16 {
  static constexpr int K = sizeof(T) / 2;
  uint4 v[2 * K];
  __device__ __forceinline__ void load(const T* p, int half) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      v[k] = ldg_stream(reinterpret_cast<const uint4*>(p) + k);
      v[K + k] = ldg_stream(reinterpret_cast<const uint4*>(p + half) + k);
    }
  }
  __device__ __forceinline__ void load_cached(const T* p, int half) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      v[k] = __ldg(reinterpret_cast<const uint4*>(p) + k);
      v[K + k] = __ldg(reinterpret_cast<const uint4*>(p + half) + k);
    }
  }
  __device__ __forceinline__ void unpack(float* f) const {
#pragma unroll
    for (int k = 0; k < 2 * K; ++k) VecT<T>::unpack(v[k], f + k * VecT<T>::N);
  }
};

// A token's cosines and sines at sixteen columns.
struct Turn {
  float c[16], s[16];
  template <typename T>
  __device__ __forceinline__ void load(const T* cosv, const T* sinv, int half) {
    Raw16<T> cr, sr;
    cr.load_cached(cosv, half);
    sr.load_cached(sinv, half);
    cr.unpack(c);
    sr.unpack(s);
  }
  __device__ __forceinline__ void apply(float* f) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float a = f[i], b = f[8 + i];
      f[i] = __fadd_rn(__fmul_rn(a, c[i]), __fmul_rn(-b, s[i]));
      f[8 + i] = __fadd_rn(__fmul_rn(b, c[8 + i]), __fmul_rn(a, s[8 + i]));
    }
  }
};

template <typename T>
__device__ __forceinline__ void append_queries(const cats_kv8& c, const KvAppendArgs<T>& A, int block) {
  const int hd = c.head_dim, half = hd >> 1, tpr = hd >> 4;
  const int side = blockDim.x / tpr, r0 = threadIdx.x / tpr, col = (threadIdx.x - r0 * tpr) * 8;
  const int chunks = (A.nh + A.q_heads - 1) / A.q_heads;
  const int tile = block / chunks, h0 = (block - tile * chunks) * A.q_heads, h1 = min(h0 + A.q_heads, A.nh);
  const int t = tile * side + r0;
  if (r0 >= side || t >= A.tokens) return;
  const T* src = A.qkv + (size_t)t * A.ld + col;
  T* dst = A.q_out + (size_t)t * A.nh * hd + col;
  constexpr int kAhead = 4;                              // heads on their way
  Raw16<T> x[kAhead];
  Turn rot;
#pragma unroll
  for (int k = 0; k < kAhead; ++k)
    if (h0 + k < h1) x[k].load(src + (size_t)(h0 + k) * hd, half);
  int b;
  if (!A.cu) {
    b = t / A.uniform;
  } else {                                               // last b with cu[b] <= t
    int lo = 0, hi = c.n_seqs - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (__ldg(A.cu + mid) <= t) lo = mid;
      else hi = mid - 1;
    }
    b = lo;
  }
  const KvSpan sp = kv_span(A.cu, A.uniform, b);
  if (t < sp.first || t - sp.first >= sp.count) return;  // behind the last sequence: left as it is
  bool turn = A.cosv != nullptr;
  if (turn) {
    const int pos = c.lens[b] - sp.count + (t - sp.first);
    turn = pos >= 0 && pos < c.max_pages * c.page;
    if (turn) rot.load(A.cosv + (size_t)pos * hd + col, A.sinv + (size_t)pos * hd + col, half);
    else kv_flag(c, KV_TOO_LONG);
  }
  for (int h = h0; h < h1; h += kAhead) {
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      if (h + k >= h1) continue;
      float f[16];
      x[k].unpack(f);
      if (h + k + kAhead < h1) x[k].load(src + (size_t)(h + k + kAhead) * hd, half);
      if (turn) rot.apply(f);
      store8(dst + (size_t)(h + k) * hd, f);
      store8(dst + (size_t)(h + k) * hd + half, f + 8);
    }
  }
}

template <typename T, int RPT>
__global__ void __launch_bounds__(RPT == 1 ? 32 : 256, RPT == 1 ? 16 : 2) k_kv8_append(const cats_kv8 c, const KvAppendArgs<T> A) {
  pdl_wait();
  pdl_launch_dependents();
  if ((int)blockIdx.x >= A.kv_blocks) {
    append_queries(c, A, blockIdx.x - A.kv_blocks);
    return;
  }
  __shared__ __align__(16) float s_max[2][8];
  const int hd = c.head_dim, half = hd >> 1, tpr = hd >> 4, nkv = c.n_kv_heads;
  const int side = blockDim.x / tpr;
  const int r0 = threadIdx.x / tpr, col = (threadIdx.x - r0 * tpr) * 8;
  const int max_len = c.max_pages * c.page;
  const int chunks = (2 * nkv + A.kv_heads - 1) / A.kv_heads;
  const int unit = blockIdx.x / chunks, x0 = (blockIdx.x - unit * chunks) * A.kv_heads, x1 = min(x0 + A.kv_heads, 2 * nkv);
  int b, j;                                            // sequence, and which of its touched pages
  if (!A.cu) {
    const int per = kv_units(A.uniform, c.page);
    b = unit / per;
    j = unit - b * per;
  } else {                                             // warps scan the sequences 32 at a time
    int before = 0;
    const int lane = threadIdx.x & 31;
    b = -1;
    j = 0;
    for (int b0 = 0; b0 < c.n_seqs && b < 0; b0 += 32) {
      const int mine = b0 + lane < c.n_seqs ? kv_units(kv_span(A.cu, 0, b0 + lane).count, c.page) : 0;
      int incl = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += v;
      }
      const unsigned hit = __ballot_sync(0xffffffffu, before + incl > unit);
      if (hit) {
        const int l = __ffs(hit) - 1;
        b = b0 + l;
        j = unit - before - __shfl_sync(0xffffffffu, incl - mine, l);
      }
      before += __shfl_sync(0xffffffffu, incl, 31);
    }
    if (b < 0) return;                                 // more CTAs than touched pages
  }
  const KvSpan sp = kv_span(A.cu, A.uniform, b);
  const int len = c.lens[b], start = len - sp.count;   // rows [start, len) are new
  const bool refused = kv_refused(c, b);
  const long long at = (long long)start / c.page + j;  // (spans that do not fit can give any j)
  if (sp.count < 1 || j < 0 || at * c.page >= len) return;
  if (refused) {                                       // rows [start, len) are not the new tokens'
    if (threadIdx.x == 0) kv_flag(c, KV_REFUSED);
    return;
  }
  if (start < 0 || len > max_len || sp.first < 0 || (long long)sp.first + sp.count > A.tokens) {
    if (threadIdx.x == 0) kv_flag(c, start < 0 || len > max_len ? KV_TOO_LONG : KV_BAD_SPAN);
    return;
  }
  const int page_i = (int)at;
  const int row0 = page_i * c.page;                    // position of the page's first row
  const int first = max(start - row0, 0), last = min(len - row0, c.page);   // its new rows

  // the first head's new rows and the page's number are on their way together; from then on the next
  // head's rows while this one's are worked on
  Raw16<T> raw[RPT];
  const T* src = A.qkv + ((long long)sp.first + row0 - start) * A.ld + (size_t)A.nh * hd + col;
  auto fetch = [&](int x) {
#pragma unroll
    for (int k = 0; k < RPT; ++k) {
      const int r = first + k * side + r0;
      if (r0 < side && r < last) raw[k].load(src + (long long)r * A.ld + (size_t)x * hd, half);
    }
  };
  fetch(x0);
  const int page = c.table[(size_t)b * c.max_pages + page_i];
  // a page that another sequence holds too is never written
  if (page < 0 || page >= c.n_pages || c.refs[page] != 1) {
    if (threadIdx.x == 0) kv_flag(c, KV_BAD_PAGE);
    return;
  }
  // (magnitudes: their order is that of their bits; the words of the call before last are free again)
  if (threadIdx.x < 16 && (threadIdx.x & 7) >= (blockDim.x >> 5)) s_max[threadIdx.x >> 3][threadIdx.x & 7] = 0.f;
  int turn_of = 0;
  auto block_max = [&](float v) {
    v = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(v)));
    if (RPT > 1) {
      if ((threadIdx.x & 31) == 0) s_max[turn_of][threadIdx.x >> 5] = v;
      __syncthreads();
      const float4 a = *reinterpret_cast<const float4*>(s_max[turn_of]), b = *reinterpret_cast<const float4*>(s_max[turn_of] + 4);
      v = fmaxf(fmaxf(fmaxf(a.x, a.y), fmaxf(a.z, a.w)), fmaxf(fmaxf(b.x, b.y), fmaxf(b.z, b.w)));
      turn_of ^= 1;
    }
    return v;
  };
  for (int x = x0; x < x1; ++x) {
    const bool turn = x < nkv && A.cosv != nullptr;
    float f[RPT][16];
#pragma unroll
    for (int k = 0; k < RPT; ++k) {
#pragma unroll
      for (int i = 0; i < 16; ++i) f[k][i] = 0.f;
      if (r0 < side && first + k * side + r0 < last) raw[k].unpack(f[k]);
    }
    if (x + 1 < x1) fetch(x + 1);
    float amax = 0.f;
#pragma unroll
    for (int k = 0; k < RPT; ++k) {
      const int r = first + k * side + r0;
      if (r0 >= side || r >= last) continue;
      if (turn) {
        Turn rot;
        rot.load(A.cosv + (size_t)(row0 + r) * hd + col, A.sinv + (size_t)(row0 + r) * hd + col, half);
        rot.apply(f[k]);
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) amax = fmaxf(amax, fabsf(f[k][i]));         // (drops NaN)
    }
    float* sc = kv_scale(c, A.layer, page, 0, x);
    const int e_old = first > 0 ? kv_exp_of(*sc) : kKvExpMin;
    amax = block_max(amax);
    if (amax > 3.402823466e38f) {                        // an infinity: a NaN from here on
      amax = 0.f;
#pragma unroll
      for (int k = 0; k < RPT; ++k)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          if (fabsf(f[k][i]) > 3.402823466e38f) f[k][i] = __uint_as_float(0x7fc00000u);
          amax = fmaxf(amax, fabsf(f[k][i]));
        }
      amax = block_max(amax);
    }
    if (RPT == 1) __syncwarp();                          // every lane has read the old scale
    const int e = max(kv_exponent(amax), e_old);
    const float inv = kv_pow2(-e);
    uint8_t* rows = kv_rows(c, A.layer, page, 0, x);
#pragma unroll
    for (int k = 0; k < RPT; ++k) {
      const int r = first + k * side + r0;
      if (r0 >= side || r >= last) continue;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float* g = f[k] + 8 * h;
        uint2 v;
        v.x = e4m3x4(g[0] * inv, g[1] * inv, g[2] * inv, g[3] * inv);
        v.y = e4m3x4(g[4] * inv, g[5] * inv, g[6] * inv, g[7] * inv);
        *reinterpret_cast<uint2*>(rows + (size_t)r * hd + col + h * half) = v;
      }
    }
    if (first > 0 && e > e_old) {                        // the older rows, at the new scale
      const float down = kv_pow2(max(e_old - e, -126));
      uint4* p = reinterpret_cast<uint4*>(rows);
      for (int i = threadIdx.x; i < first * hd / 16; i += blockDim.x) {
        uint4 v = p[i];
        uint32_t* w = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint32_t lo = e4m3_to_f16x2(w[k] & 0xffffu), hi = e4m3_to_f16x2(w[k] >> 16);
          const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&lo));
          const float2 d = __half22float2(*reinterpret_cast<const __half2*>(&hi));
          w[k] = e4m3x4(a.x * down, a.y * down, d.x * down, d.y * down);
        }
        p[i] = v;
      }
    }
    if (threadIdx.x == 0) *sc = kv_pow2(e);
  }
}

// ---------------------------------------------------------------------------------------------
// page bookkeeping
// ---------------------------------------------------------------------------------------------
// Free pages are those with refs == 0; the lowest ids are handed out first, in the order of the
// sequences, so that the result does not depend on the order in which threads run.
// Measured: 16 beams, five copies of the filled part of a page in 32 layers, 22 MB copied: 12.9 us; a
// compaction that moves 258 MB: 102 us, 5.3 TB/s read and written; grow by a token 1.9 us for 8 sequences, 10 us for
// 1024 over 60000 pages (one CTA goes through the counts twice).

// exclusive block scan over kPlanThreads values; total through *sum
__device__ __forceinline__ int plan_scan(int v, int* s_warp, int* sum) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int incl = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += u;
  }
  __syncthreads();                                     // s_warp may still be read by the last call
  if (lane == 31) s_warp[warp] = incl;
  __syncthreads();
  int w = s_warp[lane];
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, w, o);
    if (lane >= o) w += u;
  }
  *sum = __shfl_sync(0xffffffffu, w, 31);
  const int before = warp ? __shfl_sync(0xffffffffu, w, warp - 1) : 0;
  return before + incl - v;
}

// Calls give(id, rank) for the `want` lowest free ids; returns how many of them there are.
template <typename F>
__device__ __forceinline__ int plan_free(const cats_kv8& c, int want, int* s_warp, F give) {
  int found = 0;
  for (int base = 0; base < c.n_pages && found < want; base += 8 * kPlanThreads) {
    const int id0 = base + 8 * (int)threadIdx.x;
    unsigned free_bits = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (id0 + i < c.n_pages && __ldcg(c.refs + id0 + i) == 0) free_bits |= 1u << i;
    int total;
    int rank = found + plan_scan(__popc(free_bits), s_warp, &total);
    while (free_bits && rank < want) {
      give(id0 + __ffs(free_bits) - 1, rank);
      free_bits &= free_bits - 1;
      ++rank;
    }
    found += total;
  }
  return min(found, want);
}

__global__ void __launch_bounds__(kPlanThreads) k_kv8_grow(const cats_kv8 c, const int* cu, int uniform) {
  pdl_wait();
  __shared__ int s_warp[32];
  __shared__ int s_start[kPlanThreads + 1];
  __shared__ int s_limit;
  const int b = threadIdx.x;
  int len = 0, count = 0, have = 0, need = 0;
  bool grows = false;
  if (b < c.n_seqs) {
    len = c.lens[b];
    count = kv_span(cu, uniform, b).count;
    have = (len + c.page - 1) / c.page;
    if (len < 0 || (long long)len + count > (long long)c.max_pages * c.page) {
      have = 0;
      kv_flag(c, KV_TOO_LONG);
    } else {
      grows = count > 0;
      need = (len + count + c.page - 1) / c.page - have;
    }
  }
  int total;
  const int start = plan_scan(need, s_warp, &total);
  s_start[b] = start;
  if (b == 0) s_limit = total;
  __syncthreads();
  if (total > 0) {
    const int found = plan_free(c, total, s_warp, [](int, int) {});
    // a sequence gets all its pages or none: what is handed out ends before the first that lacks one
    if (need > 0 && start + need > found) {
      atomicMin(&s_limit, start);
      kv_flag(c, KV_POOL_EMPTY);
      grows = false;
    }
    __syncthreads();
    const int limit = s_limit;
    if (grows && need > 0 && start >= limit) grows = false;
    int* table = c.table;
    int* refs = c.refs;
    if (limit > 0)
      plan_free(c, limit, s_warp, [&](int id, int rank) {
        int lo = 0, hi = c.n_seqs - 1;                 // the last sequence that starts at or before rank
        while (lo < hi) {
          const int mid = (lo + hi + 1) >> 1;
          if (s_start[mid] <= rank) lo = mid;
          else hi = mid - 1;
        }
        const int l = c.lens[lo];
        table[(size_t)lo * c.max_pages + (l + c.page - 1) / c.page + rank - s_start[lo]] = id;
        refs[id] = 1;
      });
    __syncthreads();                                   // lens are read above, written below
  }
  if (grows) c.lens[b] = len + count;
  const bool asked = b < c.n_seqs && count > 0;
  kv_set_refused(c, b, asked, asked && !grows);
}

// reorder, step 1: strips of the page table.  Row i of the new table is row parents[i] of the old
// one, which an in-place update can only do column by column with the old column at hand; the
// counts of pages that gain or lose holders change here too.
__device__ __forceinline__ void reorder_table(const cats_kv8& c, const int* parents, int width, int strip, int* sm) {
  const int n = c.n_seqs;
  int* s_children = sm;                                // [n]
  int* s_parent = sm + n;                              // [n]
  int* s_tile = sm + 2 * n;                            // [n][width]
  for (int i = threadIdx.x; i < n; i += blockDim.x) s_children[i] = 0;
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += blockDim.x) {
    int p = parents[i];
    if (p < -1 || p >= n) {
      kv_flag(c, KV_BAD_PARENT);
      p = -1;
    }
    s_parent[i] = p;
    if (p >= 0) atomicAdd(&s_children[p], 1);
  }
  __syncthreads();
  const int j0 = strip * width;
  for (int k = threadIdx.x; k < n * width; k += blockDim.x) {
    const int i = k / width, j = j0 + k - i * width;
    if (j >= c.max_pages) continue;
    const int id = c.table[(size_t)i * c.max_pages + j];
    s_tile[k] = id;
    const int len = c.lens[i], full = len / c.page, held = (len + c.page - 1) / c.page;
    const int change = j < full ? s_children[i] - 1 : (j < held && s_children[i] == 0) ? -1 : 0;
    if (change && id >= 0 && id < c.n_pages) atomicAdd(c.refs + id, change);
  }
  __syncthreads();
  for (int k = threadIdx.x; k < n * width; k += blockDim.x) {
    const int i = k / width, j = j0 + k - i * width;
    if (j >= c.max_pages) continue;
    const int p = s_parent[i];
    c.table[(size_t)i * c.max_pages + j] = p < 0 ? -1 : s_tile[p * width + j - j0];
  }
}
__global__ void __launch_bounds__(256)
k_kv8_reorder_table(const cats_kv8 c, const int* __restrict__ parents, int width) {
  pdl_wait();
  pdl_launch_dependents();
  extern __shared__ int sm[];
  reorder_table(c, parents, width, blockIdx.x, sm);
}

// What the copying CTAs are told: one entry per page to copy.
struct KvCopy {
  int src, dst, rows, pad;
};

// reorder, step 2: lengths, and a page of its own for every child but the first of a parent whose
// last page is still being filled.
// table: this one CTA does step 1 as well (a table that is one strip: a launch less).
__global__ void __launch_bounds__(kPlanThreads)
k_kv8_reorder_plan(const cats_kv8 c, const int* __restrict__ parents, int* n_copies, KvCopy* copies, int table) {
  pdl_wait();
  pdl_launch_dependents();
  if (table) {
    extern __shared__ int sm[];
    reorder_table(c, parents, c.max_pages, 0, sm);
    __threadfence();                                   // the counts' atomics, before they are read below
    __syncthreads();
  }
  __shared__ int s_warp[32];
  __shared__ int s_first[kKvMaxSeqs], s_order[kKvMaxSeqs];
  const int i = threadIdx.x, n = c.n_seqs;
  s_first[i] = n;
  __syncthreads();
  int p = -1, len = 0;
  bool refused = false;
  if (i < n) {
    p = parents[i];
    if (p < 0 || p >= n) p = -1;
    if (p >= 0) {
      len = c.lens[p];
      refused = kv_refused(c, p);
      atomicMin(&s_first[p], i);
    }
  }
  __syncthreads();
  const int rows = len % c.page, at = len / c.page;
  bool more = p >= 0 && rows > 0 && s_first[p] != i && at < c.max_pages;
  int src = -1;
  if (more) {
    src = c.table[(size_t)s_first[p] * c.max_pages + at];
    if (src < 0 || src >= c.n_pages) {                 // the parent lacks the page: so does the child
      more = false;
      c.table[(size_t)i * c.max_pages + at] = -1;
      kv_flag(c, KV_BAD_PAGE);
    }
  }
  int total;
  const int rank = plan_scan(more ? 1 : 0, s_warp, &total);
  if (more) {
    s_order[rank] = i;
    copies[rank] = {src, -1, rows, 0};
  }
  if (i < n) c.lens[i] = len;                          // (every old length was read before the barriers)
  kv_set_refused(c, i, i < n, refused);
  if (i == 0) *n_copies = total;
  if (total == 0) return;
  __syncthreads();
  const int found = plan_free(c, total, s_warp, [&](int id, int r) {
    const int child = s_order[r];
    copies[r].dst = id;
    c.table[(size_t)child * c.max_pages + c.lens[child] / c.page] = id;
    c.refs[id] = 1;
  });
  if (more && rank >= found) {                         // no page left: the child's rows are not there
    c.table[(size_t)i * c.max_pages + at] = -1;
    kv_flag(c, KV_POOL_EMPTY);
  }
}

// 16-byte vectors [0, n) from src to dst by one warp, eight loads in flight per lane
__device__ __forceinline__ void warp_copy(const uint4* src, uint4* dst, int n, int lane) {
  for (int v = lane; v < n; v += 32 * 8) {
    uint4 t[8];
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (v + 32 * k < n) t[k] = __ldcs(src + v + 32 * k);
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (v + 32 * k < n) __stcs(dst + v + 32 * k, t[k]);
  }
}

// The copies of a reorder or a compaction: one warp per (copy, layer, keys / values, head).
__device__ __forceinline__ void kv_copy_pages(const cats_kv8& c, const KvCopy* copies, int n) {
  const int lane = threadIdx.x & 31, heads = 2 * c.n_kv_heads;
  const long long units = (long long)n * c.n_layers * heads;
  const long long warps = (long long)gridDim.x * (blockDim.x >> 5);
  for (long long u = (long long)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5); u < units; u += warps) {
    const int h = (int)(u % heads);
    const long long r = u / heads;
    const int layer = (int)(r % c.n_layers), k = (int)(r / c.n_layers);
    const KvCopy m = copies[k];
    if (m.src < 0 || m.src >= c.n_pages || m.dst < 0 || m.dst >= c.n_pages) {
      if (lane == 0 && m.dst >= 0) kv_flag(c, KV_BAD_PAGE);
      continue;
    }
    const uint4* src = reinterpret_cast<const uint4*>(kv_rows(c, layer, m.src, 0, h));
    uint4* dst = reinterpret_cast<uint4*>(kv_rows(c, layer, m.dst, 0, h));
    warp_copy(src, dst, m.rows * c.head_dim / 16, lane);
    if (lane == 0) *kv_scale(c, layer, m.dst, 0, h) = *kv_scale(c, layer, m.src, 0, h);
  }
}

__global__ void __launch_bounds__(256) k_kv8_copy(const cats_kv8 c, const int* n_copies, const KvCopy* copies) {
  pdl_wait();
  kv_copy_pages(c, copies, *n_copies);
}

// compact, step 1: the k-th free id below the number of live pages receives the k-th live page at
// or above it.  remap[id] = where the page goes.
__global__ void __launch_bounds__(kPlanThreads)
k_kv8_compact_plan(const cats_kv8 c, int* n_live, int* n_moves, KvCopy* moves, int* remap) {
  pdl_wait();
  __shared__ int s_warp[32];
  int mine = 0, live;
  for (int id = threadIdx.x; id < c.n_pages; id += kPlanThreads) mine += c.refs[id] > 0;
  plan_scan(mine, s_warp, &live);
  int holes = 0, movers = 0;
  for (int base = 0; base < c.n_pages; base += 8 * kPlanThreads) {
    const int id0 = base + 8 * (int)threadIdx.x;
    unsigned hole = 0, mover = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int id = id0 + i;
      if (id >= c.n_pages) continue;
      const bool alive = c.refs[id] > 0;
      if (!alive && id < live) hole |= 1u << i;
      if (alive && id >= live) mover |= 1u << i;
      else remap[id] = id;
    }
    int total;
    int rank = holes + plan_scan(__popc(hole), s_warp, &total);
    holes += total;
    for (; hole; hole &= hole - 1) moves[rank++].dst = id0 + __ffs(hole) - 1;
    rank = movers + plan_scan(__popc(mover), s_warp, &total);
    movers += total;
    for (; mover; mover &= mover - 1) {
      moves[rank].src = id0 + __ffs(mover) - 1;
      moves[rank++].rows = c.page;
    }
  }
  __syncthreads();
  for (int k = threadIdx.x; k < movers; k += kPlanThreads) remap[moves[k].src] = moves[k].dst;
  if (threadIdx.x == 0) {
    *n_live = live;
    *n_moves = movers;
  }
}

// compact, step 2: the pages, their counts and the page table
__global__ void __launch_bounds__(256)
k_kv8_compact_move(const cats_kv8 c, const int* n_moves, const KvCopy* moves, const int* __restrict__ remap) {
  pdl_wait();
  const int n = *n_moves;
  const long long t = (long long)blockIdx.x * blockDim.x + threadIdx.x, threads = (long long)gridDim.x * blockDim.x;
  for (long long k = t; k < n; k += threads) {
    const KvCopy m = moves[k];
    c.refs[m.dst] = c.refs[m.src];
    c.refs[m.src] = 0;
  }
  for (long long k = t; k < (long long)c.n_seqs * c.max_pages; k += threads) {
    const int id = c.table[k];
    if (id >= 0 && id < c.n_pages) c.table[k] = remap[id];
  }
  kv_copy_pages(c, moves, n);
}

}  // namespace cats
