// Attention of the newest tokens over the paged 8-bit cache (cats_kv8.cuh).
//
//   out[t, h] = sum_p softmax_p(scale q[t, h] . k[p]) v[p],   p = 0 .. position of t
//
// A decode step reads every code of the cache once and does two multiply-adds with each per query
// head of the group: HBM is the bound as long as a code costs the SM few instructions.  So the query
// heads that share a key head (times the new tokens of the sequence) are the 16 rows of a tensor-core
// tile (mma.m16n8k16, half precision in, fp32 out), and codes become half precision, exactly, two per
// instruction.  tcgen05 tiles have 128 rows, of which a decode step fills 1 to 16; with this shape the
// codes go from shared memory to the tensor cores through registers, where they are converted anyway.
//
// Precision: q is scaled by a power of two per row (largest magnitude just below 1) so that half
// precision holds fp16 and bf16 queries exactly (but for elements 2^-14 below the row's largest);
// softmax weights are rounded to half precision, 2^-11, below the rounding of a 16-bit result.
// fp32 queries and weights are each split in two halves (22 bits) and take two products.
// The scale of V's page is a power of two and joins the exponent: weights are
// p' = exp2(s + ev - m) with m the running maximum of s + ev, so that p' <= 1 whatever the scales,
// and the softmax's sum is that of p' 2^-ev.
//
// Work: 128 positions (a unit, 16 for each of the 8 warps) of one row tile of one key head.  All
// units of the call in a row - sequences, heads, tiles, positions - are dealt out to one CTA per SM in
// equal, contiguous shares, whatever the lengths of the sequences, and computed from the lengths on
// the device; a (head, tile) that one CTA has whole is written at once, the parts of the others are
// joined by a second kernel.
#pragma once

#include "cats_kv8.cuh"

namespace cats {

constexpr int kAttnWarps = 8;
constexpr int kAttnThreads = kAttnWarps * 32;
constexpr int kAttnStages = 4;                          // tiles a warp has in flight (one of them in use)
constexpr int kAttnTile = 16;                           // positions of a warp's tile
constexpr int kAttnUnit = kAttnWarps * kAttnTile;       // positions of a unit
constexpr int kAttnRows = 16;                           // rows of a tile: (token, query head of the group)
constexpr int kAttnStageBytes = 2 * kAttnTile * 128 + 16;  // keys, values (rows 128 bytes apart), two scales

template <typename T>
struct KvAttnArgs {
  const T* q;             // [tokens, nh, hd], tokens q_ld elements apart
  long long q_ld;
  T* out;                 // [tokens, nh, hd]
  float* parts;           // [CTAs][2][kAttnRows][hd + 2] parts of (head, tile)s that several CTAs share
  const int* cu;
  int uniform, tokens, nh, layer, ctas;
  float scale;            // of the scores, times log2(e)
};

__host__ __device__ inline size_t attn_part_floats(int hd) { return (size_t)kAttnRows * (hd + 2); }
__host__ __device__ inline size_t attn_smem(int hd) {
  return (size_t)kAttnWarps * kAttnStages * kAttnStageBytes + sizeof(float) * kAttnWarps * kAttnRows * (hd + 4) +
         sizeof(float) * 2 * kAttnWarps * kAttnRows;
}

__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
// c += a (16 x 16, row) * b (16 x 8, col)
__device__ __forceinline__ void mma16816(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t half2_bits(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// what rounding (lo, hi) to half precision left over, as half precision
__device__ __forceinline__ uint32_t half2_rest(float lo, float hi, uint32_t rounded) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&rounded));
  return half2_bits(lo - f.x, hi - f.y);
}
// Row r of a tile lies at r * 128 bytes, its 16-byte chunks exchanged by r so that the eight-byte
// reads below (four rows at a time, 32 bytes of each) use every bank once: rows {0, 1, 2, 3},
// {4 .. 7} for the keys and {0, 2, 4, 6}, {1, 3, 5, 7} for the values have different exchanges.
__device__ __forceinline__ uint32_t attn_swizzle(int row, uint32_t byte) {
  return (uint32_t)row * 128 + (byte ^ ((((uint32_t)row & 3) ^ (((uint32_t)row >> 2) & 1)) << 5));
}

// Units of every sequence, summed up: pre[b] = units before sequence b, pre[n_seqs] = all.
// Called by a CTA of kAttnThreads threads; ends with a barrier.
struct AttnSeq {
  int len, count, first, tiles, units;                  // units of one tile of one head
};
template <typename T>
__device__ __forceinline__ AttnSeq attn_seq(const cats_kv8& c, const KvAttnArgs<T>& A, int b) {
  const KvSpan sp = kv_span(A.cu, A.uniform, b);
  const int len = c.lens[b];
  AttnSeq s = {len, sp.count, sp.first, 0, 0};
  const bool fits = len >= 0 && len <= c.max_pages * c.page && sp.first >= 0 &&
                    (long long)sp.first + sp.count <= A.tokens;
  if (fits && sp.count > 0) {
    s.tiles = (int)(((long long)sp.count * (A.nh / c.n_kv_heads) + kAttnRows - 1) / kAttnRows);
    s.units = (len + kAttnUnit - 1) / kAttnUnit;
  }
  return s;
}
template <typename T>
__device__ __forceinline__ void attn_prefix(const cats_kv8& c, const KvAttnArgs<T>& A, long long* pre, long long* s_warp) {
  constexpr int kPer = kKvMaxSeqs / kAttnThreads;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  long long mine[kPer], sum = 0;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int b = threadIdx.x * kPer + i;
    mine[i] = 0;
    if (b < c.n_seqs) {
      const AttnSeq s = attn_seq(c, A, b);
      mine[i] = (long long)s.units * s.tiles * c.n_kv_heads;
    }
    sum += mine[i];
  }
  long long incl = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long v = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += v;
  }
  if (lane == 31) s_warp[warp] = incl;
  __syncthreads();
  long long before = incl - sum;
  for (int w = 0; w < warp; ++w) before += s_warp[w];
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int b = threadIdx.x * kPer + i;
    if (b <= c.n_seqs) pre[b] = before;
    before += mine[i];
  }
  if (threadIdx.x == kAttnThreads - 1 && c.n_seqs == kKvMaxSeqs) pre[kKvMaxSeqs] = before;
  __syncthreads();
}

// Where a unit lies: sequence, head, tile and number of the unit within them.
struct AttnPlace {
  int b, head, tile, unit, units;
};
template <typename T>
__device__ __forceinline__ AttnPlace attn_place(const cats_kv8& c, const KvAttnArgs<T>& A, const long long* pre,
                                                long long w, AttnSeq* seq) {
  int lo = 0, hi = c.n_seqs - 1;                         // last sequence that starts at or before w
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (pre[mid] <= w) lo = mid;
    else hi = mid - 1;
  }
  const AttnSeq s = attn_seq(c, A, lo);
  const unsigned r = (unsigned)(w - pre[lo]);            // below 2^32: checked at launch
  AttnPlace p;
  p.b = lo;
  const unsigned at = r / (unsigned)s.units;
  p.unit = (int)(r - at * (unsigned)s.units);
  p.head = (int)(at / (unsigned)s.tiles);
  p.tile = (int)(at - (unsigned)p.head * (unsigned)s.tiles);
  p.units = s.units;
  *seq = s;
  return p;
}
// CTAs that get a share (at least one unit each), and where the share of CTA c begins
__device__ __forceinline__ int attn_ctas(long long total, int ctas) { return total < ctas ? (int)total : ctas; }
__device__ __forceinline__ long long attn_share(long long total, int c, int ctas) { return total * c / ctas; }
// the CTA whose share holds unit w
__device__ __forceinline__ int attn_owner(long long total, long long w, int ctas) {
  return (int)(((w + 1) * ctas - 1) / total);
}

// O += P V for the warp's tile.  GUARD: some row must not see all of the tile's positions and V holds
// a NaN; zero weights would turn it into NaN in rows that do not see it, so NaN codes are taken out
// of the product and added to the rows that do see them (`seen`, weights 1 and 0).
template <int HD, bool SPLIT, bool GUARD>
__device__ __forceinline__ void attn_pv(float (*o)[4], const uint32_t* p, const uint32_t* p_lo, const uint32_t* seen,
                                        const unsigned char* vt, int g, int t) {
  auto group = [&](uint32_t r0, uint32_t r1, uint32_t r2, uint32_t r3, float (*acc)[4]) {
    // four channels of four positions: byte pairs (position, next position) of each channel
    const uint32_t w[4] = {__byte_perm(r0, r1, 0x5140), __byte_perm(r2, r3, 0x5140), __byte_perm(r0, r1, 0x7362),
                           __byte_perm(r2, r3, 0x7362)};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      uint32_t c0 = (w[j & 2] >> (16 * (j & 1))) & 0xffffu, c1 = (w[(j & 2) + 1] >> (16 * (j & 1))) & 0xffffu;
      if (GUARD) {
        auto nan_bytes = [](uint32_t x) { return ((((x & 0x7f7fu) + 0x0101u) & 0x8080u) >> 7) * 0xffu; };
        const uint32_t n0 = nan_bytes(c0), n1 = nan_bytes(c1);
        float hit[4] = {0.f, 0.f, 0.f, 0.f};
        mma16816(hit, seen, e4m3_to_f16x2(n0 & 0x3838u), e4m3_to_f16x2(n1 & 0x3838u));   // 0x38 is 1.0
        c0 &= ~n0;
        c1 &= ~n1;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (hit[i] > 0.f) acc[j][i] = __uint_as_float(0x7fc00000u);
      }
      const uint32_t b0 = e4m3_to_f16x2(c0), b1 = e4m3_to_f16x2(c1);
      mma16816(acc[j], p, b0, b1);
      if (SPLIT) mma16816(acc[j], p_lo, b0, b1);
    }
  };
  const int r[4] = {2 * t, 2 * t + 1, 8 + 2 * t, 9 + 2 * t};
#pragma unroll
  for (int q = 0; q < HD / 64; ++q) {
    uint2 v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = *reinterpret_cast<const uint2*>(vt + attn_swizzle(r[i], 64 * q + 8 * g));
    group(v[0].x, v[1].x, v[2].x, v[3].x, o + 8 * q);
    group(v[0].y, v[1].y, v[2].y, v[3].y, o + 8 * q + 4);
  }
  if (HD % 64) {
    uint32_t v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = *reinterpret_cast<const uint32_t*>(vt + attn_swizzle(r[i], HD / 64 * 64 + 4 * g));
    group(v[0], v[1], v[2], v[3], o + 8 * (HD / 64));
  }
}

template <typename T, int HD>
__global__ void __launch_bounds__(kAttnThreads, 1) k_kv8_attend(const cats_kv8 c, const KvAttnArgs<T> A) {
  constexpr bool SPLIT = sizeof(T) == 4;
  constexpr int KS = HD / 16;                            // k-steps of the score product
  constexpr int NT = HD / 8;                             // column tiles of the output
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ long long s_pre[kKvMaxSeqs + 1];
  __shared__ long long s_warp[kAttnWarps];
  pdl_wait();
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  unsigned char* ring = smem + (size_t)warp * kAttnStages * kAttnStageBytes;
  float* s_o = reinterpret_cast<float*>(smem + (size_t)kAttnWarps * kAttnStages * kAttnStageBytes);
  float* s_ml = s_o + kAttnWarps * kAttnRows * (HD + 4);
  const uint32_t ring_u32 = (uint32_t)__cvta_generic_to_shared(ring);

  attn_prefix(c, A, s_pre, s_warp);
  const long long total = s_pre[c.n_seqs];
  const int ctas = attn_ctas(total, A.ctas);
  if ((int)blockIdx.x >= ctas) return;
  const long long w0 = attn_share(total, blockIdx.x, ctas), w1 = attn_share(total, blockIdx.x + 1, ctas);
  const int group = A.nh / c.n_kv_heads;

  // ---- loader: lane i of the warp knows where unit `base + i` lies and which page its tile is in --
  long long base = w0;
  int d_id = -1, d_row = 0, d_rows = 0, d_head = 0;      // page, row in it, rows to load, head
  auto look = [&]() {
    const long long w = base + lane;
    d_id = -1;
    d_rows = 0;
    if (w < w1) {
      AttnSeq s;
      const AttnPlace p = attn_place(c, A, s_pre, w, &s);
      const int last = min(s.count - 1, (p.tile * kAttnRows + kAttnRows - 1) / group);
      const int end = min(s.len, s.len - s.count + last + 1);        // positions that the tile's rows see
      const int kb = p.unit * kAttnUnit + warp * kAttnTile;
      d_head = p.head;
      d_row = kb % c.page;
      d_rows = min(max(end - kb, 0), kAttnTile);
      if (d_rows > 0) {
        d_id = c.table[(size_t)p.b * c.max_pages + kb / c.page];
        if (d_id < 0 || d_id >= c.n_pages) {
          kv_flag(c, KV_BAD_PAGE);
          d_rows = 0;
        }
      }
    }
  };
  look();
  int stage_in = 0;
  long long w_in = w0;
  auto issue = [&]() {
    if (w_in < w1) {
      if (w_in - base == 32) {
        base += 32;
        look();
      }
      const int src = (int)(w_in - base);
      const int rows = __shfl_sync(0xffffffffu, d_rows, src);
      const uint32_t st = ring_u32 + stage_in * kAttnStageBytes;
      if (lane == 0)
        *reinterpret_cast<int*>(ring + stage_in * kAttnStageBytes + 2 * kAttnTile * 128 + 8) = rows;
      if (rows > 0) {
        const int id = __shfl_sync(0xffffffffu, d_id, src), row = __shfl_sync(0xffffffffu, d_row, src);
        const int head = __shfl_sync(0xffffffffu, d_head, src);
        const uint8_t* kp = kv_rows(c, A.layer, id, 0, head) + (size_t)row * HD;
        const uint8_t* vp = kp + (size_t)c.n_kv_heads * kv_block(c);
#pragma unroll
        for (int i = 0; i < 2 * HD / 32; ++i) {          // 16-byte chunks: the keys', then the values'
          const int n = lane + 32 * i;
          const int kv = n / HD, m = n - kv * HD, r = m / (HD / 16), ch = m - r * (HD / 16);
          const uint8_t* from = (kv ? vp : kp) + (size_t)m * 16;
          const uint32_t to = st + kv * kAttnTile * 128 + attn_swizzle(r, ch * 16);
          const int bytes = r < rows ? 16 : 0;           // the rest is filled with zeros, not read
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(r < rows ? from : kp), "r"(bytes)
                       : "memory");
        }
        if (lane < 2)
          asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(st + 2 * kAttnTile * 128 + 4 * lane),
                       "l"(kv_scale(c, A.layer, id, lane, head))
                       : "memory");
      }
      ++w_in;
      stage_in = stage_in + 1 == kAttnStages ? 0 : stage_in + 1;
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  for (int i = 0; i < kAttnStages - 1; ++i) issue();

  // ---- consumer ------------------------------------------------------------------------------------
  uint32_t qa[KS][4], qb[SPLIT ? KS : 1][4];
  float o[NT][4];
  float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f, f0 = 0.f, f1 = 0.f;
  int lim0 = 0, lim1 = 0, lim_min = 0;
  AttnSeq seq;
  AttnPlace at = attn_place(c, A, s_pre, w0, &seq);
  bool first_seg = true, begins_here = at.unit == 0, fresh = true;
  int stage = 0;
  for (long long w = w0; w < w1; ++w) {
    asm volatile("cp.async.wait_group %0;" ::"n"(kAttnStages - 2) : "memory");
    __syncwarp();
    issue();

    if (fresh) {                                         // a new (sequence, head, tile): its queries
      fresh = false;
      const int rows = min(kAttnRows, seq.count * group - at.tile * kAttnRows);
      float q[2][HD / 32][8];
      float top[2] = {0.f, 0.f};
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int r = at.tile * kAttnRows + g + 8 * i, tok = r / group, hq = at.head * group + r - tok * group;
        const bool on = g + 8 * i < rows;
        const T* src = A.q + (size_t)(seq.first + tok) * A.q_ld + (size_t)hq * HD + 8 * t;
#pragma unroll
        for (int p = 0; p < HD / 32; ++p) {
#pragma unroll
          for (int k = 0; k < 8; ++k) q[i][p][k] = 0.f;
          if (on) load8_cached(src + 32 * p, q[i][p]);
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const float a = fabsf(q[i][p][k]);
            if (a <= 3.402823466e38f) top[i] = fmaxf(top[i], a);
          }
        }
        const int lim = on ? min(seq.len, seq.len - seq.count + tok + 1) : 0;
        if (i) lim1 = lim;
        else lim0 = lim;
      }
      lim_min = min(seq.len, seq.len - seq.count + at.tile * kAttnRows / group + 1);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], 1));
        top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], 2));
        const int e = top[i] > 0.f ? min(max(kv_exp_of(top[i]) + 1, -126), 126) : 0;
        const float inv = kv_pow2(-e), f = kv_pow2(e) * A.scale;
        if (i) f1 = f;
        else f0 = f;
#pragma unroll
        for (int p = 0; p < HD / 32; ++p)
#pragma unroll
          for (int k = 0; k < 8; ++k) q[i][p][k] *= inv;
      }
#pragma unroll
      for (int p = 0; p < HD / 32; ++p)
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const float* f = q[x & 1][p] + 4 * e + (x & 2);
            qa[2 * p + e][x] = half2_bits(f[0], f[1]);
            if (SPLIT) qb[SPLIT ? 2 * p + e : 0][x] = half2_rest(f[0], f[1], qa[2 * p + e][x]);
          }
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[n][i] = 0.f;
      m0 = m1 = -INFINITY;
      l0 = l1 = 0.f;
    }

    const int kb = at.unit * kAttnUnit + warp * kAttnTile;
    const unsigned char* kt = ring + stage * kAttnStageBytes;
    if (*reinterpret_cast<const int*>(kt + 2 * kAttnTile * 128 + 8) > 0) {
      const unsigned char* vt = kt + kAttnTile * 128;
      const float2 sc = *reinterpret_cast<const float2*>(kt + 2 * kAttnTile * 128);
      float s[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
      for (int p = 0; p < HD / 32; ++p) {
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          const uint2 k = *reinterpret_cast<const uint2*>(kt + attn_swizzle(8 * n + g, 32 * p + 8 * t));
          const uint32_t b0 = e4m3_to_f16x2(k.x & 0xffffu), b1 = e4m3_to_f16x2(k.x >> 16);
          const uint32_t b2 = e4m3_to_f16x2(k.y & 0xffffu), b3 = e4m3_to_f16x2(k.y >> 16);
          mma16816(s[n], qa[2 * p], b0, b1);
          mma16816(s[n], qa[2 * p + 1], b2, b3);
          if (SPLIT) {
            mma16816(s[n], qb[SPLIT ? 2 * p : 0], b0, b1);
            mma16816(s[n], qb[SPLIT ? 2 * p + 1 : 0], b2, b3);
          }
        }
      }
      const int ev = kv_exp_of(sc.y);
      const float evf = (float)ev;
      const bool cut = kb + kAttnTile > lim_min;         // some row does not see all of the tile
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          s[n][i] *= sc.x * (i < 2 ? f0 : f1);
          if (cut && kb + 8 * n + 2 * t + (i & 1) >= (i < 2 ? lim0 : lim1)) s[n][i] = -INFINITY;
        }
      float n0 = fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[1][0], s[1][1]));
      float n1 = fmaxf(fmaxf(s[0][2], s[0][3]), fmaxf(s[1][2], s[1][3]));
      n0 = fmaxf(n0, __shfl_xor_sync(0xffffffffu, n0, 1));
      n1 = fmaxf(n1, __shfl_xor_sync(0xffffffffu, n1, 1));
      n0 = fmaxf(n0, __shfl_xor_sync(0xffffffffu, n0, 2));
      n1 = fmaxf(n1, __shfl_xor_sync(0xffffffffu, n1, 2));
      n0 += evf;
      n1 += evf;
      if (__any_sync(0xffffffffu, n0 > m0 || n1 > m1)) {
        n0 = fmaxf(n0, m0);
        n1 = fmaxf(n1, m1);
        const float x0 = m0 == -INFINITY ? 0.f : ex2(m0 - n0), x1 = m1 == -INFINITY ? 0.f : ex2(m1 - n1);
        m0 = n0;
        m1 = n1;
        l0 *= x0;
        l1 *= x1;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          o[n][0] *= x0;
          o[n][1] *= x0;
          o[n][2] *= x1;
          o[n][3] *= x1;
        }
      }
      // (m - ev) is the same for all tiles whose pages have the same ev: its rounding cancels
      const float u0 = m0 == -INFINITY ? 0.f : m0 - evf, u1 = m1 == -INFINITY ? 0.f : m1 - evf;
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) s[n][i] = ex2(s[n][i] - (i < 2 ? u0 : u1));
      const float vi = kv_pow2(-ev);
      l0 = fmaf((s[0][0] + s[0][1]) + (s[1][0] + s[1][1]), vi, l0);
      l1 = fmaf((s[0][2] + s[0][3]) + (s[1][2] + s[1][3]), vi, l1);
      uint32_t p[4], pl[4];
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const float* f = s[x >> 1] + 2 * (x & 1);
        p[x] = half2_bits(f[0], f[1]);
        pl[x] = SPLIT ? half2_rest(f[0], f[1], p[x]) : 0u;
      }
      bool guard = false;
      if (cut) {
        bool nan = false;
#pragma unroll
        for (int i = 0; i < HD / 32; ++i) {
          const uint4 v = *reinterpret_cast<const uint4*>(vt + attn_swizzle((lane + 32 * i) / (HD / 16), (lane + 32 * i) % (HD / 16) * 16));
          const uint32_t x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
          for (int k = 0; k < 4; ++k) nan |= (((x[k] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) != 0;
        }
        guard = __any_sync(0xffffffffu, nan);
      }
      if (guard) {
        uint32_t seen[4];
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const int k = kb + 8 * (x >> 1) + 2 * t, lim = (x & 1) ? lim1 : lim0;
          seen[x] = half2_bits(k < lim ? 1.f : 0.f, k + 1 < lim ? 1.f : 0.f);
        }
        attn_pv<HD, SPLIT, true>(o, p, pl, seen, vt, g, t);
      } else {
        attn_pv<HD, SPLIT, false>(o, p, pl, nullptr, vt, g, t);
      }
    }
    stage = stage + 1 == kAttnStages ? 0 : stage + 1;
    ++at.unit;

    if (at.unit == at.units || w + 1 == w1) {            // the segment ends here: join the warps
      const int rows = min(kAttnRows, seq.count * group - at.tile * kAttnRows);
      l0 += __shfl_xor_sync(0xffffffffu, l0, 1);
      l1 += __shfl_xor_sync(0xffffffffu, l1, 1);
      l0 += __shfl_xor_sync(0xffffffffu, l0, 2);
      l1 += __shfl_xor_sync(0xffffffffu, l1, 2);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int r = g + 8 * i;
        if (r >= rows) continue;
        float* dst = s_o + (size_t)(warp * kAttnRows + r) * (HD + 4);
        if (t == 0) {
          s_ml[warp * kAttnRows + r] = i ? m1 : m0;
          s_ml[kAttnWarps * kAttnRows + warp * kAttnRows + r] = i ? l1 : l0;
        }
        // column tile 8 q + j holds channels 64 q + 8 n + j (n = 2 t, 2 t + 1), the rest 4 n + j
#pragma unroll
        for (int q = 0; q < HD / 64; ++q)
#pragma unroll
          for (int x = 0; x < 2; ++x)
#pragma unroll
            for (int k = 0; k < 8; k += 4)
              *reinterpret_cast<float4*>(dst + 64 * q + 16 * t + 8 * x + k) =
                  make_float4(o[8 * q + k][2 * i + x], o[8 * q + k + 1][2 * i + x], o[8 * q + k + 2][2 * i + x],
                              o[8 * q + k + 3][2 * i + x]);
        if (HD % 64) {
          constexpr int n = 8 * (HD / 64);
#pragma unroll
          for (int x = 0; x < 2; ++x)
            *reinterpret_cast<float4*>(dst + HD / 64 * 64 + 8 * t + 4 * x) =
                make_float4(o[n][2 * i + x], o[n + 1][2 * i + x], o[n + 2][2 * i + x], o[n + 3][2 * i + x]);
        }
      }
      __syncthreads();
      const bool whole = begins_here && at.unit == at.units;
      float* part = A.parts + (size_t)(blockIdx.x * 2 + (first_seg ? 0 : 1)) * attn_part_floats(HD);
      for (int e = threadIdx.x; e < rows * (HD / 4); e += kAttnThreads) {
        const int r = e / (HD / 4), d = (e - r * (HD / 4)) * 4;
        float top = -INFINITY, sum = 0.f;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int x = 0; x < kAttnWarps; ++x) top = fmaxf(top, s_ml[x * kAttnRows + r]);
#pragma unroll
        for (int x = 0; x < kAttnWarps; ++x) {
          const float mx = s_ml[x * kAttnRows + r];
          const float lx = s_ml[(kAttnWarps + x) * kAttnRows + r];
          if (mx == -INFINITY && lx == 0.f) continue;    // saw nothing (a NaN sum goes on)
          const float f = ex2(mx - (top == -INFINITY ? 0.f : top));
          const float4 u = *reinterpret_cast<const float4*>(s_o + (size_t)(x * kAttnRows + r) * (HD + 4) + d);
          sum = fmaf(lx, f, sum);
          v.x = fmaf(u.x, f, v.x);
          v.y = fmaf(u.y, f, v.y);
          v.z = fmaf(u.z, f, v.z);
          v.w = fmaf(u.w, f, v.w);
        }
        if (whole) {
          const int rr = at.tile * kAttnRows + r, tok = rr / group, hq = at.head * group + rr - tok * group;
          const float inv = sum == 0.f ? 0.f : 1.f / sum;
          T* dst = A.out + ((size_t)(seq.first + tok) * A.nh + hq) * HD + d;
          dst[0] = VecT<T>::from_f(v.x * inv);
          dst[1] = VecT<T>::from_f(v.y * inv);
          dst[2] = VecT<T>::from_f(v.z * inv);
          dst[3] = VecT<T>::from_f(v.w * inv);
        } else {
          float* dst = part + (size_t)r * (HD + 2);
          *reinterpret_cast<float2*>(dst + d) = make_float2(v.x, v.y);
          *reinterpret_cast<float2*>(dst + d + 2) = make_float2(v.z, v.w);
          if (d == 0) *reinterpret_cast<float2*>(dst + HD) = make_float2(top, sum);
        }
      }
      __syncthreads();
      first_seg = false;
      fresh = true;
      if (w + 1 < w1) at = attn_place(c, A, s_pre, w + 1, &seq);
      begins_here = true;
    }
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
}

template <typename T, int HD>
__device__ __forceinline__ void attn_join_row(const cats_kv8& c, const KvAttnArgs<T>& A, const long long* s_pre,
                                              long long row, int lane) {
  const int tok = (int)(row / A.nh), hq = (int)(row - (long long)tok * A.nh), group = A.nh / c.n_kv_heads;
  int b;
  if (!A.cu) {
    b = tok / A.uniform;
  } else {
    int lo = 0, hi = c.n_seqs - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (__ldg(A.cu + mid) <= tok) lo = mid;
      else hi = mid - 1;
    }
    b = lo;
  }
  const AttnSeq s = attn_seq(c, A, b);
  const int i = tok - s.first;
  if (i < 0 || i >= s.count) return;                     // a row that belongs to no sequence
  T* dst = A.out + (size_t)row * HD;
  if (s.units == 0 || s.tiles == 0) {
    if (lane == 0 && i == 0 && (s.len < 0 || s.len > c.max_pages * c.page)) kv_flag(c, KV_TOO_LONG);
    if (lane == 0 && i == 0 && (s.first < 0 || (long long)s.first + s.count > A.tokens)) kv_flag(c, KV_BAD_SPAN);
    for (int d = lane; d < HD; d += 32) dst[d] = VecT<T>::from_f(0.f);
    return;
  }
  const int head = hq / group, at = i * group + hq - head * group, tile = at / kAttnRows, r = at - tile * kAttnRows;
  const long long total = s_pre[c.n_seqs];
  const long long u0 = s_pre[b] + ((long long)head * s.tiles + tile) * s.units, u1 = u0 + s.units - 1;
  const int ctas = attn_ctas(total, A.ctas), c0 = attn_owner(total, u0, ctas), c1 = attn_owner(total, u1, ctas);
  if (c0 == c1) return;                                  // written already
  float top = -INFINITY;
  auto part = [&](int x) {
    const int slot = attn_share(total, x, ctas) >= u0 ? 0 : 1;
    return A.parts + (size_t)(2 * x + slot) * attn_part_floats(HD) + (size_t)r * (HD + 2);
  };
  for (int x = c0 + lane; x <= c1; x += 32) top = fmaxf(top, part(x)[HD]);
#pragma unroll
  for (int w = 16; w > 0; w >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
  const float ref = top == -INFINITY ? 0.f : top;
  float sum = 0.f, v[HD / 32];
#pragma unroll
  for (int k = 0; k < HD / 32; ++k) v[k] = 0.f;
  for (int x = c0; x <= c1; ++x) {
    const float* p = part(x);
    const float m = p[HD], l = p[HD + 1];
    if (m == -INFINITY && l == 0.f) continue;
    const float f = ex2(m - ref);
    sum = fmaf(l, f, sum);
#pragma unroll
    for (int k = 0; k < HD / 32; ++k) v[k] = fmaf(p[lane + 32 * k], f, v[k]);
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
  for (int k = 0; k < HD / 32; ++k) dst[lane + 32 * k] = VecT<T>::from_f(v[k] * inv);
}

// Joins the parts of the (head, tile)s that several CTAs share: one warp per (token, query head).
// Rows without any position become zeros here.
template <typename T, int HD>
__global__ void __launch_bounds__(kAttnThreads) k_kv8_attend_join(const cats_kv8 c, const KvAttnArgs<T> A) {
  __shared__ long long s_pre[kKvMaxSeqs + 1];
  __shared__ long long s_warp[kAttnWarps];
  pdl_wait();
  attn_prefix(c, A, s_pre, s_warp);
  const int lane = threadIdx.x & 31;
  const long long rows = (long long)A.tokens * A.nh, step = (long long)gridDim.x * kAttnWarps;
  for (long long row = (long long)blockIdx.x * kAttnWarps + (threadIdx.x >> 5); row < rows; row += step)
    attn_join_row<T, HD>(c, A, s_pre, row, lane);
}

}  // namespace cats
