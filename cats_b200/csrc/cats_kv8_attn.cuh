// Attention of the newest tokens over the paged 8-bit cache (cats_kv8.cuh).
//
//   out[t, h] = sum_p softmax_p(scale q[t, h] . k[p]) v[p],   p = 0 .. position of t
//
// A decode step reads every code of the cache once and does two multiply-adds with each per query
// head of the group: HBM is the bound as long as a code costs the SM few instructions.  So codes
// become half precision, exactly, two per instruction, and go to the tensor cores (mma.m16n8k16, fp32
// accumulation) as the 16-row operand, of which nothing is padding: positions x channels for
// S^T = K Q^T, channels x positions for O^T = V^T P^T.  The query heads that share a key head (times
// the new tokens of the sequence) are the eight columns.  tcgen05 tiles have 128 rows and take their
// operands from shared memory, where converted codes would first have to be written back.
//
// Precision: q is scaled by a power of two per row (largest magnitude just below 1) so that half
// precision holds fp16 and bf16 queries exactly (but for elements 2^-14 below the row's largest);
// softmax weights are rounded to half precision, 2^-11, below the rounding of a 16-bit result.
// fp32 queries and weights are each split in two halves (22 bits) and take two products.
// The scale of V's page is a power of two and joins the exponent: weights are
// p' = exp2(s - m + ev - ec) with m the running maximum of s, ev the page's exponent and ec the one that the
// accumulators are held at; the softmax's sum is that of p' 2^(ec - ev).  ec follows ev when they are more than
// kAttnSpan apart (the accumulators are rescaled, exactly), so that what half precision loses of a weight does not
// depend on the scales of other pages: 2^-11 of it, or 2^-21 of the largest weight of the row for a small one.
//
// Work: a unit is 16 positions for each warp of one tile (8, 16 or 32 rows) of one key head.  All units
// of the call in a row - sequences, heads, tiles, positions - are dealt out to one CTA per SM in
// equal, contiguous shares, whatever the lengths of the sequences, and computed from the lengths on
// the device; a (head, tile) that one CTA has whole is written at once, the parts of the others are
// joined by the CTA that finishes last (nobody waits).
//
// Measured (head_dim 128, 8 key heads): 16 sequences of 32768 positions 171 us, 6.27 TB/s of codes (0.95
// of a plain copy's rate); 32 sequences of 1000 .. 32000, 603 MB: 110 to 115 us replayed from a graph, 120 to 124 us a
// call; 8 sequences of 512 .. 1536: 14.3 us, on 80 of 148 SMs (units of 256 positions, of which joining two parts
// costs as much, leave most segments to one CTA), one sequence of 640 with 32 key heads: 9.8 us on 32 of them.
#pragma once

#include "cats_kv8.cuh"

namespace cats {

constexpr int kAttnTile = 16;                           // positions of a warp's tile
constexpr int kAttnStageBytes = 2 * kAttnTile * 128;    // keys, values (rows 128 bytes apart)
constexpr float kAttnSlack = 8.f;                       // see the running maximum
// How far a page's exponent may be from the accumulators'.  (These go down by up to 84, the range of scales; a sum of
// 2^21 products of weights up to 2^12 and codes up to 2^9 is still a number of fp32 then.)
constexpr int kAttnSpan = 4;
constexpr int kAttnNoExp = -1000;                       // nothing in the accumulators yet
// (a scale outside the cache's range counts as the nearest inside)
__device__ __forceinline__ int attn_exp_of(float scale) { return min(max(kv_exp_of(scale), kKvExpMin), kKvExpMax); }

// NQ columns of eight rows ((token, query head of the group) pairs) per tile.  Eight rows leave room
// for 16 warps of 128 registers, which hide the latency of the chain load - convert - multiply -
// exponential - multiply best; 16 rows need twice the accumulators; 32 rows (many new tokens: the
// conversions are shared by four products) leave no registers for the queries, which are read from
// shared memory then.
template <int NQ>
struct AttnShape {
  static constexpr int kRows = 8 * NQ;
  static constexpr int kWarps = NQ == 1 || NQ == 16 ? 16 : 8;
  static constexpr int kThreads = 32 * kWarps;
  static constexpr int kStages = NQ == 1 ? 3 : 6;       // tiles a warp has in its ring (one of them in use)
  static constexpr int kUnit = NQ == 1 ? 256 : 128;     // positions of a unit (a tile for each warp up to NQ = 4)
  static constexpr int kJoin = 512 / kUnit;             // joining parts takes about as long as 512 positions
  static constexpr int kSwitch = 768 / kUnit;           // going over to another segment, as long as 768
  static constexpr bool kQueriesShared = NQ == 4;
};

template <typename T>
struct KvAttnArgs {
  const T* q;             // [tokens, nh, hd], tokens q_ld elements apart
  long long q_ld;
  T* out;                 // [tokens, nh, hd]
  float* parts;           // [CTAs][2][rows of a tile][hd + 2] parts of (head, tile)s that several CTAs share
  int* counters;          // [CTAs], zero between calls
  const int* cu;
  int uniform, tokens, nh, layer, ctas, wait_kc;
  float scale;            // of the scores, times log2(e)
};

// Rows of a key head, (new tokens) x (query heads per key head), on average over the sequences: what
// the kernels are chosen by, and the rows that a part of theirs can have.
__host__ __device__ inline long long attn_rows(const cats_kv8& c, int tokens, int nh) {
  return ((long long)tokens + c.n_seqs - 1) / c.n_seqs * (nh / c.n_kv_heads);
}
constexpr int kAttnFewRows = 16, kAttnSomeRows = 32;    // up to here 8 or 16, 32 rows a tile
inline int attn_part_rows(const cats_kv8& c, int tokens, int nh) {
  return attn_rows(c, tokens, nh) > kAttnFewRows ? 128 : 16;
}
__host__ __device__ inline size_t attn_part_floats(int rows, int hd) { return (size_t)rows * (hd + 2); }
template <int NQ>
constexpr size_t attn_smem() {
  return 128 + (size_t)AttnShape<NQ>::kWarps * (AttnShape<NQ>::kStages * (kAttnStageBytes + 16) + 2 * 8 * sizeof(float)) +
         (AttnShape<NQ>::kQueriesShared ? NQ * 128 / 32 * 32 * sizeof(uint4) : 0);
}

__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
// an 8 x 8 matrix of 16-bit values, two of a row per lane, transposed
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
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

// What the CTA knows of the sequences (shared memory).
struct AttnTable {
  int pre[kKvMaxSeqs + 1];                              // units before sequence b; all of them
  int cost[kKvMaxSeqs + 1];                             // CTAs before sequence b where they are dealt out by
                                                        // segments, else the cost (below) of what is before it
  int len[kKvMaxSeqs], first[kKvMaxSeqs], count[kKvMaxSeqs];
};
struct AttnSeq {
  int len, count, first, tiles, units;                  // tiles of a key head, units of a tile
};
template <int NQ>
__device__ __forceinline__ AttnSeq attn_seq(const AttnTable& tab, int b, int group) {
  AttnSeq s = {tab.len[b], tab.count[b], tab.first[b], 0, 0};
  s.tiles = (int)(((long long)s.count * group + 8 * NQ - 1) / (8 * NQ));
  s.units = (s.len + AttnShape<NQ>::kUnit - 1) / AttnShape<NQ>::kUnit;
  return s;
}
// How the units are dealt out to the CTAs.
// By segments ((head, tile)s of a sequence), when there are no more of them than CTAs: every segment
// gets one CTA and a part of the spare ones by its length, and no CTA has two.  Otherwise in shares of
// the row of all units that cost the same, counting kSwitch units for every segment (its queries, the
// join of its warps: a batch of uneven lengths took 130 us with shares of as many units each, since
// some CTAs had a dozen short segments); a share's border gives way to a segment's border that is
// next to it while shares are short.  A unit takes 1.3 us, joining parts 2.7 us and a second segment in a CTA
// 3.7 us (measured, head_dim 128; the smaller heads go by the same numbers): equal shares, where a CTA mostly has two segments and joins one, win
// only where dealing out by segments makes the largest share that much larger (measured: 64 segments
// of 1024 positions 16.7 us in equal shares, 12.1 us by segments).
struct AttnPlan {
  int total, ctas, spare;                               // units (equal shares: their cost), CTAs; spare < 0: equal shares
};
// CTAs of a segment: one and its part of the spare ones, or one where the others do not bring more
// than the joining costs.
template <int NQ>
__device__ __forceinline__ int attn_pieces(const AttnPlan& p, int units) {
  int n = min(1 + (int)((float)units * (float)p.spare / (float)p.total), units);
  // parts of 128 rows (66 KB) are joined one after the other, about two to the time of a unit: n parts
  // cost units / n + n / 2 (548 rows over 9000 positions: 84 us with 28 parts a segment)
  // small parts cost a thirtieth of a unit (one sequence of 131000 positions with one key head: 35 us
  // with 148 parts)
  n = min(n, (int)sqrtf((NQ == 16 ? 2.f : 16.f) * (float)units) + 1);
  return (units + n - 1) / n + AttnShape<NQ>::kJoin >= units ? 1 : n;
}
// the time of a segment's CTA, in units
template <int NQ>
__device__ __forceinline__ int attn_load(int units, int pieces) {
  return (units + pieces - 1) / pieces + (pieces > 1 ? AttnShape<NQ>::kJoin : 0);
}
template <int NQ>
__device__ __forceinline__ bool attn_by_segments(int largest, int dealt, int total, int ctas) {
  // (`dealt` can be one or two too many where a quotient was rounded up)
  return dealt <= ctas && largest <= total / ctas + AttnShape<NQ>::kJoin * 5 / 2;
}

// Sequence b into the table; its units and segments.  A sequence whose length or span does not fit
// counts as one that holds nothing; with `drop` (spans that are not in order) none has any tokens.
template <int NQ, typename T>
__device__ __forceinline__ AttnSeq attn_enter(const cats_kv8& c, const KvAttnArgs<T>& A, AttnTable& tab, int b, int group,
                                              bool drop) {
  const KvSpan sp = kv_span(A.cu, A.uniform, b);
  int len = c.lens[b], first = sp.first, count = drop ? 0 : sp.count;
  const bool long_ok = len >= 0 && len <= c.max_pages * c.page;
  const bool span_ok = first >= 0 && (long long)first + count <= A.tokens;
  if (count > 0 && !(long_ok && span_ok)) {
    if (blockIdx.x == 0) kv_flag(c, long_ok ? KV_BAD_SPAN : KV_TOO_LONG);
    len = 0;
    const long long end = min((long long)first + count, (long long)A.tokens);
    first = max(first, 0);
    count = (int)max(end - first, 0LL);
  }
  if (len < 0) len = 0;
  tab.len[b] = len;
  tab.first[b] = first;
  tab.count[b] = count;
  return attn_seq<NQ>(tab, b, group);
}

// Up to 32 sequences: one warp, a lane each, no barrier in between.
template <int NQ, typename T>
__device__ __forceinline__ AttnPlan attn_plan_warp(const cats_kv8& c, const KvAttnArgs<T>& A, AttnTable& tab, int group) {
  const int lane = threadIdx.x & 31;
  AttnSeq s = {0, 0, 0, 0, 0};
  const bool drop = __any_sync(0xffffffffu, A.cu && lane < c.n_seqs && kv_descends(A.cu, lane));
  if (drop && blockIdx.x == 0 && lane == 0) kv_flag(c, KV_BAD_SPAN);
  if (lane < c.n_seqs) s = attn_enter<NQ>(c, A, tab, lane, group, drop);
  auto scan = [&](int v) {
    int incl = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += u;
    }
    return incl;
  };
  const int segments = s.units ? s.tiles * c.n_kv_heads : 0, mine = s.units * segments;
  const int incl = scan(mine), total = __shfl_sync(0xffffffffu, incl, 31);
  if (lane < c.n_seqs) tab.pre[lane + 1] = incl;
  if (lane == 0) tab.pre[0] = 0;
  const int all = __reduce_add_sync(0xffffffffu, segments);
  if (all <= A.ctas && total > 0) {
    AttnPlan plan = {total, 0, A.ctas - all};
    const int n = segments ? attn_pieces<NQ>(plan, s.units) : 0;
    const int ctas = scan(n * segments);
    if (lane < c.n_seqs) tab.cost[lane + 1] = ctas;
    if (lane == 0) tab.cost[0] = 0;
    plan.ctas = __shfl_sync(0xffffffffu, ctas, 31);
    const int largest = __reduce_max_sync(0xffffffffu, n ? attn_load<NQ>(s.units, n) : 0);
    if (attn_by_segments<NQ>(largest, plan.ctas, total, A.ctas)) return plan;
  }
  const int cost = scan(segments * (s.units + AttnShape<NQ>::kSwitch));
  if (lane < c.n_seqs) tab.cost[lane + 1] = cost;
  if (lane == 0) tab.cost[0] = 0;
  const int whole = __shfl_sync(0xffffffffu, cost, 31);
  return {whole, min(total, A.ctas), -1};
}

// Exclusive scan over the values that the threads hold for their sequences; all of them together.
template <int THREADS>
__device__ __forceinline__ int attn_scan(const int* mine, int* pre, int n_seqs, int* s_warp) {
  constexpr int kPer = kKvMaxSeqs / THREADS;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int sum = 0;
#pragma unroll
  for (int i = 0; i < kPer; ++i) sum += mine[i];
  int incl = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += v;
  }
  __syncthreads();                                      // s_warp may still be read
  if (lane == 31) s_warp[warp] = incl;
  __syncthreads();
  int before = incl - sum;
  for (int w = 0; w < warp; ++w) before += s_warp[w];
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int b = threadIdx.x * kPer + i;
    if (b <= n_seqs) pre[b] = before;
    before += mine[i];
  }
  if (threadIdx.x == THREADS - 1 && n_seqs == kKvMaxSeqs) pre[kKvMaxSeqs] = before;
  __syncthreads();
  return pre[n_seqs];
}
// Any number of sequences: all threads.
template <int NQ, typename T>
__device__ __forceinline__ AttnPlan attn_plan_block(const cats_kv8& c, const KvAttnArgs<T>& A, AttnTable& tab, int group,
                                                    int* s_warp) {
  constexpr int kThreads = AttnShape<NQ>::kThreads, kPer = kKvMaxSeqs / kThreads;
  int mine[kPer], segments = 0;
  bool drop = false;
  if (A.cu) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int b = threadIdx.x * kPer + i;
      drop = drop || (b < c.n_seqs && kv_descends(A.cu, b));
    }
    drop = __syncthreads_or(drop);
    if (drop && blockIdx.x == 0 && threadIdx.x == 0) kv_flag(c, KV_BAD_SPAN);
  }
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int b = threadIdx.x * kPer + i;
    mine[i] = 0;
    if (b < c.n_seqs) {
      const AttnSeq s = attn_enter<NQ>(c, A, tab, b, group, drop);
      mine[i] = s.units * s.tiles * c.n_kv_heads;
      if (s.units) segments += s.tiles * c.n_kv_heads;
    }
  }
  const int total = attn_scan<kThreads>(mine, tab.pre, c.n_seqs, s_warp);
  // (the threads' numbers go through the same words as the scan's)
  auto all_of = [&](int v, bool sum) {
    v = sum ? __reduce_add_sync(0xffffffffu, v) : __reduce_max_sync(0xffffffffu, v);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) s_warp[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0;
    for (int w = 0; w < kThreads / 32; ++w) v = sum ? v + s_warp[w] : max(v, s_warp[w]);
    return v;
  };
  const int all = all_of(segments, true);
  if (all <= A.ctas && total > 0) {
    AttnPlan plan = {total, 0, A.ctas - all};
    int largest = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int b = threadIdx.x * kPer + i;
      mine[i] = 0;
      if (b < c.n_seqs) {
        const AttnSeq s = attn_seq<NQ>(tab, b, group);
        if (s.units && s.tiles) {
          const int n = attn_pieces<NQ>(plan, s.units);
          mine[i] = n * s.tiles * c.n_kv_heads;
          largest = max(largest, attn_load<NQ>(s.units, n));
        }
      }
    }
    plan.ctas = attn_scan<kThreads>(mine, tab.cost, c.n_seqs, s_warp);
    largest = all_of(largest, false);
    if (attn_by_segments<NQ>(largest, plan.ctas, total, A.ctas)) return plan;
  }
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int b = threadIdx.x * kPer + i;
    mine[i] = 0;
    if (b < c.n_seqs) {
      const AttnSeq s = attn_seq<NQ>(tab, b, group);
      if (s.units) mine[i] = s.tiles * c.n_kv_heads * (s.units + AttnShape<NQ>::kSwitch);
    }
  }
  const int whole = attn_scan<kThreads>(mine, tab.cost, c.n_seqs, s_warp);
  return {whole, min(total, A.ctas), -1};
}

// The plan and its table (called by all threads; ends with a barrier); zeroes the rows of the
// sequences that hold nothing.
template <int NQ, int HD, typename T>
__device__ __forceinline__ AttnPlan attn_table(const cats_kv8& c, const KvAttnArgs<T>& A, AttnTable& tab, AttnPlan* s_plan,
                                               int* s_warp) {
  constexpr int kThreads = AttnShape<NQ>::kThreads;
  const int group = A.nh / c.n_kv_heads;
  AttnPlan plan;
  if (c.n_seqs <= 32) {
    if (threadIdx.x < 32) {
      plan = attn_plan_warp<NQ>(c, A, tab, group);
      if (threadIdx.x == 0) *s_plan = plan;
    }
    __syncthreads();
    plan = *s_plan;
  } else {
    plan = attn_plan_block<NQ>(c, A, tab, group, s_warp);
  }
  for (int b = blockIdx.x; b < c.n_seqs; b += gridDim.x) {
    if (tab.pre[b + 1] != tab.pre[b] || tab.count[b] == 0) continue;
    T* dst = A.out + (size_t)tab.first[b] * A.nh * HD;
    const size_t n = (size_t)tab.count[b] * A.nh * HD;
    for (size_t k = threadIdx.x; k < n; k += kThreads) dst[k] = VecT<T>::from_f(0.f);
  }
  return plan;
}

// the last sequence that begins at or before x
__device__ __forceinline__ int attn_find(const int* pre, int n_seqs, int x) {
  int lo = 0, hi = n_seqs - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (pre[mid] <= x) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}
// Where a unit lies: sequence, head, tile and number of the unit within them.
struct AttnPlace {
  int b, head, tile, unit;
};
template <int NQ>
__device__ __forceinline__ AttnPlace attn_place(const AttnTable& tab, int n_seqs, int group, int w, AttnSeq* seq) {
  const int lo = attn_find(tab.pre, n_seqs, w);
  const AttnSeq s = attn_seq<NQ>(tab, lo, group);
  const int r = w - tab.pre[lo];
  AttnPlace p;
  p.b = lo;
  const int at = r / s.units;
  p.unit = r - at * s.units;
  p.head = s.tiles == 1 ? at : at / s.tiles;
  p.tile = at - p.head * s.tiles;
  *seq = s;
  return p;
}
// Where the share of CTA c begins, as a unit.
template <int NQ>
__device__ __forceinline__ int attn_share(const AttnTable& tab, const AttnPlan& p, int n_seqs, int group, int c) {
  if (c >= p.ctas) return tab.pre[n_seqs];
  if (p.spare >= 0) {
    const int b = attn_find(tab.cost, n_seqs, c);
    const AttnSeq s = attn_seq<NQ>(tab, b, group);
    const int n = attn_pieces<NQ>(p, s.units), r = c - tab.cost[b], seg = r / n, piece = r - seg * n, q = s.units / n;
    return tab.pre[b] + seg * s.units + q * piece + min(piece, s.units - q * n);
  }
  // (shares cost at least one unit each and differ)
  const int q = p.total / p.ctas, w = q * c + (int)((unsigned)(p.total - q * p.ctas) * (unsigned)c / (unsigned)p.ctas);
  const int b = attn_find(tab.cost, n_seqs, w);
  const AttnSeq s = attn_seq<NQ>(tab, b, group);
  const int each = s.units + AttnShape<NQ>::kSwitch, r = w - tab.cost[b], seg = r / each;
  int unit = max(r - seg * each - AttnShape<NQ>::kSwitch, 0);
  constexpr int kNear = 256 / AttnShape<NQ>::kUnit;
  if (q < 16 * kNear) {
    if (unit <= kNear) unit = 0;
    else if (s.units - unit <= kNear) unit = s.units;
  }
  return tab.pre[b] + seg * s.units + unit;
}
// The CTAs that have units u0 (a segment's first) and u0 + units - 1.
template <int NQ>
__device__ __forceinline__ void attn_owners(const AttnTable& tab, const AttnPlan& p, int n_seqs, int group, int b, int u0,
                                            int units, int* c0, int* c1) {
  const int seg = (u0 - tab.pre[b]) / units;
  if (p.spare >= 0) {
    const int n = attn_pieces<NQ>(p, units);
    *c0 = tab.cost[b] + seg * n;
    *c1 = *c0 + n - 1;
    return;
  }
  const int each = units + AttnShape<NQ>::kSwitch;
  for (int x = 0; x < 2; ++x) {
    const int w = x ? u0 + units - 1 : u0, at = tab.cost[b] + seg * each + (x ? each - 1 : 0);
    int c = min((int)((float)at * (float)p.ctas / (float)p.total), p.ctas - 1);
    while (c > 0 && attn_share<NQ>(tab, p, n_seqs, group, c) > w) --c;
    while (c + 1 < p.ctas && attn_share<NQ>(tab, p, n_seqs, group, c + 1) <= w) ++c;
    *(x ? c1 : c0) = c;
  }
}
__device__ __forceinline__ uint2 lds2(uint32_t addr) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr));
  return v;
}
__device__ __forceinline__ uint32_t lds1(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(addr));
  return v;
}

// O^T += V^T P^T for the warp's tile: the codes of V are the rows operand (channels x positions),
// the weights the columns (positions x rows of the tile).
// GUARD: some row must not see all of the tile's positions and V holds a NaN; zero weights would turn
// it into NaN in rows that do not see it, so NaN codes are taken out of the product and added to the
// rows that do see them (`seen`, weights 1 and 0).
template <int HD, int NQ, bool SPLIT, bool GUARD>
__device__ __forceinline__ void attn_pv(float (*o)[NQ][4], const uint32_t (*p)[2], const uint32_t (*p_lo)[2],
                                        const uint32_t (*seen)[2], uint32_t v0, uint32_t v1, uint32_t v2,
                                        uint32_t v3) {
  // r0 .. r3: four channels at the lane's four positions (2 t, 2 t + 1, 2 t + 8, 2 t + 9)
  auto group = [&](uint32_t r0, uint32_t r1, uint32_t r2, uint32_t r3, float (*acc)[NQ][4]) {
    // byte pairs (position, next position) of each channel
    const uint32_t w[4] = {__byte_perm(r0, r1, 0x5140), __byte_perm(r2, r3, 0x5140), __byte_perm(r0, r1, 0x7362),
                           __byte_perm(r2, r3, 0x7362)};
#pragma unroll
    for (int j = 0; j < 2; ++j) {                        // channels 2 j, 2 j + 1: rows g and g + 8 of a tile
      uint32_t a[4], x = w[2 * j], y = w[2 * j + 1];
      if (GUARD) {
        auto nan_bytes = [](uint32_t v) { return ((((v & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) >> 7) * 0xffu; };
        const uint32_t nx = nan_bytes(x), ny = nan_bytes(y);
        uint32_t ind[4];
        e4m3x4_to_f16x2(nx & 0x38383838u, ind[0], ind[1]);   // 0x38 is 1.0
        e4m3x4_to_f16x2(ny & 0x38383838u, ind[2], ind[3]);
        x &= ~nx;
        y &= ~ny;
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
          float hit[4] = {0.f, 0.f, 0.f, 0.f};
          mma16816(hit, ind, seen[n][0], seen[n][1]);
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (hit[i] > 0.f) acc[j][n][i] = __uint_as_float(0x7fc00000u);
        }
      }
      e4m3x4_to_f16x2(x, a[0], a[1]);
      e4m3x4_to_f16x2(y, a[2], a[3]);
#pragma unroll
      for (int n = 0; n < NQ; ++n) {
        mma16816(acc[j][n], a, p[n][0], p[n][1]);
        if (SPLIT) mma16816(acc[j][n], a, p_lo[n][0], p_lo[n][1]);
      }
    }
  };
  // v0, v1: rows 2 t and 2 t + 1 at byte 8 g; rows 8 further on have the same exchange of chunks
#pragma unroll
  for (int q = 0; q < HD / 64; ++q) {
    const uint2 r0 = lds2(v0 ^ (64 * q)), r1 = lds2(v1 ^ (64 * q));
    const uint2 r2 = lds2((v0 ^ (64 * q)) + 1024), r3 = lds2((v1 ^ (64 * q)) + 1024);
    group(r0.x, r1.x, r2.x, r3.x, o + 4 * q);
    group(r0.y, r1.y, r2.y, r3.y, o + 4 * q + 2);
  }
  if (HD % 64) {                                         // 32 channels left: byte 4 g
    constexpr int q = HD / 64;
    group(lds1(v2), lds1(v3), lds1(v2 + 1024), lds1(v3 + 1024), o + 4 * q);
  }
}

// (top, sum, v) += a part with reference m, sum l and products w.  A part that saw nothing is left
// out (a NaN sum is not: it stays NaN).
__device__ __forceinline__ void attn_add(float m, float l, float4 w, float& top, float& sum, float4& v) {
  if (m == -INFINITY && l == 0.f) return;
  const float to = fmaxf(top, m), ref = to == -INFINITY ? 0.f : to;
  const float x = ex2(m - ref), y = top == -INFINITY && sum == 0.f ? 0.f : ex2(top - ref);
  top = to;
  sum = fmaf(l, x, sum * y);
  v.x = fmaf(w.x, x, v.x * y);
  v.y = fmaf(w.y, x, v.y * y);
  v.z = fmaf(w.z, x, v.z * y);
  v.w = fmaf(w.w, x, v.w * y);
}
// four channels of row r of the tile at `at`
template <typename T>
__device__ __forceinline__ void attn_store(const KvAttnArgs<T>& A, const AttnSeq& seq, const AttnPlace& at, int group,
                                           int tile_rows, int r, int d, int hd, float sum, float4 v) {
  const int rr = at.tile * tile_rows + r, tok = rr / group, hq = at.head * group + rr - tok * group;
  const float inv = sum == 0.f ? 0.f : 1.f / sum;        // no position seen: zeros
  __align__(16) T w[4] = {VecT<T>::from_f(v.x * inv), VecT<T>::from_f(v.y * inv), VecT<T>::from_f(v.z * inv),
                          VecT<T>::from_f(v.w * inv)};
  T* dst = A.out + ((size_t)(seq.first + tok) * A.nh + hq) * hd + d;
  if (sizeof(T) == 4) *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(w);
  else *reinterpret_cast<uint2*>(dst) = *reinterpret_cast<const uint2*>(w);
}

template <typename T, int HD, int NQ>
__global__ void __launch_bounds__(AttnShape<NQ>::kThreads, 1) k_kv8_attend(const cats_kv8 c, const KvAttnArgs<T> A) {
  using S = AttnShape<NQ>;
  constexpr bool SPLIT = sizeof(T) == 4;
  constexpr int KS = HD / 16;                            // k-steps of the score product
  constexpr int MT = HD / 16;                            // row tiles of O^T
  extern __shared__ __align__(128) unsigned char smem_raw[];
  // (aligned by hand: the exchange of chunks is applied to whole addresses)
  unsigned char* smem = smem_raw + ((128 - ((uint32_t)__cvta_generic_to_shared(smem_raw) & 127)) & 127);
  __shared__ AttnTable s_tab;
  __shared__ int s_warp[S::kWarps];
  __shared__ int s_last, s_owners[2];
  __shared__ AttnPlan s_plan;
  pdl_wait();
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  unsigned char* ring = smem + (size_t)warp * S::kStages * kAttnStageBytes;
  unsigned char* after = smem + (size_t)S::kWarps * S::kStages * kAttnStageBytes;
  float4* meta = reinterpret_cast<float4*>(after) + warp * S::kStages;   // scales of keys and values, rows
  float* s_ml = reinterpret_cast<float*>(after + (size_t)S::kWarps * S::kStages * 16);
  uint4* s_q = reinterpret_cast<uint4*>(s_ml + S::kWarps * 16);         // [HD / 32][NQ][32 lanes], where shared
  const uint32_t ring_u32 = (uint32_t)__cvta_generic_to_shared(ring);
  const uint32_t meta_u32 = (uint32_t)__cvta_generic_to_shared(meta);

  const AttnPlan plan = attn_table<NQ, HD>(c, A, s_tab, &s_plan, s_warp);
  if ((int)blockIdx.x >= plan.ctas) return;
  const int group = A.nh / c.n_kv_heads;
  const int share0 = attn_share<NQ>(s_tab, plan, c.n_seqs, group, blockIdx.x);
  const int n_units = attn_share<NQ>(s_tab, plan, c.n_seqs, group, blockIdx.x + 1) - share0;
  if (n_units <= 0) return;

  // ---- loader: lane i of the warp knows where unit `base + i` lies and which page its tile is in --
  int d_rows = 0, d_scale = 0;                           // rows to load; the keys' scale in its layer
  long long d_off = 0;                                   // the keys' first byte in the layer
  const uint8_t* layer_codes = kv_rows(c, A.layer, 0, 0, 0);
  const float* layer_scales = kv_scale(c, A.layer, 0, 0, 0);
  auto look = [&](int base) {
    d_rows = 0;
    if (base + lane < n_units) {
      AttnSeq s;
      const AttnPlace p = attn_place<NQ>(s_tab, c.n_seqs, group, share0 + base + lane, &s);
      const int last = min(s.count - 1, (p.tile * S::kRows + S::kRows - 1) / group);
      const int end = min(s.len, s.len - s.count + last + 1);        // positions that the tile's rows see
      const int kb = p.unit * S::kUnit + warp * kAttnTile;
      d_rows = min(max(end - kb, 0), kAttnTile);
      if (d_rows > 0) {
        const int id = c.table[(size_t)p.b * c.max_pages + kb / c.page];
        if (id < 0 || id >= c.n_pages) {
          kv_flag(c, KV_BAD_PAGE);
          d_rows = 0;
        } else {
          d_off = ((long long)id * 2 * c.n_kv_heads + p.head) * (c.page * HD) + (kb % c.page) * HD;
          d_scale = id * 2 * c.n_kv_heads + p.head;
        }
      }
    }
  };
  // 16-byte chunk `lane + 32 i` of the tile's keys (i < HD / 32) and of its values goes to byte
  // (to0 ^ flip) + step: the exchange of chunks depends on a row's three low bits
  constexpr int kChunks = HD / 16;                       // of a row
  const uint32_t to0 = ring_u32 + attn_swizzle(lane / kChunks, lane % kChunks * 16);
  auto chunk_to = [&](int i) -> uint32_t {
    if (HD == 128) return (to0 ^ ((i & 1) * 32)) + 512 * i;          // four rows further on
    if (HD == 64) return to0 + 1024 * i;                              // eight rows
    return ring_u32 + attn_swizzle((lane + 32 * i) / kChunks, (lane + 32 * i) % kChunks * 16);
  };
  const long long v_off = (long long)c.n_kv_heads * c.page * HD;
  int stage_in = 0, n_in = 0;
  auto issue = [&]() {
    if (n_in < n_units) {
      if ((n_in & 31) == 0) look(n_in);
      const int src = n_in & 31;
      const int rows = __shfl_sync(0xffffffffu, d_rows, src);
      const uint32_t st = stage_in * kAttnStageBytes;
      if (lane == 0) reinterpret_cast<int*>(meta + stage_in)[2] = rows;
      if (rows > 0) {
        const uint8_t* kp = layer_codes + __shfl_sync(0xffffffffu, d_off, src) + lane * 16;
        const uint8_t* vp = kp + v_off;
        const int sc = __shfl_sync(0xffffffffu, d_scale, src);
        if (lane < 2)
          asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(meta_u32 + 16 * stage_in + 4 * lane),
                       "l"(layer_scales + sc + lane * c.n_kv_heads)
                       : "memory");
        if (rows == kAttnTile) {
#pragma unroll
          for (int i = 0; i < HD / 32; ++i) {
            const uint32_t to = st + chunk_to(i);
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(kp + 512 * i) : "memory");
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + kAttnTile * 128), "l"(vp + 512 * i)
                         : "memory");
          }
        } else {                                         // the last rows of a sequence: the others become zeros
#pragma unroll
          for (int i = 0; i < HD / 32; ++i) {
            const uint32_t to = st + chunk_to(i);
            const bool in = (lane + 32 * i) / kChunks < rows;
            const int bytes = in ? 16 : 0, off = in ? 512 * i : -16 * lane;
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(kp + off), "r"(bytes) : "memory");
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to + kAttnTile * 128), "l"(vp + off),
                         "r"(bytes)
                         : "memory");
          }
        }
      }
      ++n_in;
      stage_in = stage_in + 1 == S::kStages ? 0 : stage_in + 1;
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  for (int i = 0; i < S::kStages - 1; ++i) issue();

  // the lane's reads of a tile (offsets in a stage): keys at rows g and g + 8, byte 8 t; values at
  // rows 2 t, 2 t + 1 (and 8 further on), byte 8 g, and byte 4 g of the last 32 channels of 32 and 96
  const uint32_t k_off = attn_swizzle(g, 8 * t);
  const uint32_t v0_off = kAttnTile * 128 + attn_swizzle(2 * t, 8 * g), v1_off = kAttnTile * 128 + attn_swizzle(2 * t + 1, 8 * g);
  const uint32_t v2_off = HD % 64 ? kAttnTile * 128 + attn_swizzle(2 * t, HD / 64 * 64 + 4 * g) : 0;
  const uint32_t v3_off = HD % 64 ? kAttnTile * 128 + attn_swizzle(2 * t + 1, HD / 64 * 64 + 4 * g) : 0;

  // ---- consumer: S^T = K Q^T, so a lane has rows (columns) 2 t and 2 t + 1 of each group of eight ----
  uint32_t qa[S::kQueriesShared ? 1 : KS][NQ][2], qb[SPLIT ? KS : 1][NQ][2];
  float o[MT][NQ][4];
  float m[NQ][2], l[NQ][2], f[NQ][2];
  int lim[NQ][2], lim_min = 0;                           // positions that a row sees, and the least of them
  int ec = kAttnNoExp;                                   // exponent that o is held at
  AttnSeq seq;
  AttnPlace at = attn_place<NQ>(s_tab, c.n_seqs, group, share0, &seq);
  bool first_seg = true, begins_here = at.unit == 0, fresh = true;
  int stage = 0;
  for (int u = 0; u < n_units; ++u) {
    if (fresh) {                                         // a new (sequence, head, tile): its queries
      fresh = false;
      ec = kAttnNoExp;
      const int rows = min(S::kRows, seq.count * group - at.tile * S::kRows);
      lim_min = min(seq.len, seq.len - seq.count + at.tile * S::kRows / group + 1);
#pragma unroll
      for (int n = 0; n < NQ; ++n) {
        const int r = at.tile * S::kRows + 8 * n + g, tok = r / group, hq = at.head * group + r - tok * group;
        const bool on = 8 * n + g < rows;
        const T* src = A.q + (size_t)(seq.first + tok) * A.q_ld + (size_t)hq * HD + 8 * t;
        float q[HD / 32][8], top = 0.f;
#pragma unroll
        for (int p = 0; p < HD / 32; ++p) {
#pragma unroll
          for (int k = 0; k < 8; ++k) q[p][k] = 0.f;
          if (on) load8_cached(src + 32 * p, q[p]);
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const float a = fabsf(q[p][k]);
            if (a <= 3.402823466e38f) top = fmaxf(top, a);
          }
        }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const int e = top > 0.f ? min(max(kv_exp_of(top) + 1, -126), 126) : 0;
        const float inv = kv_pow2(-e), back = kv_pow2(e) * A.scale;
        const int sees = on ? min(seq.len, seq.len - seq.count + tok + 1) : 0;
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          f[n][x] = __shfl_sync(0xffffffffu, back, 4 * (2 * t + x));
          lim[n][x] = __shfl_sync(0xffffffffu, sees, 4 * (2 * t + x));
          m[n][x] = -INFINITY;
          l[n][x] = 0.f;
        }
#pragma unroll
        for (int p = 0; p < HD / 32; ++p)
#pragma unroll
          for (int k = 0; k < 8; ++k) q[p][k] *= inv;
        if (S::kQueriesShared) {                         // the same for all warps: each writes its share
#pragma unroll
          for (int p = 0; p < HD / 32; ++p)
            if ((p * NQ + n) % S::kWarps == warp)
              s_q[(p * NQ + n) * 32 + lane] = make_uint4(half2_bits(q[p][0], q[p][1]), half2_bits(q[p][2], q[p][3]),
                                                         half2_bits(q[p][4], q[p][5]), half2_bits(q[p][6], q[p][7]));
        } else {
#pragma unroll
          for (int p = 0; p < HD / 32; ++p)
#pragma unroll
            for (int e2 = 0; e2 < 2; ++e2)
#pragma unroll
              for (int x = 0; x < 2; ++x) {
                const float* v = q[p] + 4 * e2 + 2 * x;
                constexpr int last = S::kQueriesShared ? 0 : KS - 1;
                uint32_t& to = qa[2 * p + e2 < last ? 2 * p + e2 : last][n][x];
                to = half2_bits(v[0], v[1]);
                if (SPLIT) qb[SPLIT ? 2 * p + e2 : 0][n][x] = half2_rest(v[0], v[1], to);
              }
        }
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int x = 0; x < 4; ++x) o[i][n][x] = 0.f;
      }
      if (S::kQueriesShared) __syncthreads();            // (all warps are at the same unit)
    }
    asm volatile("cp.async.wait_group %0;" ::"n"(S::kStages - 2) : "memory");
    __syncwarp();
    issue();

    const int kb = at.unit * S::kUnit + warp * kAttnTile;
    unsigned char* kt = ring + stage * kAttnStageBytes;
    const float4 sc = meta[stage];
    if (__float_as_int(sc.z) > 0) {
      const uint32_t st = ring_u32 + stage * kAttnStageBytes;
      float s[NQ][4];
#pragma unroll
      for (int n = 0; n < NQ; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) s[n][i] = 0.f;
#pragma unroll
      for (int p = 0; p < HD / 32; ++p) {
        const uint32_t ka = (st + k_off) ^ (32 * p);
        const uint2 k0 = lds2(ka), k1 = lds2(ka + 1024);
        uint32_t a[2][4];
#pragma unroll
        for (int e2 = 0; e2 < 2; ++e2) {
          const uint32_t x0 = e2 ? k0.y : k0.x, x1 = e2 ? k1.y : k1.x;
          e4m3x4_to_f16x2(x0, a[e2][0], a[e2][2]);
          e4m3x4_to_f16x2(x1, a[e2][1], a[e2][3]);
        }
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
          if (S::kQueriesShared) {
            const uint4 q = s_q[(p * NQ + n) * 32 + lane];
            mma16816(s[n], a[0], q.x, q.y);
            mma16816(s[n], a[1], q.z, q.w);
          } else {
#pragma unroll
            for (int e2 = 0; e2 < 2; ++e2) {
              constexpr int last = S::kQueriesShared ? 0 : KS - 1;
              const int k = 2 * p + e2 < last ? 2 * p + e2 : last;
              mma16816(s[n], a[e2], qa[k][n][0], qa[k][n][1]);
              if (SPLIT) mma16816(s[n], a[e2], qb[SPLIT ? k : 0][n][0], qb[SPLIT ? k : 0][n][1]);
            }
          }
        }
      }
      int ev = kv_exp_of(sc.y);
      if ((unsigned)(ev - ec + kAttnSpan) > 2u * kAttnSpan) {          // (the same for all lanes)
        ev = attn_exp_of(sc.y);
        const float by = kv_pow2(max(ec - ev, -126));    // (the first time o is zero)
        ec = ev;
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int n = 0; n < NQ; ++n)
#pragma unroll
            for (int x = 0; x < 4; ++x) o[i][n][x] *= by;
      }
      const float evf = (float)(ev - ec), vi = kv_pow2(ec - ev);
      const bool cut = kb + kAttnTile > lim_min;         // some row does not see all of the tile
      uint32_t p[NQ][2], pl[NQ][2];
      float top[NQ][2];
#pragma unroll
      for (int n = 0; n < NQ; ++n)
#pragma unroll
        for (int x = 0; x < 2; ++x) {                    // s[x], s[2 + x]: positions g, g + 8 of row 2 t + x
          const float by = sc.x * f[n][x];
          s[n][x] *= by;
          s[n][2 + x] *= by;
          if (cut) {
            if (kb + g >= lim[n][x]) s[n][x] = -INFINITY;
            if (kb + 8 + g >= lim[n][x]) s[n][2 + x] = -INFINITY;
          }
          top[n][x] = fmaxf(s[n][x], s[n][2 + x]);
        }
#pragma unroll
      for (int w = 4; w < 32; w <<= 1)
#pragma unroll
        for (int n = 0; n < NQ; ++n)
#pragma unroll
          for (int x = 0; x < 2; ++x) top[n][x] = fmaxf(top[n][x], __shfl_xor_sync(0xffffffffu, top[n][x], w));
      // The reference m of the weights follows the running maximum only when that is more than
      // 2^kAttnSlack ahead: weights up to 2^(kAttnSlack + kAttnSpan) do half precision no harm, and the
      // accumulators are rescaled a few times per sequence instead of at every second tile.
      bool ahead = false;
#pragma unroll
      for (int n = 0; n < NQ; ++n)
#pragma unroll
        for (int x = 0; x < 2; ++x) ahead |= top[n][x] > m[n][x] + kAttnSlack;
      if (__any_sync(0xffffffffu, ahead)) {
#pragma unroll
        for (int n = 0; n < NQ; ++n)
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const float to = fmaxf(top[n][x], m[n][x]), by = m[n][x] == -INFINITY ? 0.f : ex2(m[n][x] - to);
            m[n][x] = to;
            l[n][x] *= by;
#pragma unroll
            for (int i = 0; i < MT; ++i) {
              o[i][n][x] *= by;
              o[i][n][2 + x] *= by;
            }
          }
      }
#pragma unroll
      for (int n = 0; n < NQ; ++n) {
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          // (the same for all tiles whose pages have the same ev, while m and ec stay: its rounding cancels)
          const float ref = m[n][x] == -INFINITY ? 0.f : m[n][x] - evf;
          s[n][x] = ex2(s[n][x] - ref);
          s[n][2 + x] = ex2(s[n][2 + x] - ref);
          l[n][x] = fmaf(s[n][x] + s[n][2 + x], vi, l[n][x]);
        }
#pragma unroll
        for (int x = 0; x < 2; ++x) {                    // positions 0 .. 7, 8 .. 15
          const uint32_t h = half2_bits(s[n][2 * x], s[n][2 * x + 1]);
          p[n][x] = transpose8x8(h);
          pl[n][x] = SPLIT ? transpose8x8(half2_rest(s[n][2 * x], s[n][2 * x + 1], h)) : 0u;
        }
      }
      bool guard = false;
      if (cut) {
        bool nan = false;
#pragma unroll
        for (int i = 0; i < HD / 32; ++i) {
          const uint4 v = *reinterpret_cast<const uint4*>(ring + stage * kAttnStageBytes + kAttnTile * 128 + (chunk_to(i) - ring_u32));
          const uint32_t x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
          for (int k = 0; k < 4; ++k) nan |= (((x[k] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) != 0;
        }
        guard = __any_sync(0xffffffffu, nan);
      }
      if (guard) {
        uint32_t seen[NQ][2];
#pragma unroll
        for (int n = 0; n < NQ; ++n) {                   // lane: row g, positions 2 t, 2 t + 1 (+ 8)
          const int a = __shfl_sync(0xffffffffu, lim[n][0], g >> 1), b = __shfl_sync(0xffffffffu, lim[n][1], g >> 1);
          const int mine = (g & 1) ? b : a;
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const int k = kb + 8 * x + 2 * t;
            seen[n][x] = half2_bits(k < mine ? 1.f : 0.f, k + 1 < mine ? 1.f : 0.f);
          }
        }
        attn_pv<HD, NQ, SPLIT, true>(o, p, pl, seen, st + v0_off, st + v1_off, st + v2_off, st + v3_off);
      } else {
        attn_pv<HD, NQ, SPLIT, false>(o, p, pl, nullptr, st + v0_off, st + v1_off, st + v2_off, st + v3_off);
      }
    }
    stage = stage + 1 == S::kStages ? 0 : stage + 1;
    ++at.unit;

    if (at.unit == seq.units || u + 1 == n_units) {      // the segment ends here: join the warps
      const int rows = min(S::kRows, seq.count * group - at.tile * S::kRows);
      const bool whole = begins_here && at.unit == seq.units;
      float* part = A.parts + (size_t)(blockIdx.x * 2 + (first_seg ? 0 : 1)) * attn_part_floats(S::kRows, HD);
      // eight rows at a time, in the codes' bytes of the stage that this tile was in (free until the
      // next call of issue): [8][HD] floats of each warp
      const size_t pitch = (size_t)S::kStages * kAttnStageBytes;
      const float held = kv_pow2(max(ec, -126));         // (no tile seen: o is zero)
      __syncwarp();
#pragma unroll
      for (int n = 0; n < NQ; ++n) {
        if (8 * n >= rows) break;
#pragma unroll
        for (int x = 0; x < 2; ++x) {
#pragma unroll
          for (int w = 4; w < 32; w <<= 1) l[n][x] += __shfl_xor_sync(0xffffffffu, l[n][x], w);
          if (g == 0) {
            s_ml[(warp * 2 + 0) * 8 + 2 * t + x] = m[n][x];
            s_ml[(warp * 2 + 1) * 8 + 2 * t + x] = l[n][x];
          }
          if (8 * n + 2 * t + x < rows) {
            // row tile 4 q + i holds channels 64 q + 8 g + 2 i and the next; the rest 4 g + 2 i
            float* dst = reinterpret_cast<float*>(kt) + (2 * t + x) * HD;
#pragma unroll
            for (int i = 0; i < MT; i += 2) {
              const int d = i < 4 * (HD / 64) ? 64 * (i / 4) + 8 * g + 2 * (i % 4) : HD / 64 * 64 + 4 * g;
              *reinterpret_cast<float4*>(dst + d) = make_float4(o[i][n][x] * held, o[i][n][2 + x] * held, o[i + 1][n][x] * held,
                                                                o[i + 1][n][2 + x] * held);
            }
          }
        }
        __syncthreads();
        const int here = min(8, rows - 8 * n);
        for (int e = threadIdx.x; e < here * (HD / 4); e += S::kThreads) {
          const int r = e / (HD / 4), d = (e - r * (HD / 4)) * 4;
          const float* src = reinterpret_cast<const float*>(smem + (kt - ring)) + r * HD + d;
          float top = -INFINITY, sum = 0.f;
          float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
          for (int x = 0; x < S::kWarps; ++x) top = fmaxf(top, s_ml[x * 16 + r]);
          const float ref = top == -INFINITY ? 0.f : top;
#pragma unroll 4
          for (int x = 0; x < S::kWarps; ++x) {
            const float mx = s_ml[x * 16 + r], lx = s_ml[x * 16 + 8 + r];
            if (mx == -INFINITY && lx == 0.f) continue;  // saw nothing (a NaN sum goes on)
            const float by = ex2(mx - ref);
            const float4 w = *reinterpret_cast<const float4*>(src + x * (pitch / sizeof(float)));
            sum = fmaf(lx, by, sum);
            v.x = fmaf(w.x, by, v.x);
            v.y = fmaf(w.y, by, v.y);
            v.z = fmaf(w.z, by, v.z);
            v.w = fmaf(w.w, by, v.w);
          }
          if (whole) {
            attn_store(A, seq, at, group, S::kRows, 8 * n + r, d, HD, sum, v);
          } else {
            float* dst = part + (size_t)(8 * n + r) * (HD + 2);
            *reinterpret_cast<float2*>(dst + d) = make_float2(v.x, v.y);
            *reinterpret_cast<float2*>(dst + d + 2) = make_float2(v.z, v.w);
            if (d == 0) *reinterpret_cast<float2*>(dst + HD) = make_float2(top, sum);
          }
        }
        __syncthreads();
      }
      if (!whole) {
        // The CTA that brings the last part of a (head, tile) joins them all, in the order of the
        // CTAs.  The counter belongs to the CTA that has the first part (at most one of its
        // segments goes on in the next CTA) and is left at zero.
        const int u0 = share0 + u + 1 - at.unit;
        __threadfence();
        __syncthreads();
        if (threadIdx.x == 0) {
          attn_owners<NQ>(s_tab, plan, c.n_seqs, group, at.b, u0, seq.units, &s_owners[0], &s_owners[1]);
          s_last = atomicAdd(A.counters + s_owners[0], 1) == s_owners[1] - s_owners[0];
          if (s_last) A.counters[s_owners[0]] = 0;
        }
        __syncthreads();
        if (s_last) {
          const int c0 = s_owners[0], c1 = s_owners[1];
          __threadfence();
          // `sets` threads share a (row, four channels), each takes every sets-th part
          const int items = rows * (HD / 4), sets = max(1, min(S::kThreads / items, c1 - c0 + 1));
          const int first_begins = attn_share<NQ>(s_tab, plan, c.n_seqs, group, c0);
          float* s_set = reinterpret_cast<float*>(kt - ring + smem);       // [warps] x a stage: six floats a thread
          for (int e0 = 0; e0 < items; e0 += S::kThreads) {
            const int e = sets > 1 ? threadIdx.x % items : e0 + threadIdx.x, set = sets > 1 ? threadIdx.x / items : 0;
            float top = -INFINITY, sum = 0.f;
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
            if (e < items && set < sets) {
              const int r = e / (HD / 4), d = (e - r * (HD / 4)) * 4;
              auto part_of = [&](int x) {                // (only c0 can have another segment first)
                const int slot = x > c0 || first_begins >= u0 ? 0 : 1;
                return A.parts + (size_t)(2 * x + slot) * attn_part_floats(S::kRows, HD) + (size_t)r * (HD + 2);
              };
              if (c1 - c0 < 8) {
                for (int x = c0 + set; x <= c1; x += sets) {
                  const float* src = part_of(x);
                  const float2 ml = __ldcg(reinterpret_cast<const float2*>(src + HD));
                  const float2 a = __ldcg(reinterpret_cast<const float2*>(src + d)), b = __ldcg(reinterpret_cast<const float2*>(src + d + 2));
                  attn_add(ml.x, ml.y, make_float4(a.x, a.y, b.x, b.y), top, sum, v);
                }
              } else {                                   // many: the largest reference first, then the parts'
                                                         // weights do not wait for one another
#pragma unroll 8
                for (int x = c0 + set; x <= c1; x += sets) top = fmaxf(top, __ldcg(part_of(x) + HD));
                const float ref = top == -INFINITY ? 0.f : top;
#pragma unroll 4
                for (int x = c0 + set; x <= c1; x += sets) {
                  const float* src = part_of(x);
                  const float2 ml = __ldcg(reinterpret_cast<const float2*>(src + HD));
                  const float2 a = __ldcg(reinterpret_cast<const float2*>(src + d)), b = __ldcg(reinterpret_cast<const float2*>(src + d + 2));
                  const float by = ex2(ml.x - ref);      // saw nothing: 0 (and a NaN sum stays one)
                  sum = fmaf(ml.y, by, sum);
                  v.x = fmaf(a.x, by, v.x);
                  v.y = fmaf(a.y, by, v.y);
                  v.z = fmaf(b.x, by, v.z);
                  v.w = fmaf(b.y, by, v.w);
                }
              }
            }
            if (sets > 1) {
              float* mine = s_set + (threadIdx.x >> 5) * (S::kStages * kAttnStageBytes / 4) + (threadIdx.x & 31) * 6;
              mine[0] = top;
              mine[1] = sum;
              mine[2] = v.x;
              mine[3] = v.y;
              mine[4] = v.z;
              mine[5] = v.w;
              __syncthreads();
              if (set == 0)
                for (int k = 1; k < sets; ++k) {
                  const int other = threadIdx.x + k * items;
                  const float* p = s_set + (other >> 5) * (S::kStages * kAttnStageBytes / 4) + (other & 31) * 6;
                  attn_add(p[0], p[1], make_float4(p[2], p[3], p[4], p[5]), top, sum, v);
                }
            }
            if (e < items && set == 0) {
              const int r = e / (HD / 4), d = (e - r * (HD / 4)) * 4;
              attn_store(A, seq, at, group, S::kRows, r, d, HD, sum, v);
            }
          }
          __syncthreads();
        }
      }
      first_seg = false;
      fresh = true;
      begins_here = true;
      if (u + 1 < n_units) at = attn_place<NQ>(s_tab, c.n_seqs, group, share0 + u + 1, &seq);
    }
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
}

}  // namespace cats
