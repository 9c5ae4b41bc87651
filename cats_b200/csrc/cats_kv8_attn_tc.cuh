// Attention of many new tokens over the paged 8-bit cache, on the 5th-generation tensor cores.
//
// With 128 rows ((token, query head of the group) pairs) to a key head the work is no longer bound by
// the codes' bytes but by the two products, and both fill a tcgen05 tile: S = Q K^T and O += P V, 128
// rows x 128 positions, accumulators in tensor memory (S 128 columns, O head_dim columns).  A CTA
// takes a tile of rows through its positions, 128 at a time:
//   1 codes become half precision, exactly, and go to shared memory, both K-major under the 128-byte
//     swizzle: K, in registers since the last step, as it lies; V, copied to shared memory meanwhile (a
//     gather of four positions per lane from global memory costs L1 a lookup per row), transposed;
//   2 the next step's codes are asked for;
//   3 one thread issues S = Q K^T;
//   4 four threads per row take a quarter of a row of S each from tensor memory: maximum, exponentials, sum;
//     the weights go to shared memory in half precision;
//   5 one thread issues O += P V, which runs while the next step's codes are converted (V has two
//     buffers; the next S is committed behind it, so waiting for S waits for it too).
// Precision as in cats_kv8_attn.cuh (queries and weights in half precision, scales of pages in the
// exponents), and so is the way the positions are dealt out to the CTAs.  A NaN among the values must
// only reach the rows that see its position: it is taken out of the product, and the least such
// position of every channel is kept for the end.
// A page whose values' exponent lies far below the others' of a step would lose its weights in half precision: the
// positions of a step go in classes of pages that lie close together, one product for each (nearly always one).
// Bound: latency.  A step takes 3.3 us (head_dim 128; 2 x 256 tokens x 4 heads per key head over 2000 ..
// 6000 positions: 128 us, 254 TFLOP/s): conversions 0.6, asking for the next codes 0.45, exponentials 0.35,
// the exchange of maxima 0.3, S 0.2, writing the weights 0.1 and the rest barriers and round trips, which
// follow one another in all 16 warps; the MMA pipe is busy 14 % of the time and instructions are issued
// 41 % of it.  A tile goes through all positions of its sequence, also those behind its last row (their codes are not
// loaded): a prompt into an empty cache takes twice the steps that it needs (four of 700 .. 4096 tokens: 1163 us, 169
// TFLOP/s).  Slower: S issued a step ahead into a second S (135 us), two CTAs an SM with steps of 64
// positions (137 us: as many instructions a step and thread for half the positions).
#pragma once

#include "cats_dense.cuh"
#include "cats_kv8_attn.cuh"

namespace cats {

constexpr int kTcRows = 128, kTcKeys = 128, kTcThreads = 512;
using TcShape = AttnShape<16>;
static_assert(TcShape::kRows == kTcRows && TcShape::kUnit == kTcKeys && TcShape::kThreads == kTcThreads, "tile");

constexpr uint32_t kTcBlock = 128 * 128;               // 128 rows of 64 half-precision values
__host__ __device__ constexpr size_t attn_tc_smem(int hd) {
  // Q, K: hd / 64 blocks; V: two buffers of two blocks of hd rows; P: two blocks; V's codes
  return 1024 + (size_t)(hd / 64) * kTcBlock * 2 + (size_t)2 * 2 * hd * 128 + 2 * kTcBlock + kTcBlock;
}

// byte of 16-byte chunk `chunk` of row `row` in a block under the 128-byte swizzle
__device__ __forceinline__ uint32_t tc_at(int row, int chunk) { return (uint32_t)row * 128 + (((uint32_t)chunk ^ (row & 7)) << 4); }
__device__ __forceinline__ void sts16(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ void sts8(uint32_t addr, uint32_t a, uint32_t b) {
  asm volatile("st.shared.v2.u32 [%0], {%1, %2};" ::"r"(addr), "r"(a), "r"(b) : "memory");
}
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, float* v) {
  uint32_t r[32];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const float* v) {
  uint32_t r[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) r[i] = __float_as_uint(v[i]);
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::"r"(r[0]),
      "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
      "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(taddr)
      : "memory");
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}
// half precision, M = 128, both operands K-major
__host__ __device__ constexpr uint32_t tc_idesc(int n) { return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(128 >> 4) << 24); }

template <typename T, int HD>
__global__ void __launch_bounds__(kTcThreads, 1) k_kv8_attend_tc(const cats_kv8 c, const KvAttnArgs<T> A) {
  constexpr int NQ = 16, HB = HD / 64, kChunks = HD / 16, NK = HD / 64;   // NK: 16-byte loads of K per thread
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  __shared__ AttnTable s_tab;
  __shared__ AttnPlan s_plan;
  __shared__ int s_warp[kTcThreads / 32], s_last, s_owners[2], s_ctl[2];
  __shared__ uint64_t s_bar;
  __shared__ uint32_t s_tmem;
  __shared__ int s_id[2][8];                             // page of 16 positions each of this and the next step,
  __shared__ __align__(8) float s_ks[2][8];              // scale of its keys,
  __shared__ __align__(8) int s_ev[2][8];                // exponent of its values' scale (kAttnNoExp: no page)
  __shared__ int2 s_span[2];                             // and a step's largest and least of them
  __shared__ float s_x[4][kTcRows];                      // what the four threads of a row tell one another
  __shared__ int s_nan[HD];
  pdl_wait();
  pdl_launch_dependents();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int row = (warp & 3) * 32 + lane, quarter = warp >> 2;
  const int page_mask = c.page - 1;                      // (pages are powers of two)
  const int page_log = 31 - __clz(c.page);
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t q_u = base, k_u = q_u + HB * kTcBlock, v_u = k_u + HB * kTcBlock, p_u = v_u + 2 * 2 * HD * 128;
  const uint32_t raw_u = p_u + 2 * kTcBlock;               // rows 128 bytes apart, chunks exchanged by row / 4
  const uint32_t bar = smem_u32(&s_bar);

  const AttnPlan plan = attn_table<NQ, HD>(c, A, s_tab, &s_plan, s_warp);
  if ((int)blockIdx.x >= plan.ctas) return;
  const int group = A.nh / c.n_kv_heads;
  const int share0 = attn_share<NQ>(s_tab, plan, c.n_seqs, group, blockIdx.x);
  const int share1 = attn_share<NQ>(s_tab, plan, c.n_seqs, group, blockIdx.x + 1);
  if (share1 <= share0) return;
  if (tid == 0) {
    mbar_init(bar, 1);
    s_ctl[0] = 0;
    s_ctl[1] = A.wait_kc;
    mbar_fence_init();
  }
  if (warp == 0) tmem_alloc(smem_u32(&s_tmem), 256);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s_tmem, t_lane = (uint32_t)((warp & 3) * 32) << 16;
  const uint32_t t_s = tmem, t_o = tmem + 128;
  uint32_t phase = 0;
  // one thread's MMAs so far are complete (a wait that runs out is recorded and the work goes on to
  // its end without waiting; no later wait blocks)
  auto wait_mma = [&]() {
    mbar_wait_warp(bar, phase, s_ctl);
    phase ^= 1;
    tc_fence_after();
  };

  const uint8_t* layer_codes = kv_rows(c, A.layer, 0, 0, 0);
  const float* layer_scales = kv_scale(c, A.layer, 0, 0, 0);
  const size_t block = kv_block(c), v_off = (size_t)c.n_kv_heads * block;
  bool first_seg = true;

  for (int u = share0; u < share1;) {
    AttnSeq seq;
    AttnPlace at = attn_place<NQ>(s_tab, c.n_seqs, group, u, &seq);
    const int u_first = at.unit, u_end = min(seq.units, at.unit + share1 - u);       // units of this segment here
    const int rows = min(kTcRows, seq.count * group - at.tile * kTcRows);
    const int last = min(seq.count - 1, (at.tile * kTcRows + kTcRows - 1) / group);
    const int end = min(seq.len, seq.len - seq.count + last + 1);    // positions that the tile's rows see
    const int* table = c.table + (size_t)at.b * c.max_pages;

    // pages of a step: looked up by the first eight threads, one step before its codes are asked for
    int n_id = -1, n_ev = kAttnNoExp;
    float n_ks = 0.f;
    auto look = [&](int unit) {
      n_id = -1;
      n_ks = 0.f;
      n_ev = kAttnNoExp;
      const int p = unit * kTcKeys + 16 * tid;
      if (tid < 8 && unit < u_end && p < end) {
        const int id = table[p >> page_log];
        if (id < 0 || id >= c.n_pages) {
          kv_flag(c, KV_BAD_PAGE);
        } else {
          n_id = id;
          n_ks = layer_scales[(size_t)id * 2 * c.n_kv_heads + at.head];
          n_ev = attn_exp_of(layer_scales[((size_t)id * 2 + 1) * c.n_kv_heads + at.head]);
        }
      }
    };
    auto keep = [&](int unit) {
      if (tid < 8) {
        s_id[unit & 1][tid] = n_id;
        s_ks[unit & 1][tid] = n_ks;
        s_ev[unit & 1][tid] = n_ev;
        const int high = __reduce_max_sync(0xffu, n_ev), low = __reduce_min_sync(0xffu, n_id >= 0 ? n_ev : -kAttnNoExp);
        s_span[unit & 1] = make_int2(high, low);         // (the same from all eight)
      }
    };
    // a step's codes: 16 bytes of rows tid / kChunks + i * (512 / kChunks)
    uint4 kc[NK];
    auto fetch = [&](int unit) {
      const int kb = unit * kTcKeys, ch = tid % kChunks;
#pragma unroll
      for (int i = 0; i < NK; ++i) {
        const int r = tid / kChunks + i * (kTcThreads / kChunks);
        const int id = s_id[unit & 1][r >> 4];
        const bool in = id >= 0 && kb + r < end;
        const uint8_t* src = layer_codes + ((size_t)(in ? id : 0) * 2 * c.n_kv_heads + at.head) * block +
                             (size_t)(r & page_mask) * HD + 16 * ch;
        kc[i] = make_uint4(0, 0, 0, 0);
        if (in) kc[i] = ldg_stream(reinterpret_cast<const uint4*>(src));
        const uint32_t to = raw_u + r * 128 + ((ch ^ ((r >> 2) & 7)) << 4);
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(src + v_off), "r"(in ? 16 : 0) : "memory");
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
    auto settle = [&]() { asm volatile("cp.async.wait_all;" ::: "memory"); };   // (then a barrier)

    look(u_first);
    // ---- queries: four threads per row, a quarter of the channels each
    const int rr = at.tile * kTcRows + row, tok = rr / group, hq = at.head * group + rr - tok * group;
    const bool on = row < rows;
    const int lim = on ? min(seq.len, seq.len - seq.count + tok + 1) : 0;
    float f;
    {
      constexpr int NC = HD / 4;
      float q[NC], top = 0.f;
      const T* src = A.q + (size_t)(seq.first + tok) * A.q_ld + (size_t)hq * HD + quarter * NC;
#pragma unroll
      for (int i = 0; i < NC; i += 8) {
#pragma unroll
        for (int k = 0; k < 8; ++k) q[i + k] = 0.f;
        if (on) load8_cached(src + i, q + i);
      }
#pragma unroll
      for (int i = 0; i < NC; ++i) {
        const float a = fabsf(q[i]);
        if (a <= 3.402823466e38f) top = fmaxf(top, a);
      }
      __syncthreads();                                   // s_x, s_id, s_nan of the last segment are read
      keep(u_first);
      look(u_first + 1);
      keep(u_first + 1);
      for (int d = tid; d < HD; d += kTcThreads) s_nan[d] = 0x7fffffff;
      s_x[quarter][row] = top;
      __syncthreads();
      top = fmaxf(fmaxf(s_x[0][row], s_x[1][row]), fmaxf(s_x[2][row], s_x[3][row]));
      const int e = top > 0.f ? min(max(kv_exp_of(top) + 1, -126), 126) : 0;
      const float inv = kv_pow2(-e);
      f = kv_pow2(e) * A.scale;
#pragma unroll
      for (int i = 0; i < NC; i += 8) {
        const int d = quarter * NC + i;
        sts16(q_u + (d / 64) * kTcBlock + tc_at(row, (d % 64) / 8), half2_bits(q[i] * inv, q[i + 1] * inv),
              half2_bits(q[i + 2] * inv, q[i + 3] * inv), half2_bits(q[i + 4] * inv, q[i + 5] * inv),
              half2_bits(q[i + 6] * inv, q[i + 7] * inv));
      }
    }
    fetch(u_first);
    settle();
    __syncthreads();
    float m = -INFINITY, l = 0.f;
    int ec = kAttnNoExp;                                 // exponent that O is held at

    for (int unit = u_first; unit < u_end; ++unit) {
      const int kb = unit * kTcKeys;
      // ---- 1 codes to half precision
#pragma unroll
      for (int i = 0; i < NK; ++i) {
        const int r = tid / kChunks + i * (kTcThreads / kChunks), ch = tid % kChunks;
        const uint32_t w[4] = {kc[i].x, kc[i].y, kc[i].z, kc[i].w};
        uint32_t h[8];
#pragma unroll
        for (int k = 0; k < 4; ++k) e4m3x4_to_f16x2(w[k], h[2 * k], h[2 * k + 1]);
        const uint32_t to = k_u + (ch / 4) * kTcBlock;
        // (the lanes of a row's second block write their chunks the other way round: no bank twice)
        const int o = ch / 4;
        const uint32_t a0 = to + tc_at(r, 2 * (ch % 4) + o), a1 = to + tc_at(r, 2 * (ch % 4) + 1 - o);
        if (o == 0) {
          sts16(a0, h[0], h[1], h[2], h[3]);
          sts16(a1, h[4], h[5], h[6], h[7]);
        } else {
          sts16(a0, h[4], h[5], h[6], h[7]);
          sts16(a1, h[0], h[1], h[2], h[3]);
        }
      }
      if (warp < 2 * kChunks) {
        const uint32_t vb = v_u + (unit & 1) * (2 * HD * 128) + (lane >> 4) * (HD * 128) + (lane & 1) * 8;
        uint2 vc[4];                                     // 8 channels of positions 4 lane ..
#pragma unroll
        for (int i = 0; i < 4; ++i) vc[i] = lds2(raw_u + (4 * lane + i) * 128 + (((warp >> 1) ^ (lane & 7)) << 4) + (warp & 1) * 8);
        uint32_t nan = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          nan |= ((vc[i].x & 0x7f7f7f7fu) + 0x01010101u) | ((vc[i].y & 0x7f7f7f7fu) + 0x01010101u);
        const bool bad = (nan & 0x80808080u) != 0;
#pragma unroll
        for (int k = 0; k < 2; ++k) {                    // four channels at a time
          uint32_t w[4] = {k ? vc[0].y : vc[0].x, k ? vc[1].y : vc[1].x, k ? vc[2].y : vc[2].x, k ? vc[3].y : vc[3].x};
          if (bad) {
            for (int i = 0; i < 4; ++i)
              for (int j = 0; j < 4; ++j)
                if (((w[i] >> (8 * j)) & 0x7fu) == 0x7fu) {
                  atomicMin(&s_nan[8 * warp + 4 * k + j], kb + 4 * lane + i);
                  w[i] &= ~(0xffu << (8 * j));
                }
          }
          // four positions of each channel: bytes (p0, p1, p2, p3)
          const uint32_t a = __byte_perm(w[0], w[1], 0x5140), b = __byte_perm(w[2], w[3], 0x5140);
          const uint32_t cc = __byte_perm(w[0], w[1], 0x7362), d = __byte_perm(w[2], w[3], 0x7362);
          const uint32_t ch[4] = {__byte_perm(a, b, 0x5410), __byte_perm(a, b, 0x7632), __byte_perm(cc, d, 0x5410),
                                  __byte_perm(cc, d, 0x7632)};
#pragma unroll
          for (int j = 0; j < 4; ++j) {                  // row 8 warp + 4 k + j: its chunks are exchanged by 4 k + j
            uint32_t lo, hi;
            e4m3x4_to_f16x2(ch[j], lo, hi);
            sts8(vb + (8 * warp + 4 * k + j) * 128 + ((((lane & 15) >> 1) ^ (4 * k + j)) << 4), lo, hi);
          }
        }
      }
      fence_proxy_async_smem();
      tc_fence_before();
      __syncthreads();
      // ---- 3 S = Q K^T
      if (tid == 0) {
        tc_fence_after();
#pragma unroll
        for (int k = 0; k < HD / 16; ++k)
          umma_f16(t_s, umma_desc_k128(q_u + (k / 4) * kTcBlock) + 2 * (k % 4), umma_desc_k128(k_u + (k / 4) * kTcBlock) + 2 * (k % 4),
                   tc_idesc(kTcKeys), k > 0);
        umma_commit(bar);
      }
      // ---- 2 the next step's codes (and the page numbers of the one after it)
      look(unit + 2);
      if (unit + 1 < u_end) fetch(unit + 1);
      int high = s_span[unit & 1].x;
      const int low = s_span[unit & 1].y;
      const float2 ks = *reinterpret_cast<const float2*>(&s_ks[unit & 1][2 * quarter]);
      const int2 evs = *reinterpret_cast<const int2*>(&s_ev[unit & 1][2 * quarter]);
      wait_mma();
      // ---- 4 a quarter of a row each: weights
      const int k0 = kb + 32 * quarter;
      float s[32];
      // scores of sixteen positions (the same page for all), -inf where the row does not see them
      auto score = [&](int j) {
        const float by = (j ? ks.y : ks.x) * f;
#pragma unroll
        for (int i = 0; i < 16; ++i) s[16 * j + i] *= by;
        const bool none = (j ? evs.y : evs.x) == kAttnNoExp;
        if (k0 + 16 * j + 16 > lim || none) {
          const int sees = none ? 0 : lim - k0 - 16 * j;                       // of the sixteen
#pragma unroll
          for (int i = 0; i < 16; ++i)
            if (i >= sees) s[16 * j + i] = -INFINITY;
        }
      };
      auto rescale = [&](float by) {
#pragma unroll
        for (int d = 0; d < HD / 4; d += 16) {
          float o[16];
          tmem_ld16(t_o + t_lane + quarter * (HD / 4) + d, o);
#pragma unroll
          for (int i = 0; i < 16; ++i) o[i] *= by;
          tmem_st16(t_o + t_lane + quarter * (HD / 4) + d, o);
        }
      };
      // The exponent of O for the positions whose exponents are `high` and less, and the least that can go with
      // them: sixteen positions are a k-step of the product, those within kAttnSpan of O's exponent take part, the
      // others' weights are 0.  In earnest all of them take part.
      int least = kAttnNoExp + 1;
      auto follow = [&](int high) {
        float by = 1.f;
        least = kAttnNoExp + 1;
        if (high > ec + kAttnSpan || low < ec - kAttnSpan) {
          const int to = low < high - kAttnSpan ? high - kAttnSpan : high;
          least = to - kAttnSpan;
          by = kv_pow2(max(ec - to, -126));
          ec = to;
        }
        return by;
      };
      auto weigh = [&](int j, int high) {
        const int ev = j ? evs.y : evs.x;
        const uint32_t to = p_u + (quarter >> 1) * kTcBlock;
        const uint32_t p0 = to + tc_at(row, 4 * (quarter & 1) + 2 * j), p1 = to + tc_at(row, 4 * (quarter & 1) + 2 * j + 1);
        if (ev < least || ev > high) {                   // (the same for all lanes of a warp)
          sts16(p0, 0, 0, 0, 0);
          sts16(p1, 0, 0, 0, 0);
          return;
        }
        const float ref = m == -INFINITY ? 0.f : m - (float)(ev - ec);
        float part = 0.f;
        float* x = s + 16 * j;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          x[i] = ex2(x[i] - ref);
          part += x[i];
        }
        l = fmaf(part, kv_pow2(ec - ev), l);
        sts16(p0, half2_bits(x[0], x[1]), half2_bits(x[2], x[3]), half2_bits(x[4], x[5]), half2_bits(x[6], x[7]));
        sts16(p1, half2_bits(x[8], x[9]), half2_bits(x[10], x[11]), half2_bits(x[12], x[13]), half2_bits(x[14], x[15]));
      };
      // ---- 5 O += P V
      auto multiply = [&](bool add) {
        fence_proxy_async_smem();
        tc_fence_before();
        __syncthreads();
        if (tid == 0) {
          tc_fence_after();
          const uint32_t vb = v_u + (unit & 1) * (2 * HD * 128);
#pragma unroll
          for (int k = 0; k < kTcKeys / 16; ++k)
            umma_f16(t_o, umma_desc_k128(p_u + (k / 4) * kTcBlock) + 2 * (k % 4), umma_desc_k128(vb + (k / 4) * (HD * 128)) + 2 * (k % 4),
                     tc_idesc(HD), add || k > 0);
        }
      };
      tmem_ld32(t_s + t_lane + 32 * quarter, s);
      float top = -INFINITY;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        score(j);
#pragma unroll
        for (int i = 0; i < 16; ++i) top = fmaxf(top, s[16 * j + i]);
      }
      s_x[quarter][row] = top;
      asm volatile("bar.sync %0, 128;" ::"r"(1 + (warp & 3)) : "memory");    // the four warps of these rows
      top = fmaxf(fmaxf(s_x[0][row], s_x[1][row]), fmaxf(s_x[2][row], s_x[3][row]));
      const float by = follow(high);
      if (__any_sync(0xffffffffu, top > m + kAttnSlack || by != 1.f)) {
        const float to = fmaxf(top, m), down = m == -INFINITY ? 0.f : ex2(m - to);
        m = to;
        l *= down;
        if (unit > u_first) rescale(by * down);
      }
#pragma unroll
      for (int j = 0; j < 2; ++j) weigh(j, high);
      settle();
      multiply(unit > u_first);
      // pages of this step whose exponents lie far below the others': one class of them after the other
      while (least > low) {
        int next = kAttnNoExp;
        for (int z = 0; z < 8; ++z)
          if (s_ev[unit & 1][z] < least) next = max(next, s_ev[unit & 1][z]);
        high = next;
        if (tid == 0) umma_commit(bar);
        wait_mma();                                      // before P and O change
        rescale(follow(high));
        tmem_ld32(t_s + t_lane + 32 * quarter, s);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          score(j);
          weigh(j, high);
        }
        multiply(true);
      }
      if (tid == 0 && unit + 1 == u_end) umma_commit(bar);
      keep(unit + 2);                                    // (this step's are read; the next barrier is before their use)
    }
    wait_mma();

    // ---- the segment's end
    __syncthreads();
    s_x[quarter][row] = l;
    __syncthreads();
    l = (s_x[0][row] + s_x[1][row]) + (s_x[2][row] + s_x[3][row]);
    const bool whole = u_first == 0 && u_end == seq.units;
    const float held = kv_pow2(max(ec, -126));           // (no page seen: O is zero)
    float* part = A.parts + (size_t)(blockIdx.x * 2 + (first_seg ? 0 : 1)) * attn_part_floats(kTcRows, HD);
#pragma unroll
    for (int d0 = 0; d0 < HD / 4; d0 += 16) {
      float o[16];
      tmem_ld16(t_o + t_lane + quarter * (HD / 4) + d0, o);
      if (on) {
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
          const int d = quarter * (HD / 4) + d0 + i;
          float4 v = make_float4(o[i] * held, o[i + 1] * held, o[i + 2] * held, o[i + 3] * held);
          const float bad = __uint_as_float(0x7fc00000u);
          if (s_nan[d] < lim) v.x = bad;
          if (s_nan[d + 1] < lim) v.y = bad;
          if (s_nan[d + 2] < lim) v.z = bad;
          if (s_nan[d + 3] < lim) v.w = bad;
          if (whole) {
            attn_store(A, seq, at, group, kTcRows, row, d, HD, l, v);
          } else {
            float* dst = part + (size_t)row * (HD + 2);
            *reinterpret_cast<float2*>(dst + d) = make_float2(v.x, v.y);
            *reinterpret_cast<float2*>(dst + d + 2) = make_float2(v.z, v.w);
            if (d == 0) *reinterpret_cast<float2*>(dst + HD) = make_float2(m, l);
          }
        }
      }
    }
    tc_fence_before();                                   // (tensor memory is read; the next MMA is behind a barrier)
    if (!whole) {
      // as in k_kv8_attend: the CTA that brings the last part joins them, in the order of the CTAs
      const int u0 = u - u_first;
      __threadfence();
      __syncthreads();
      if (tid == 0) {
        attn_owners<NQ>(s_tab, plan, c.n_seqs, group, at.b, u0, seq.units, &s_owners[0], &s_owners[1]);
        s_last = atomicAdd(A.counters + s_owners[0], 1) == s_owners[1] - s_owners[0];
        if (s_last) A.counters[s_owners[0]] = 0;
      }
      __syncthreads();
      if (s_last) {
        __threadfence();
        const int c0 = s_owners[0], c1 = s_owners[1];
        const int first_begins = attn_share<NQ>(s_tab, plan, c.n_seqs, group, c0);
        const int items = rows * (HD / 4);
        for (int e0 = tid; e0 < items; e0 += 4 * kTcThreads) {         // four at a time: their loads go together
          float top[4], sum[4];
          float4 v[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            top[k] = -INFINITY;
            sum[k] = 0.f;
            v[k] = make_float4(0.f, 0.f, 0.f, 0.f);
          }
#pragma unroll 2
          for (int x = c0; x <= c1; ++x) {
            const int slot = x > c0 || first_begins >= u0 ? 0 : 1;
            const float* src = A.parts + (size_t)(2 * x + slot) * attn_part_floats(kTcRows, HD);
            float2 ml[4], a[4], b[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const int e = min(e0 + k * kTcThreads, items - 1), r = e / (HD / 4), d = (e - r * (HD / 4)) * 4;
              const float* p = src + (size_t)r * (HD + 2);
              ml[k] = __ldcg(reinterpret_cast<const float2*>(p + HD));
              a[k] = __ldcg(reinterpret_cast<const float2*>(p + d));
              b[k] = __ldcg(reinterpret_cast<const float2*>(p + d + 2));
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) attn_add(ml[k].x, ml[k].y, make_float4(a[k].x, a[k].y, b[k].x, b[k].y), top[k], sum[k], v[k]);
          }
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int e = e0 + k * kTcThreads, r = e / (HD / 4), d = (e - r * (HD / 4)) * 4;
            if (e < items) attn_store(A, seq, at, group, kTcRows, r, d, HD, sum[k], v[k]);
          }
        }
      }
    }
    first_seg = false;
    u += u_end - u_first;
  }
  if (tid == 0 && s_ctl[0]) kv_flag(c, KV_WAIT);
  tc_fence_before();
  __syncthreads();
  if (warp == 0) tmem_dealloc(tmem, 256);
}

}  // namespace cats
