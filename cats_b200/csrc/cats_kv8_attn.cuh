// Attention of the newest tokens over the paged 8-bit cache (cats_kv8.cuh).
#pragma once

#include "cats_kv8.cuh"

namespace cats {

template <typename T>
struct KvAttnArgs {
  const T* q;             // [tokens, nh, hd], tokens q_ld elements apart
  long long q_ld;
  T* out;                 // [tokens, nh, hd]
  const int* cu;
  int uniform, tokens, nh, layer;
  float scale;            // of the scores, times log2(e)
};

// One warp per (token, query head), lanes over head_dim: running maximum and sum over the keys.
template <typename T>
__global__ void __launch_bounds__(256) k_kv8_attend_simple(const cats_kv8 c, const KvAttnArgs<T> A) {
  pdl_wait();
  const int lane = threadIdx.x & 31, hd = c.head_dim, per = hd >> 5;
  const long long w = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (w >= (long long)A.tokens * A.nh) return;
  const int t = (int)(w / A.nh), h = (int)(w - (long long)t * A.nh), kvh = h / (A.nh / c.n_kv_heads);
  int b = 0;
  if (!A.cu) b = t / A.uniform;
  else
    while (b + 1 < c.n_seqs && A.cu[b + 1] <= t) ++b;
  const KvSpan sp = kv_span(A.cu, A.uniform, b);
  const int len = c.lens[b];
  const bool fits = len >= 0 && len <= c.max_pages * c.page;
  if (!fits && lane == 0) kv_flag(c, KV_TOO_LONG);
  const int keys = fits ? min(len, len - sp.count + (t - sp.first) + 1) : 0;
  float q[4], o[4], m = -INFINITY, l = 0.f;
  for (int i = 0; i < per; ++i) {
    q[i] = VecT<T>::to_f(A.q[(size_t)t * A.q_ld + (size_t)h * hd + lane * per + i]);
    o[i] = 0.f;
  }
  for (int p = 0; p < keys; ++p) {
    const int page = c.table[(size_t)b * c.max_pages + p / c.page];
    if (page < 0 || page >= c.n_pages) {
      if (lane == 0) kv_flag(c, KV_BAD_PAGE);
      continue;
    }
    const uint8_t* kr = kv_rows(c, A.layer, page, 0, kvh) + (size_t)(p % c.page) * hd + lane * per;
    const uint8_t* vr = kv_rows(c, A.layer, page, 1, kvh) + (size_t)(p % c.page) * hd + lane * per;
    auto value = [](uint8_t code) {
      const uint32_t two = e4m3_to_f16x2(code);
      return __low2float(*reinterpret_cast<const __half2*>(&two));
    };
    float s = 0.f;
    for (int i = 0; i < per; ++i) s = fmaf(q[i], value(kr[i]), s);
    s = warp_sum(s) * *kv_scale(c, A.layer, page, 0, kvh) * A.scale;
    const float m_new = fmaxf(m, s);
    const float f = m == -INFINITY ? 0.f : exp2f(m - m_new), e = exp2f(s - m_new);
    const float ev = e * *kv_scale(c, A.layer, page, 1, kvh);
    l = l * f + e;
    for (int i = 0; i < per; ++i) o[i] = o[i] * f + ev * value(vr[i]);
    m = m_new;
  }
  for (int i = 0; i < per; ++i)
    A.out[(size_t)w * hd + lane * per + i] = VecT<T>::from_f(keys > 0 ? o[i] / l : 0.f);
}

}  // namespace cats
