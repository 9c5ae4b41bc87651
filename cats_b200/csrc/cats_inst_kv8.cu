// extern "C" entry points of the paged 8-bit cache and of beam selection: argument checks, grid
// sizing and launches.
#include <math.h>

#include "cats_beam.cuh"
#include "cats_kv8_run.cuh"
#include "cats_kv8_steps.cuh"

namespace {

using namespace cats;

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
bool known_dtype(int d) { return d == CATS_F32 || d == CATS_F16 || d == CATS_BF16; }
int esize(int dtype) { return dtype == CATS_F32 ? 4 : 2; }

int check_cache(const cats_kv8* c) {
  if (!c || !c->codes || !c->scales || !c->table || !c->lens || !c->refs || !c->status) return CATS_ERR_NULL;
  if (!aligned16(c->codes)) return CATS_ERR_ALIGN;
  if (c->n_layers < 1 || c->n_pages < 1 || c->n_seqs < 1 || c->n_seqs > kKvMaxSeqs || c->max_pages < 1 ||
      c->n_kv_heads < 1 || c->n_kv_heads > 1024)
    return CATS_ERR_RANGE;
  if (c->page != 16 && c->page != 32 && c->page != 64 && c->page != 128) return CATS_ERR_RANGE;
  if (c->head_dim != 32 && c->head_dim != 64 && c->head_dim != 96 && c->head_dim != 128) return CATS_ERR_RANGE;
  if ((long long)c->max_pages * c->page > 0x7fffffffLL || (long long)c->max_pages * c->n_seqs > 0x7fffffffLL) return CATS_ERR_RANGE;
  return CATS_OK;
}

// New tokens: `tokens` of them, by cu or the same number of every sequence.
int check_tokens(const cats_kv8* c, const int* cu, int tokens, int n_heads) {
  if (tokens < 1 || n_heads < 1 || n_heads % c->n_kv_heads || n_heads > 16384) return CATS_ERR_RANGE;
  if ((long long)tokens * n_heads > 0x7fffffffLL) return CATS_ERR_RANGE;
  if (!cu && tokens % c->n_seqs) return CATS_ERR_RANGE;
  return CATS_OK;
}

// The units of a call have to fit 32 bits (cats_kv8_attn.cuh).
bool units_fit(const cats_kv8* c, int tokens, int n_heads) {
  const double units = (double)c->max_pages * c->page / AttnShape<2>::kUnit + 1 + AttnShape<2>::kSwitch;
  return units * ((double)tokens * n_heads / AttnShape<1>::kRows + (double)c->n_kv_heads * c->n_seqs) < 2147483648.0;
}

template <typename T>
cudaError_t append(const cats_kv8& c, int layer, const void* qkv, long long ld, const int* cu, int tokens,
                   const void* cosv, const void* sinv, void* q_out, int nh, cudaStream_t st) {
  KvAppendArgs<T> A;
  A.qkv = (const T*)qkv;
  A.ld = ld;
  A.cosv = (const T*)cosv;
  A.sinv = (const T*)sinv;
  A.q_out = (T*)q_out;
  A.cu = cu;
  A.uniform = cu ? 0 : tokens / c.n_seqs;
  A.tokens = tokens;
  A.nh = nh;
  A.layer = layer;
  // One new token of every sequence (a decode step): a warp per block of rows; else half a page's
  // rows (a quarter of a 128-row page's) side by side, two (four) of them in a thread's registers.
  const bool single = !cu && A.uniform == 1;
  const int tpr = c.head_dim / 16;
  const int rpt = single ? 1 : c.page == 128 ? 4 : 2;
  const int threads = single ? 32 : (c.page / rpt * tpr + 31) / 32 * 32;
  const long long units = cu ? (long long)tokens / c.page + 2LL * (tokens < c.n_seqs ? tokens : c.n_seqs)
                             : (long long)c.n_seqs * kv_units(A.uniform, c.page);
  // A CTA goes through several blocks of rows, the next one's loads under way, where that still leaves
  // four CTAs per SM and more (finding the page costs as long as a block's load).
  A.kv_heads = 1;
  while (!single && A.kv_heads < 16 && units * 2 * c.n_kv_heads / (2 * A.kv_heads) >= 4LL * dev_info().sms) A.kv_heads *= 2;
  const long long kv_blocks = units * ((2 * c.n_kv_heads + A.kv_heads - 1) / A.kv_heads);
  // query CTAs: a thread keeps its token's rotation for as many heads as still leave work for all SMs
  const long long tiles = (tokens + threads / tpr - 1) / (threads / tpr);
  A.q_heads = tiles * ((nh + 15) / 16) >= 4LL * dev_info().sms ? 16 : 4;
  const long long q_blocks = q_out ? tiles * ((nh + A.q_heads - 1) / A.q_heads) : 0;
  if (kv_blocks + q_blocks > 0x7fffffffLL) return cudaErrorInvalidValue;
  A.kv_blocks = (int)kv_blocks;
  const dim3 grid((unsigned)(kv_blocks + q_blocks)), block(threads);
  if (single) return launch(k_kv8_append<T, 1>, grid, block, 0, st, c, A);
  if (rpt == 4) return launch(k_kv8_append<T, 4>, grid, block, 0, st, c, A);
  return launch(k_kv8_append<T, 2>, grid, block, 0, st, c, A);
}

template <typename T>
cudaError_t attend(const cats_kv8& c, int layer, const void* q, long long q_ld, const int* cu, int tokens, int nh,
                   float scale, void* out, void* ws, cudaStream_t st) {
  KvAttnArgs<T> A;
  A.q = (const T*)q;
  A.q_ld = q_ld;
  A.out = (T*)out;
  A.cu = cu;
  A.uniform = cu ? 0 : tokens / c.n_seqs;
  A.tokens = tokens;
  A.nh = nh;
  A.layer = layer;
  A.scale = scale * 1.4426950408889634f;
  A.parts = (float*)ws;
  A.ctas = dev_info().sms < kKvRefusedAt - 1 ? dev_info().sms : kKvRefusedAt - 1;   // (a counter each)
  A.counters = c.status + 1;
  A.wait_kc = wait_kcycles();
  return inst_kv8_attend<T>(c, A, st);
}

// Parts of a row: as many CTAs as run at once (four per SM; a second, partly filled round costs up to
// a third), no part below a tile of the kernel, and the keys of an
// item's parts (8 bytes, `beams * splits * k` of them) within 48 KB of the joining CTA.
int beam_splits(long long rows, int beams, int vocab, int k) {
  const long long want = 4LL * dev_info().sms / rows, tiles = ((long long)vocab + kBeamTile - 1) / kBeamTile;
  const long long most = 6144 / ((long long)beams * k);
  long long s = want < tiles ? want : tiles;
  if (s > most) s = most;
  return s < 1 ? 1 : (int)s;
}

}  // namespace

extern "C" {

int cats_kv8_grow(const cats_kv8* cache, const int* cu, int n_new, void* stream) {
  int s = check_cache(cache);
  if (s) return s;
  if (!cu && n_new < 1) return CATS_ERR_RANGE;
  return launch_status(launch(k_kv8_grow, dim3(1), dim3(kPlanThreads), 0, (cudaStream_t)stream, *cache, cu, n_new));
}

int cats_kv8_append(const cats_kv8* cache, int layer, const void* qkv, long long ld, const int* cu, int n_tokens,
                    const void* cos_table, const void* sin_table, int rope_len, void* q_out, int n_heads, int dtype,
                    void* stream) {
  if (!known_dtype(dtype)) return CATS_ERR_DTYPE;
  int s = check_cache(cache);
  if (s) return s;
  if ((s = check_tokens(cache, cu, n_tokens, n_heads))) return s;
  if (layer < 0 || layer >= cache->n_layers) return CATS_ERR_RANGE;
  if (!qkv || (!cos_table) != (!sin_table)) return CATS_ERR_NULL;
  if (cos_table && rope_len < cache->max_pages * cache->page) return CATS_ERR_RANGE;
  const long long width = ((long long)n_heads + 2 * cache->n_kv_heads) * cache->head_dim;
  if (ld < width) return CATS_ERR_RANGE;
  if (!aligned16(qkv) || (ld * esize(dtype)) % 16 || !aligned16(cos_table) || !aligned16(sin_table) ||
      !aligned16(q_out))
    return CATS_ERR_ALIGN;
  cudaStream_t st = (cudaStream_t)stream;
  cudaError_t e;
  if (dtype == CATS_F32)
    e = append<float>(*cache, layer, qkv, ld, cu, n_tokens, cos_table, sin_table, q_out, n_heads, st);
  else if (dtype == CATS_F16)
    e = append<__half>(*cache, layer, qkv, ld, cu, n_tokens, cos_table, sin_table, q_out, n_heads, st);
  else
    e = append<__nv_bfloat16>(*cache, layer, qkv, ld, cu, n_tokens, cos_table, sin_table, q_out, n_heads, st);
  return launch_status(e);
}

size_t cats_kv8_attend_bytes(const cats_kv8* cache, int n_tokens, int n_heads) {
  if (check_cache(cache) || n_tokens < 1 || n_heads < 1) return 0;
  return sizeof(float) * 2 * (size_t)dev_info().sms * attn_part_floats(attn_part_rows(*cache, n_tokens, n_heads), cache->head_dim);
}

int cats_kv8_attend(const cats_kv8* cache, int layer, const void* q, long long q_ld, const int* cu, int n_tokens,
                    int n_heads, float scale, void* out, void* ws, size_t ws_bytes, int dtype, void* stream) {
  if (!known_dtype(dtype)) return CATS_ERR_DTYPE;
  int s = check_cache(cache);
  if (s) return s;
  if ((s = check_tokens(cache, cu, n_tokens, n_heads))) return s;
  if (layer < 0 || layer >= cache->n_layers || !(fabsf(scale) < INFINITY)) return CATS_ERR_RANGE;
  if (!units_fit(cache, n_tokens, n_heads)) return CATS_ERR_RANGE;
  if (!q || !out || !ws) return CATS_ERR_NULL;
  if (q_ld < (long long)n_heads * cache->head_dim) return CATS_ERR_RANGE;
  if (!aligned16(q) || (q_ld * esize(dtype)) % 16 || !aligned16(out) || !aligned16(ws)) return CATS_ERR_ALIGN;
  if (ws_bytes < cats_kv8_attend_bytes(cache, n_tokens, n_heads)) return CATS_ERR_WORKSPACE;
  cudaStream_t st = (cudaStream_t)stream;
  cudaError_t e;
  if (dtype == CATS_F32) e = attend<float>(*cache, layer, q, q_ld, cu, n_tokens, n_heads, scale, out, ws, st);
  else if (dtype == CATS_F16) e = attend<__half>(*cache, layer, q, q_ld, cu, n_tokens, n_heads, scale, out, ws, st);
  else e = attend<__nv_bfloat16>(*cache, layer, q, q_ld, cu, n_tokens, n_heads, scale, out, ws, st);
  return launch_status(e);
}

size_t cats_kv8_reorder_bytes(const cats_kv8* cache) {
  return cache && cache->n_seqs > 0 ? sizeof(KvCopy) * ((size_t)cache->n_seqs + 1) : 0;
}

int cats_kv8_reorder(const cats_kv8* cache, const int* parents, void* ws, size_t ws_bytes, void* stream) {
  int s = check_cache(cache);
  if (s) return s;
  if (!parents || !ws) return CATS_ERR_NULL;
  if (!aligned16(ws)) return CATS_ERR_ALIGN;
  if (ws_bytes < cats_kv8_reorder_bytes(cache)) return CATS_ERR_WORKSPACE;
  cudaStream_t st = (cudaStream_t)stream;
  int* n_copies = (int*)ws;
  KvCopy* copies = (KvCopy*)ws + 1;
  // a strip holds `width` columns of every row (at most 48 KB with the two arrays beside it); a table
  // that fits one strip of 4096 entries is dealt with by the CTA that hands out the pages
  const int n = cache->n_seqs;
  const bool small = (long long)n * cache->max_pages <= 4096;
  cudaError_t e = cudaSuccess;
  if (!small) {
    int width = 32;
    while (width > 8 && (size_t)n * (width + 2) * 4 > 48 * 1024) width >>= 1;
    e = launch(k_kv8_reorder_table, dim3((cache->max_pages + width - 1) / width), dim3(256),
               (size_t)n * (width + 2) * sizeof(int), st, *cache, parents, width);
  }
  if (e == cudaSuccess)
    e = launch(k_kv8_reorder_plan, dim3(1), dim3(kPlanThreads),
               small ? (size_t)n * (cache->max_pages + 2) * sizeof(int) : 0, st, *cache, parents, n_copies, copies,
               small ? 1 : 0);
  if (e == cudaSuccess)
    e = launch(k_kv8_copy, dim3(dev_info().sms * 4), dim3(256), 0, st, *cache, (const int*)n_copies,
               (const KvCopy*)copies);
  return launch_status(e);
}

size_t cats_kv8_compact_bytes(const cats_kv8* cache) {
  return cache && cache->n_pages > 0 ? (sizeof(KvCopy) + sizeof(int)) * (size_t)cache->n_pages + sizeof(KvCopy) : 0;
}

int cats_kv8_compact(const cats_kv8* cache, int* n_live, void* ws, size_t ws_bytes, void* stream) {
  int s = check_cache(cache);
  if (s) return s;
  if (!n_live || !ws) return CATS_ERR_NULL;
  if (!aligned16(ws)) return CATS_ERR_ALIGN;
  if (ws_bytes < cats_kv8_compact_bytes(cache)) return CATS_ERR_WORKSPACE;
  cudaStream_t st = (cudaStream_t)stream;
  int* n_moves = (int*)ws;
  KvCopy* moves = (KvCopy*)ws + 1;
  int* remap = (int*)(moves + cache->n_pages);
  cudaError_t e = launch(k_kv8_compact_plan, dim3(1), dim3(kPlanThreads), 0, st, *cache, n_live, n_moves, moves, remap);
  if (e == cudaSuccess)
    e = launch(k_kv8_compact_move, dim3(dev_info().sms * 4), dim3(256), 0, st, *cache, (const int*)n_moves,
               (const KvCopy*)moves, (const int*)remap);
  return launch_status(e);
}

size_t cats_beam_select_bytes(int n, int beams, int vocab, int k) {
  if (n < 1 || beams < 1 || vocab < 1 || k < 1) return 0;
  const size_t parts = (size_t)n * beams * beam_splits((long long)n * beams, beams, vocab, k);
  return parts * (sizeof(BeamPart) + k * sizeof(unsigned long long));
}

int cats_beam_select(const void* logits, long long ld, const float* scores, const uint8_t* done, int n, int beams,
                     int vocab, int k, int eos, int dtype, float* out_scores, int* out_rows, long long* out_tokens,
                     uint8_t* out_done, void* ws, size_t ws_bytes, void* stream) {
  if (!known_dtype(dtype)) return CATS_ERR_DTYPE;
  if (n < 1 || beams < 1 || beams > kBeamMaxBeams || vocab < 1 || vocab > (1 << 30) || k < 1 ||
      k > kBeamMaxK || ld < vocab)
    return CATS_ERR_RANGE;
  if ((long long)n * beams > 65535 || (long long)beams * vocab < k) return CATS_ERR_RANGE;
  if (done && (eos < 0 || eos >= vocab)) return CATS_ERR_RANGE;
  if (!logits || !scores || !out_scores || !out_rows || !out_tokens || !ws) return CATS_ERR_NULL;
  if (reinterpret_cast<uintptr_t>(logits) % esize(dtype) || !aligned16(ws)) return CATS_ERR_ALIGN;
  if (ws_bytes < cats_beam_select_bytes(n, beams, vocab, k)) return CATS_ERR_WORKSPACE;
  cudaStream_t st = (cudaStream_t)stream;
  BeamArgs A;
  const int rows = n * beams;
  A.logits = logits; A.ld = ld; A.scores = scores; A.done = done;
  A.n = n; A.beams = beams; A.vocab = vocab; A.k = k; A.eos = eos;
  A.splits = beam_splits(rows, beams, vocab, k);
  A.keys = (unsigned long long*)ws;
  A.parts = (BeamPart*)(A.keys + (size_t)rows * A.splits * k);
  A.out_scores = out_scores; A.out_rows = out_rows; A.out_tokens = out_tokens; A.out_done = out_done;
  cudaError_t e;
  const dim3 grid(A.splits, rows), block(kBeamThreads);
  if (dtype == CATS_F32) e = launch(k_beam_rows<float>, grid, block, 0, st, A);
  else if (dtype == CATS_F16) e = launch(k_beam_rows<__half>, grid, block, 0, st, A);
  else e = launch(k_beam_rows<__nv_bfloat16>, grid, block, 0, st, A);
  if (e != cudaSuccess) return launch_status(e);
  const size_t smem = (size_t)beams * k * 8 + (size_t)beams * A.splits * k * 8 + (size_t)beams * 8 + (size_t)beams * k * 8;
  return launch_status(launch(k_beam_join, dim3(n), block, smem, st, A));
}

}  // extern "C"
