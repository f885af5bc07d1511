// C ABI of the paged cache and of rotary positions (include/adaptq_paged.h).
#include "../../include/adaptq_paged.h"
#include "../../include/adaptq.h"
#include "host_common.h"
#include "paged_attend_host.h"
#include "paged_rows.cuh"
#include "rotary.cuh"

#include <algorithm>
#include <cmath>

using namespace aq;

namespace {

struct DeviceScope { // the call's device is current while this lives
  int prev = -1;
  bool ok = true;
  explicit DeviceScope(int dev) {
    int now = -1;
    if (cudaGetDevice(&now) != cudaSuccess) { cudaGetLastError(); ok = false; return; }
    if (now != dev) {
      if (cudaSetDevice(dev) != cudaSuccess) { cudaGetLastError(); ok = false; return; }
      prev = now;
    }
  }
  ~DeviceScope() { if (prev >= 0) cudaSetDevice(prev); }
};

bool fail(const char *fn, const char *what) { aq_set_error("%s: %s", fn, what); return false; }

bool aligned(const void *p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }
// Addresses that the kernels could not read or write element by element.
template <typename... T> bool misaligned(size_t n, const T *...p) { return ((reinterpret_cast<uintptr_t>(p) | ...) & (n - 1)) != 0; }
int size_of(int type) { return type == TYPE_F32 ? 4 : 2; }
int padded_of(int dim) { int p = 64; while (p < dim) p <<= 1; return p; }

// Rows that may be moved 16 bytes at a time.
bool vector_rows(const void *p, int64_t stride0, int64_t stride1, int dim, int type) {
  const int per = 16 / size_of(type);
  return aligned(p, 16) && stride0 % per == 0 && stride1 % per == 0 && dim % 8 == 0;
}

bool check_cache(const char *fn, const adaptq_paged_t *c, PagedView &v) {
  if (!c) return fail(fn, "null cache");
  if (!c->k_pages || !c->v_pages || !c->k_scales || !c->v_scales || !c->signs || !c->status) return fail(fn, "null pointer in the cache");
  if (c->dim < 33 || c->dim > 256) return fail(fn, "head dimensions from 33 to 256 are supported");
  if (c->k_bits < 2 || c->k_bits > 4 || c->v_bits < 2 || c->v_bits > 4) return fail(fn, "k_bits and v_bits must be 2, 3 or 4");
  if (c->page_size != 16 && c->page_size != 32 && c->page_size != 64 && c->page_size != 128 && c->page_size != 256)
    return fail(fn, "page_size must be 16, 32, 64, 128 or 256");
  if (c->n_pages <= 0 || c->n_pages > 0x7fffffff || c->n_kv_heads <= 0 || c->n_kv_heads > 65535) return fail(fn, "invalid number of pages or heads");
  if (!aligned(c->k_pages, 16) || !aligned(c->v_pages, 16) || !aligned(c->k_scales, 16) || !aligned(c->v_scales, 16))
    return fail(fn, "pages and scales must be 16-byte aligned");
  if (misaligned(4, c->signs, c->status)) return fail(fn, "a pointer in the cache is not aligned to its elements");
  int shift = 4;
  while ((1 << shift) < c->page_size) ++shift;
  v = PagedView{static_cast<uint8_t *>(c->k_pages), static_cast<uint8_t *>(c->v_pages), c->k_scales, c->v_scales, c->signs, c->status,
                c->n_pages, c->n_kv_heads, c->page_size, shift, c->dim};
  return true;
}

bool check_rotary(const char *fn, const adaptq_rotary_t *r, int dim, RotaryView &v) {
  v = RotaryView{nullptr, 1.f, 0, 0};
  if (!r) return true;
  if (!r->turns || misaligned(8, r->turns)) return fail(fn, "null or unaligned rotary frequencies");
  if (r->dim < 2 || r->dim % 2 || r->dim > dim) return fail(fn, "the rotary dimension must be even and at most the head dimension");
  v = RotaryView{reinterpret_cast<const unsigned long long *>(r->turns), r->factor, r->dim, r->interleaved != 0};
  return true;
}

bool check_type(const char *fn, int type) { return type >= 0 && type <= 2 ? true : fail(fn, "type must be 0 (float32), 1 (float16) or 2 (bfloat16)"); }

bool launched(const char *fn) { return aq_launched(fn); }

template <int P, int KB, int VB> void launch_rows(const RowsLaunch &a, bool append, int sms, cudaStream_t s) {
  if (append) {
    constexpr int ROWS = rows_per_warp<P>, WARPS = ROWS_THREADS / 32;
    RowsLaunch b = a;
    b.turn_tokens = std::min(ROWS, (ROWS + a.c.heads - 2) / a.c.heads + 1);
    // several tokens a warp, since what it sets up is paid once, and three rounds of warps (24 an SM, keys and values), for
    // keys take longer than values
    b.job_tokens = (int)std::max(1ll, std::min(32ll, 2 * a.n_tokens / (3 * 24 * sms)));
    const unsigned blocks = (unsigned)((a.n_tokens + b.job_tokens * WARPS - 1) / (b.job_tokens * WARPS));
    paged_append_kernel<P, KB, VB><<<dim3(blocks, 2), ROWS_THREADS, (size_t)WARPS * b.turn_tokens * a.r.dim * sizeof(float), s>>>(b);
  } else {
    RowsLaunch b = a;
    // blocks of 64 tokens (keys and values), smaller ones where those would not make four an SM
    for (b.block_tokens = READ_TOKENS; b.block_tokens > 16 && 2 * ((a.n_tokens + b.block_tokens - 1) / b.block_tokens) < 4 * sms;) b.block_tokens /= 2;
    const unsigned tiles = (unsigned)((a.n_tokens + b.block_tokens - 1) / b.block_tokens);
    const long long items = (long long)(b.block_tokens / 16) * a.c.heads;
    const unsigned shares = (unsigned)std::max(1ll, std::min((items + READ_WARPS - 1) / READ_WARPS, 4ll * sms / (2 * tiles)));
    paged_read_kernel<P, KB, VB><<<dim3(tiles, 2, shares), READ_WARPS * 32, 0, s>>>(b);
  }
}
template <int P, int KB> void launch_rows_v(const RowsLaunch &a, int vb, bool append, int sms, cudaStream_t s) {
  if (vb == 2) launch_rows<P, KB, 2>(a, append, sms, s);
  else if (vb == 3) launch_rows<P, KB, 3>(a, append, sms, s);
  else launch_rows<P, KB, 4>(a, append, sms, s);
}
template <int P> void launch_rows_k(const RowsLaunch &a, int kb, int vb, bool append, int sms, cudaStream_t s) {
  if (kb == 2) launch_rows_v<P, 2>(a, vb, append, sms, s);
  else if (kb == 3) launch_rows_v<P, 3>(a, vb, append, sms, s);
  else launch_rows_v<P, 4>(a, vb, append, sms, s);
}

int rows_call(const char *fn, bool append, const adaptq_paged_t *cache, void *k, int64_t k_token, int64_t k_head, void *v,
              int64_t v_token, int64_t v_head, int type, const int *table, int64_t table_stride, int table_width,
              const int *starts, int start_bias, const int *cu_tokens, int n_seqs, int64_t n_tokens,
              const adaptq_rotary_t *rotary, void *stream) {
  aq_clear_error();
  RowsLaunch a{};
  if (!check_cache(fn, cache, a.c) || !check_rotary(fn, rotary, cache->dim, a.r) || !check_type(fn, type)) return -1;
  if (n_seqs < 0 || n_tokens < 0 || table_width < 0) return fail(fn, "negative size"), -1;
  if (n_seqs == 0 || n_tokens == 0) return 0;
  if (!k || !v || !table || !starts) return fail(fn, "null pointer"), -1;
  if (misaligned(size_of(type), k, v) || misaligned(4, table, starts, cu_tokens)) return fail(fn, "a pointer is not aligned to its elements"), -1;
  const int P = padded_of(cache->dim);
  if (cu_tokens && n_seqs > 1 << 30) return fail(fn, "too many sequences for one call"), -1; // owner_of looks up to n_seqs + 32 ahead, in 32 bits
  if (n_tokens > (1ll << 31) / cache->n_kv_heads) return fail(fn, "too many tokens for one call"), -1;
  a.table = TableView{table, table_stride, table_width};
  a.starts = starts; a.start_bias = start_bias; a.cu = cu_tokens; a.n_seqs = n_seqs; a.n_tokens = n_tokens;
  a.k = k; a.k_token = k_token; a.k_head = k_head; a.v = v; a.v_token = v_token; a.v_head = v_head; a.type = type;
  a.k_vec = vector_rows(k, k_token, k_head, cache->dim, type);
  a.v_vec = vector_rows(v, v_token, v_head, cache->dim, type);
  const int per = 32 / size_of(type); // elements of a 32-byte store
  const auto wide = [&](const void *p, int64_t s0, int64_t s1) { return aligned(p, 32) && s0 % per == 0 && s1 % per == 0 && cache->dim % 16 == 0; };
  if (!append && a.k_vec && wide(k, k_token, k_head)) a.k_vec = 2;
  if (!append && a.v_vec && wide(v, v_token, v_head)) a.v_vec = 2;
  DeviceScope dev(cache->device);
  if (!dev.ok) return fail(fn, "no usable CUDA device (this library has no CPU path)"), -1;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int sms = aq_sm_count(cache->device);
  if (P == 64) launch_rows_k<64>(a, cache->k_bits, cache->v_bits, append, sms, s);
  else if (P == 128) launch_rows_k<128>(a, cache->k_bits, cache->v_bits, append, sms, s);
  else launch_rows_k<256>(a, cache->k_bits, cache->v_bits, append, sms, s);
  return launched(fn) ? 0 : -1;
}

// The kernels of one pair of bit widths are a translation unit of their own (paged_attend.cu).
typedef bool (*attend_unit_t)(const AttendCall &);
const attend_unit_t attend_units[3][3] = {{aq_attend_2_2, aq_attend_2_3, aq_attend_2_4},
                                          {aq_attend_3_2, aq_attend_3_3, aq_attend_3_4},
                                          {aq_attend_4_2, aq_attend_4_3, aq_attend_4_4}};

// float32: two parts throughout.  float16: queries and weights in two parts, four queries a pass, so that what is lost
// on the way stays below the output's own rounding (one part: 4.3e-4 of the output's norm instead of 2.1e-4, and 32.7
// us instead of 33.6 for 33 x 14 heads of one query; above four queries the further passes cost their share).  bfloat16: one part, eight queries a pass; its output rounding is eight times coarser.
int attend_mode(int type) { return type == TYPE_F32 ? ATTEND_EXACT : type == TYPE_F16 ? ATTEND_SPLIT : ATTEND_EIGHT; }

// One exchange, so that a bit set by a call on another stream is either taken or left for the next time.
__global__ void take_status_kernel(int *status, int *taken) {
  int bits = atomicExch(status, 0);
#ifdef ADAPTQ_CHECKED
  bits |= atomicExch(&rotary_status, 0);
#endif
  *taken = bits;
}

} // namespace

extern "C" {

int adaptq_rotary_apply(const adaptq_rotary_t *rotary, const void *x, int64_t x_token_stride, int64_t x_head_stride, void *y,
                        int64_t y_token_stride, int64_t y_head_stride, int type, const void *positions, int positions_64,
                        int64_t n_tokens, int n_heads, int dim, int inverse, int device, void *stream) {
  const char *fn = "adaptq_rotary_apply";
  aq_clear_error();
  RotaryLaunch a{};
  if (!rotary) return fail(fn, "null rotary"), -1;
  if (dim <= 0 || dim > 65536 || n_heads < 0 || n_heads > 65535 || n_tokens < 0) return fail(fn, "invalid sizes"), -1;
  if (!check_rotary(fn, rotary, dim, a.r) || !check_type(fn, type)) return -1;
  if (n_tokens == 0 || n_heads == 0) return 0;
  if (!x || !y || !positions) return fail(fn, "null pointer"), -1;
  if (misaligned(size_of(type), x, y) || misaligned(positions_64 ? 8 : 4, positions)) return fail(fn, "a pointer is not aligned to its elements"), -1;
  const int half = rotary->dim / 2;
  if (half * (int)sizeof(float2) > 32768) return fail(fn, "rotary dimensions above 8192 are not supported"), -1;
  a.x = x; a.y = y; a.positions = positions; a.positions_64 = positions_64 != 0;
  a.x_token = x_token_stride; a.x_head = x_head_stride; a.y_token = y_token_stride; a.y_head = y_head_stride;
  a.n_tokens = n_tokens; a.heads = n_heads; a.dim = dim; a.type = type; a.inverse = inverse != 0;
  a.vec = vector_rows(x, x_token_stride, x_head_stride, dim, type) && vector_rows(y, y_token_stride, y_head_stride, dim, type) &&
          (rotary->interleaved || half % 8 == 0);
  DeviceScope dev(device);
  if (!dev.ok) return fail(fn, "no usable CUDA device (this library has no CPU path)"), -1;
  // Several tokens a block where there are enough of them: all its threads form turns (16384 tokens x 32 heads x 128,
  // bf16: 46.4 us with four, 50.1 with one; few tokens would leave SMs idle).
  a.tokens_per_block = 1;
  while (a.tokens_per_block < 4 && a.tokens_per_block * half < ROTARY_THREADS && n_tokens / (2 * a.tokens_per_block) >= 8 * aq_sm_count(device)) a.tokens_per_block *= 2;
  const long long blocks = (n_tokens + a.tokens_per_block - 1) / a.tokens_per_block;
  if (blocks > 0x7fffffff) return fail(fn, "too many tokens for one call"), -1;
  a.heads_per_block = std::min(n_heads, (1 << 28) / dim); // all heads, as long as they are below 2^28 coordinates
  const unsigned head_blocks = (unsigned)((n_heads + a.heads_per_block - 1) / a.heads_per_block);
  rotary_kernel<<<dim3((unsigned)blocks, head_blocks), ROTARY_THREADS, a.tokens_per_block * half * sizeof(float2), static_cast<cudaStream_t>(stream)>>>(a);
  return launched(fn) ? 0 : -1;
}

int adaptq_paged_signs(uint64_t seed, int n_heads, int dim, uint32_t *words) {
  const char *fn = "adaptq_paged_signs";
  aq_clear_error();
  if (n_heads <= 0 || dim < 33 || dim > 256 || !words) return fail(fn, "invalid parameters"), -1;
  const int P = padded_of(dim);
  for (int h = 0; h < n_heads; ++h) // head seeds as adaptq_mha_create gives them (upstream core/adaptq_c_api.cpp:160)
    aq_sign_words(seed ^ ((uint64_t)h * 0xDEADBEEFCAFEULL), P, words + (size_t)h * (P / 32), P / 32);
  return 0;
}

int adaptq_paged_take_status(const adaptq_paged_t *cache, int *taken, void *stream) {
  const char *fn = "adaptq_paged_take_status";
  aq_clear_error();
  PagedView v;
  if (!check_cache(fn, cache, v)) return -1;
  if (!taken) return fail(fn, "null pointer"), -1;
  if (misaligned(4, taken)) return fail(fn, "a pointer is not aligned to its elements"), -1;
  DeviceScope dev(cache->device);
  if (!dev.ok) return fail(fn, "no usable CUDA device (this library has no CPU path)"), -1;
  take_status_kernel<<<1, 1, 0, static_cast<cudaStream_t>(stream)>>>(v.status, taken);
  return launched(fn) ? 0 : -1;
}

int adaptq_paged_append(const adaptq_paged_t *cache, const void *k, int64_t k_token_stride, int64_t k_head_stride, const void *v,
                        int64_t v_token_stride, int64_t v_head_stride, int type, const int *table, int64_t table_stride,
                        int table_width, const int *starts, int start_bias, const int *cu_tokens, int n_seqs,
                        int64_t n_tokens, const adaptq_rotary_t *rotary, void *stream) {
  return rows_call("adaptq_paged_append", true, cache, const_cast<void *>(k), k_token_stride, k_head_stride, const_cast<void *>(v),
                   v_token_stride, v_head_stride, type, table, table_stride, table_width, starts, start_bias, cu_tokens, n_seqs,
                   n_tokens, rotary, stream);
}

int adaptq_paged_read(const adaptq_paged_t *cache, void *k_out, int64_t k_token_stride, int64_t k_head_stride, void *v_out,
                      int64_t v_token_stride, int64_t v_head_stride, int type, const int *table, int64_t table_stride,
                      int table_width, const int *starts, const int *cu_tokens, int n_seqs, int64_t n_tokens, void *stream) {
  return rows_call("adaptq_paged_read", false, cache, k_out, k_token_stride, k_head_stride, v_out, v_token_stride, v_head_stride,
                   type, table, table_stride, table_width, starts, 0, cu_tokens, n_seqs, n_tokens, nullptr, stream);
}

size_t adaptq_paged_attend_workspace(const adaptq_paged_t *cache, int n_seqs, int n_q_heads, int type) {
  if (!cache || n_seqs < 0 || cache->dim < 33 || cache->dim > 256 || cache->k_bits < 2 || cache->k_bits > 4 || cache->v_bits < 2 || cache->v_bits > 4 ||
      cache->n_kv_heads <= 0 || n_q_heads <= 0 || n_q_heads % cache->n_kv_heads)
    return 0;
  size_t bytes = 0;
  AttendLaunch a{};
  a.n_seqs = n_seqs; a.group = n_q_heads / cache->n_kv_heads; a.c.heads = cache->n_kv_heads;
  attend_units[cache->k_bits - 2][cache->v_bits - 2]({"adaptq_paged_attend_workspace", &a, padded_of(cache->dim), attend_mode(type), cache->device,
                                                      nullptr, nullptr, &bytes});
  return bytes;
}

int adaptq_paged_attend(const adaptq_paged_t *cache, const void *q, int64_t q_seq_stride, int64_t q_head_stride, void *out,
                        int64_t out_seq_stride, int64_t out_head_stride, int type, const int *table, int64_t table_stride,
                        int table_width, const int *lengths, int n_seqs, int n_q_heads, float scale,
                        const adaptq_rotary_t *rotary, void *workspace, size_t workspace_bytes, void *stream) {
  const char *fn = "adaptq_paged_attend";
  aq_clear_error();
  AttendLaunch a{};
  if (!check_cache(fn, cache, a.c) || !check_rotary(fn, rotary, cache->dim, a.r) || !check_type(fn, type)) return -1;
  if (n_seqs < 0 || table_width < 0) return fail(fn, "negative size"), -1;
  if (n_q_heads <= 0 || n_q_heads % cache->n_kv_heads) return fail(fn, "the number of query heads must be a multiple of that of KV heads"), -1;
  if (!(scale > 0.f) || !std::isfinite(scale)) return fail(fn, "scale must be positive and finite"), -1;
  if (n_seqs == 0) return 0;
  if (!q || !out || !table || !lengths) return fail(fn, "null pointer"), -1;
  if (misaligned(size_of(type), q, out) || misaligned(4, table, lengths)) return fail(fn, "a pointer is not aligned to its elements"), -1;
  if (n_q_heads > 1 << 20) return fail(fn, "at most 1048576 query heads are supported"), -1;
  if (n_q_heads / cache->n_kv_heads > 65536) return fail(fn, "at most 65536 queries per KV head are supported"), -1;
  if ((long long)n_seqs * n_q_heads > 0x3fffffff) return fail(fn, "too many sequences for one call"), -1;
  a.table = TableView{table, table_stride, table_width};
  a.lengths = lengths; a.q = q; a.out = out; a.q_seq = q_seq_stride; a.q_head = q_head_stride;
  a.out_seq = out_seq_stride; a.out_head = out_head_stride;
  a.n_seqs = n_seqs; a.group = n_q_heads / cache->n_kv_heads; a.type = type; a.scale = scale;
  a.out_vec = vector_rows(out, out_seq_stride, out_head_stride, cache->dim, type);
  if (!workspace || !aligned(workspace, 16) || workspace_bytes < adaptq_paged_attend_workspace(cache, n_seqs, n_q_heads, type))
    return fail(fn, "the workspace is too small or not 16-byte aligned"), -1;
  DeviceScope dev(cache->device);
  if (!dev.ok) return fail(fn, "no usable CUDA device (this library has no CPU path)"), -1;
  const AttendCall call{fn, &a, padded_of(cache->dim), attend_mode(type), cache->device, workspace, static_cast<cudaStream_t>(stream), nullptr};
  return attend_units[cache->k_bits - 2][cache->v_bits - 2](call) ? 0 : -1;
}

} // extern "C"
