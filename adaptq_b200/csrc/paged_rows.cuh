// Rows into the pages and out of them.
//
// Append: a row of P coordinates is held by P/32 lanes, 32 consecutive ones each, two in a
// register pair (the float2 instructions round each half like the scalar ones): five of the
// log2 P butterfly stages stay inside a lane, the others are shuffles, and a lane's codes are
// a whole number of words.  Bound by instructions: 117 a row of 128 coordinates (transform 22,
// quantiser 24 of those of a 4-bit key), 2.6 a clock; four prompts of 3277 to 8192
// tokens x 8 heads in bf16 at K4/V2 take 61 us, 19 at the copy rate.
// Read-back: see paged_read_kernel.
#pragma once
#include "paged.cuh"

namespace aq {

constexpr int ROWS_THREADS = 256;
template <int P> constexpr int rows_per_warp = 32 / (P / 32);

struct RowsLaunch {
  PagedView c;
  RotaryView r;
  TableView table;
  const int *starts, *cu;
  int start_bias, n_seqs;
  long long n_tokens;
  // the model's rows: keys and values (read by the append, written by the read-back)
  void *k, *v;
  long long k_token, k_head, v_token, v_head;
  int job_tokens;         // append: tokens of a warp, at most 32
  int turn_tokens;        // append: tokens of a warp's rows in hand at most
  int block_tokens;       // read-back: tokens of a block
  int type, k_vec, v_vec; // 0; 1: rows 16-byte aligned, dim a multiple of 8; 2: 32-byte aligned, a multiple of 16 as well
};

struct TokenPlace { int page, off; long long pos; }; // page < 0: nowhere

// Where token t + lane goes to, or is read from, for lanes below `count` (the whole warp calls).
__device__ __forceinline__ TokenPlace find_place(const RowsLaunch &a, long long t, int lane, int count) {
  const int b = a.cu ? owner_of(a.cu, a.n_seqs, t, lane, count) : (lane < count && t + lane < a.n_seqs ? (int)t + lane : -1);
  TokenPlace p{-1, 0, 0};
  if (b >= 0 && !(a.start_bias < 0 && a.starts[b] == 0)) { // a decode step leaves empty sequences out
    p.pos = (long long)a.starts[b] + a.start_bias + (a.cu ? t + lane - a.cu[b] : 0);
    if (!find_slot(a.c, a.table.entries + b * a.table.stride, a.table.width, p.pos, p.page, p.off)) p.page = -1;
  }
  return p;
}

__device__ __forceinline__ float2 add2(float2 a, float2 b) { return __fadd2_rn(a, b); }
__device__ __forceinline__ float2 sub2(float2 a, float2 b) { return __ffma2_rn(b, make_float2(-1.f, -1.f), a); }

// Walsh-Hadamard butterflies over a row: 32 values a lane, P/32 lanes.
template <int P> __device__ __forceinline__ void row_butterflies(float2 (&x)[16], int lane) {
#pragma unroll
  for (int i = 0; i < 16; ++i) x[i] = make_float2(x[i].x + x[i].y, x[i].x - x[i].y);
#pragma unroll
  for (int len = 1; len < 16; len <<= 1) {
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (!(i & len)) {
        const float2 a = x[i], b = x[i + len];
        x[i] = add2(a, b);
        x[i + len] = sub2(a, b);
      }
  }
#pragma unroll
  for (int m = 1; m < P / 32; m <<= 1) {
    const float s = (lane & m) ? -1.f : 1.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const float2 o = make_float2(__shfl_xor_sync(0xffffffffu, x[i].x, m), __shfl_xor_sync(0xffffffffu, x[i].y, m));
      x[i] = __ffma2_rn(x[i], make_float2(s, s), o);
    }
  }
}

// Quantisers: a code is the count of thresholds at or below the coordinate.  2 bits: evenly spaced thresholds, one
// rounding.  3 and 4 bits: the 128 buckets of a quarter from -16 on hold at most one threshold each, so a code is the
// count of thresholds at or below the bucket's start and one comparison.  16 copies of the table, entry by entry, keep the
// half-warps of a 64-bit read apart.  A coordinate is at most sqrt(P) = 16 in size.
constexpr int BUCKETS = 128, BUCKET_COPIES = 16;
template <int BITS> __device__ __forceinline__ void fill_buckets(uint2 *table, int tid) {
  if (tid < BUCKETS) {
    const float start = (tid - 64) * 0.25f;
    float threshold = INFINITY;
    uint32_t below = 0;
    for (int i = (1 << BITS) - 2; i >= 0; --i) {
      const float t = c_thr[BITS - 2][i];
      if (t <= start) ++below;
      else if (t < start + 0.25f) threshold = t;
    }
    for (int i = 0; i < BUCKET_COPIES; ++i) table[tid * BUCKET_COPIES + i] = make_uint2(__float_as_uint(threshold), below);
  }
}
// word = word << BITS | code of u
template <int P, int BITS> __device__ __forceinline__ void push_code(uint32_t &word, float u, const uint2 *table, uint32_t copy /* 8 * lane's copy */) {
  if constexpr (BITS == 2) {
    // thresholds -T, 0, T: the code is floor(u / T) + 2 within 0 .. 3.  T * (1 / T) rounds to less than one, which
    // is right at -T (a threshold counts from itself on) and would be wrong at T: that one is a comparison.
    constexpr float T = (0.4528f + 1.5104f) * 0.5f;
    const float v = u >= T ? 1.5f * T : fmaxf(u, -1.5f * T);
    word = word * 4 + (__float_as_uint(__fmaf_rd(v, 1.f / T, 8388608.f + 2.f)) & 3u);
  } else {
    if constexpr (P == 256) u = fminf(fmaxf(u, -16.f), 15.75f);
    // 4 u + 64 in units of 2^-7, rounded down: the bucket lies where a byte offset into the table wants it (any for NaN)
    const uint32_t at = (__float_as_uint(__fmaf_rd(u, 4.f, 65536.f + 64.f)) & ((BUCKETS - 1) << 7)) | copy;
    const uint2 e = *reinterpret_cast<const uint2 *>(reinterpret_cast<const uint8_t *>(table) + at);
    word = word * (1u << BITS) + e.y;
    if (u >= __uint_as_float(e.x)) ++word;
  }
}

// 32 coordinates -> BITS words of codes, most significant bits of each byte first.
template <int P, int BITS> __device__ __forceinline__ void pack_codes(const float2 (&u)[16], const uint2 *table, uint32_t copy, uint32_t (&w)[BITS]) {
  if constexpr (BITS == 3) {
    uint32_t r[4];
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      uint32_t v = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        push_code<P, BITS>(v, u[4 * g + i].x, table, copy);
        push_code<P, BITS>(v, u[4 * g + i].y, table, copy);
      }
      r[g] = __byte_perm(v, 0, 0x4012);
    }
    w[0] = r[0] | r[1] << 24;
    w[1] = r[1] >> 8 | r[2] << 16;
    w[2] = r[2] >> 16 | r[3] << 8;
  } else {
    constexpr int PAIRS = 16 / BITS;
#pragma unroll
    for (int g = 0; g < BITS; ++g) {
      uint32_t v = 0;
#pragma unroll
      for (int i = 0; i < PAIRS; ++i) {
        push_code<P, BITS>(v, u[PAIRS * g + i].x, table, copy);
        push_code<P, BITS>(v, u[PAIRS * g + i].y, table, copy);
      }
      w[g] = __byte_perm(v, 0, 0x0123); // the first code is on top
    }
  }
}

template <int BITS> __device__ __forceinline__ void store_words(uint8_t *p, const uint32_t (&w)[BITS]) {
  if constexpr (BITS == 4) *reinterpret_cast<uint4 *>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  else if constexpr (BITS == 2) *reinterpret_cast<uint2 *>(p) = make_uint2(w[0], w[1]);
  else {
#pragma unroll
    for (int i = 0; i < 3; ++i) reinterpret_cast<uint32_t *>(p)[i] = w[i];
  }
}
// One side of the append.  A warp takes 32 / (P/32) rows at a time, token by token, and meets no barrier; the turns of its
// tokens (usually one: the heads of a token are neighbours) go through its own shared memory, cosines and sines apart so
// that they are read as pairs.
template <int P, int BITS>
__device__ __forceinline__ void append_rows(const RowsLaunch &a, const void *src, long long src_token, long long src_head,
                                            bool vec, uint8_t *pages, float *scales, bool rotate, float *turns, const uint2 *table) {
  constexpr int LANES = P / 32, ROWS = rows_per_warp<P>;
  const int heads = a.c.heads, dim = a.c.dim, half = a.r.dim >> 1;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, part = lane % LANES, d0 = part * 32;
  const uint32_t copy = (lane & (BUCKET_COPIES - 1)) * 8;
  // a job: the rows of a.job_tokens tokens; lane i finds the place of the i-th
  const long long t0 = ((long long)blockIdx.x * (ROWS_THREADS / 32) + warp) * a.job_tokens;
  if (t0 >= a.n_tokens) return;
  const int tokens = (int)min((long long)a.job_tokens, a.n_tokens - t0), n_rows = tokens * heads;
  const TokenPlace mine = find_place(a, t0, lane, tokens);
  for (int r0 = 0; r0 < n_rows; r0 += ROWS) {
    const int row = min(r0 + lane / LANES, n_rows - 1), dt = row / heads, h = row - dt * heads;
    const int first_token = r0 / heads, nt = min(r0 + ROWS - 1, n_rows - 1) / heads - first_token + 1;
    const long long at = (t0 + dt) * src_token + h * src_head;
    const bool row_exists = PAGED_CHECK(a.c.status, row >= 0 && t0 + dt < a.n_tokens && h < heads && first_token + nt <= tokens && d0 < P);

    float2 x[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i] = make_float2(0.f, 0.f);
    if (vec) with_type(a.type, [&](auto type) {
#pragma unroll
      for (int i = 0; i < 32; i += 8)
        if (row_exists && d0 + i < dim) {
          float v[8];
          load_eight<decltype(type)::value>(src, at + d0 + i, v);
#pragma unroll
          for (int j = 0; j < 4; ++j) x[i / 2 + j] = make_float2(v[2 * j], v[2 * j + 1]);
        }
    }); else {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        if (row_exists && d0 + 2 * i < dim) x[i].x = load_one(src, at + d0 + 2 * i, a.type);
        if (row_exists && d0 + 2 * i + 1 < dim) x[i].y = load_one(src, at + d0 + 2 * i + 1, a.type);
      }
    }
    const uint32_t signs = a.c.signs[h * LANES + part];
    const int page = __shfl_sync(0xffffffffu, mine.page, dt), off = __shfl_sync(0xffffffffu, mine.off, dt);

    if (rotate) {
      __syncwarp();
      for (int i = 0; i < nt; ++i) {
        const long long pos = __shfl_sync(0xffffffffu, mine.pos, first_token + i);
        for (int pair = lane; pair < half; pair += 32) {
          const float2 k = rotary_turn(a.r, pair, pos);
          if (!PAGED_CHECK(a.c.status, i < a.turn_tokens)) continue;
          turns[i * 2 * half + pair] = k.x;
          turns[i * 2 * half + half + pair] = k.y;
        }
      }
      __syncwarp();
      const float *cs = turns + (dt - first_token) * 2 * half, *sn = cs + half;
      if (a.r.interleaved) {
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (d0 + 2 * i < a.r.dim) {
            const float2 k = make_float2(cs[(d0 >> 1) + i], sn[(d0 >> 1) + i]);
            x[i] = make_float2(rotary_first(x[i].x, x[i].y, k), rotary_second(x[i].y, x[i].x, k));
          }
      } else if ((half & 31) == 0) { // the partners of a lane's 32 coordinates are another lane's 32
        const int m = half >> 5;
        const bool first = part < m, in = part < 2 * m;
        const int from = lane + (first ? m : in ? -m : 0);
        const float sign = first ? -1.f : 1.f;
        const float *c = cs + (first ? d0 : d0 - half), *s = c + half;
#pragma unroll
        for (int i = 0; i < 16; i += 2) {
          float2 o[2];
#pragma unroll
          for (int j = 0; j < 2; ++j)
            o[j] = __fmul2_rn(make_float2(__shfl_sync(0xffffffffu, x[i + j].x, from), __shfl_sync(0xffffffffu, x[i + j].y, from)), make_float2(sign, sign));
          if (in) {
            const float4 kc = *reinterpret_cast<const float4 *>(c + 2 * i), ks = *reinterpret_cast<const float4 *>(s + 2 * i);
            // as rotary_first and rotary_second round it
            x[i] = __ffma2_rn(x[i], make_float2(kc.x, kc.y), __fmul2_rn(o[0], make_float2(ks.x, ks.y)));
            x[i + 1] = __ffma2_rn(x[i + 1], make_float2(kc.z, kc.w), __fmul2_rn(o[1], make_float2(ks.z, ks.w)));
          }
        }
      } else { // any other: the partner is fetched again (from L1)
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          const int d = d0 + i;
          if (d < a.r.dim) {
            const bool first = d < half;
            const int pair = first ? d : d - half;
            const float2 k = make_float2(cs[pair], sn[pair]);
            const float other = load_one(src, at + (first ? d + half : pair), a.type);
            float &v = (i & 1) ? x[i >> 1].y : x[i >> 1].x;
            v = first ? rotary_first(v, other, k) : rotary_second(v, other, k);
          }
        }
      }
    }

    float2 sum2 = make_float2(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < 16; ++i) sum2 = __ffma2_rn(x[i], x[i], sum2);
    float sum = sum2.x + sum2.y;
#pragma unroll
    for (int m = 1; m < LANES; m <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, m);
    const float norm = sqrtf(sum + 1e-12f), inv = 1.f / norm;
    // the transform first, the norm after it: sums of 16-bit values that are zero (a threshold) stay zero
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      x[i].x = __uint_as_float(__float_as_uint(x[i].x) ^ ((signs << (31 - 2 * i)) & 0x80000000u));
      x[i].y = __uint_as_float(__float_as_uint(x[i].y) ^ ((signs << (30 - 2 * i)) & 0x80000000u));
    }
    row_butterflies<P>(x, lane);
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i] = __fmul2_rn(x[i], make_float2(inv, inv));
    uint32_t w[BITS];
    pack_codes<P, BITS>(x, table, copy, w);

    if (r0 + lane / LANES < n_rows && page >= 0) {
      const long long slot = (((long long)page * heads + h) << a.c.page_shift) + off;
      if (!PAGED_CHECK(a.c.status, rows_exist(a.c, slot, 1) && off >= 0 && off < a.c.page_size)) continue;
      store_words<BITS>(pages + slot * (P * BITS / 8) + part * (4 * BITS), w);
      if (part == 0) scales[slot] = norm;
    }
  }
}

// blockIdx.y: 0 = keys, 1 = values.  Dynamic shared memory: the warps' turns.
template <int P, int KB, int VB> __global__ void __launch_bounds__(ROWS_THREADS, 3) paged_append_kernel(const RowsLaunch a) {
  extern __shared__ __align__(16) float turns[];
  __shared__ __align__(128) uint2 table[BUCKETS * BUCKET_COPIES];
  float *mine = turns + (threadIdx.x >> 5) * a.turn_tokens * a.r.dim;
  if (blockIdx.y == 0) {
    if constexpr (KB != 2) { fill_buckets<KB>(table, threadIdx.x); __syncthreads(); }
    append_rows<P, KB>(a, a.k, a.k_token, a.k_head, a.k_vec, a.c.k_pages, a.c.k_scales, a.r.dim > 0, mine, table);
  } else {
    if constexpr (VB != 2) { fill_buckets<VB>(table, threadIdx.x); __syncthreads(); }
    append_rows<P, VB>(a, a.v, a.v_token, a.v_head, a.v_vec, a.c.v_pages, a.c.v_scales, false, mine, table);
  }
}

// Read-back.  A warp takes 16 tokens of one head.  A code becomes the pair {upper, lower} of float16 parts of its
// codebook value, which is one register of the first operand of mma.sync m16n8k16: the contracted dimension holds both parts
// of eight codes, the second operand the signs of a Walsh-Hadamard transform of eight (twice, once for each part).  Lane
// (g, t) holds the coordinates t*P/4 .. of the rows g and g+8; the eight of a step are {t*P/4 + 2s + i}, i < 2, so
// the product transforms along t and i, and log2(P/8) stages of butterflies along s remain inside the lane.  22 bits
// of the codebook and float32 sums: as exact as the butterflies alone, which cost a quarter more time.  Bound by
// instructions (49 a row of 128, 2.2 a clock at 16 warps an SM): 30512 tokens x 8 heads at K4/V4 in fp16 take 44 us, 24 at
// the copy rate.
template <int BITS> __device__ __forceinline__ uint32_t code_bytes(const uint32_t *w, int i, const uint32_t *g24) {
  // a word that holds code i in its byte (see code_byte)
  if constexpr (BITS == 4) return (i & 1) ? w[i >> 3] & 0x0f0f0f0fu : (w[i >> 3] >> 4) & 0x0f0f0f0fu;
  else if constexpr (BITS == 2) return (w[i >> 4] >> (6 - 2 * (i & 3))) & 0x03030303u;
  else return (i & 1) ? g24[i >> 3] & 0x07070707u : (g24[i >> 3] >> 3) & 0x07070707u;
}
template <int BITS> __device__ __forceinline__ constexpr int code_byte(int i) { return BITS == 4 ? (i >> 1) & 3 : BITS == 2 ? (i >> 2) & 3 : 3 - ((i >> 1) & 3); }

constexpr int READ_WARPS = 8, READ_TOKENS = 64;

// 16-bit rows that are not made of aligned eights go out through shared memory, eight at a time, so that a warp stores
// neighbours: [8 rows][4 parts of P/8 words and a gap], which keeps the lanes' words in different banks.
template <int P> constexpr int stage_part = P / 8 + 1;
template <int P> constexpr int stage_words = 8 * 4 * stage_part<P>; // of a warp

template <int P, int BITS>
__device__ __forceinline__ void read_rows(const RowsLaunch &a, void *dst, long long dst_token, long long dst_head, int vec,
                                          const uint8_t *pages, const float *scales, uint32_t (*level)[32], TokenPlace *place,
                                          uint32_t *stage) {
  constexpr int N = P / 4, S = N / 2, WORDS = (N * BITS / 8 + 3) / 4;
  const int heads = a.c.heads, dim = a.c.dim, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const long long t0 = (long long)blockIdx.x * a.block_tokens;
  const int nt = (int)min((long long)a.block_tokens, a.n_tokens - t0);
  // a copy of the codebook for every lane: 32 reads of any codes hit 32 banks
  for (int i = threadIdx.x; i < (32 << BITS); i += READ_WARPS * 32) {
    const float c = c_cb[BITS - 2][i >> 5], upper = __half2float(__float2half_rn(c));
    level[i >> 5][i & 31] = pack2(upper, c - upper, TYPE_F16);
  }
  if (warp * 32 < nt) {
    const TokenPlace p = find_place(a, t0 + warp * 32, lane, min(32, nt - warp * 32));
    if (warp * 32 + lane < nt) place[warp * 32 + lane] = p;
  }
  __syncthreads();
  const uint32_t mine = smem_u32(&level[0][lane]);
  const int odd = __popc(t & (g >> 1)) & 1;
  const uint32_t b0 = odd ? 0xbc00bc00u : 0x3c003c00u, b1 = odd ^ (g & 1) ? 0xbc00bc00u : 0x3c003c00u; // {1, 1} or {-1, -1}
  // items: tiles of 16 tokens, heads; the codes of the next one are on their way while one is worked on
  const int items = (nt + 15) / 16 * heads, step = gridDim.z * READ_WARPS;
  uint32_t next[2][WORDS];
  float norm[2];
  auto fetch = [&](int item) {
    const int tile = item / heads, h = item - tile * heads;
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      norm[r] = 0.f;
#pragma unroll
      for (int i = 0; i < WORDS; ++i) next[r][i] = 0;
      const int row = 16 * tile + g + 8 * r;
      if (row < nt && place[row].page >= 0) {
        const long long slot = (((long long)place[row].page * heads + h) << a.c.page_shift) + place[row].off;
        if (!PAGED_CHECK(a.c.status, row < READ_TOKENS && h < heads && rows_exist(a.c, slot, 1))) continue;
        load_packed<N * BITS / 8>(pages + slot * (P * BITS / 8) + t * (N * BITS / 8), next[r]);
        norm[r] = scales[slot];
      }
    }
  };
  int item = blockIdx.z * READ_WARPS + warp;
  if (item < items) fetch(item);
  for (; item < items; item += step) {
    const int tile = item / heads, h = item - tile * heads;
    uint32_t w[2][WORDS], g24[2][BITS == 3 ? N / 8 : 1];
    float scale[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
#pragma unroll
      for (int i = 0; i < WORDS; ++i) w[r][i] = next[r][i];
      scale[r] = norm[r] * (1.f / P);
      if constexpr (BITS == 3) {
#pragma unroll
        for (int i = 0; i < N / 8; ++i) g24[r][i] = spread6(group24<WORDS>(w[r], i));
      }
    }
    if (item + step < items) fetch(item + step);
    float2 x[2][S]; // coordinates 2s, 2s+1 of this lane's part
#pragma unroll
    for (int s = 0; s < S; ++s) {
      uint32_t e[2][2];
#pragma unroll
      for (int r = 0; r < 2; ++r)
#pragma unroll
        for (int i = 0; i < 2; ++i)
          e[r][i] = table_one(__dp4a(code_bytes<BITS>(w[r], 2 * s + i, g24[r]), 0x80u << (8 * code_byte<BITS>(2 * s + i)), mine));
      float d[4];
      mma_16816_zero(d, e[0][0], e[1][0], e[0][1], e[1][1], b0, b1);
      x[0][s] = make_float2(d[0], d[1]);
      x[1][s] = make_float2(d[2], d[3]);
    }
#pragma unroll
    for (int len = 1; len < S; len <<= 1)
#pragma unroll
      for (int s = 0; s < S; ++s)
        if (!(s & len)) {
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const float2 u = x[r][s], v = x[r][s + len];
            x[r][s] = add2(u, v);
            x[r][s + len] = sub2(u, v);
          }
        }
    const uint32_t *signs = a.c.signs + h * (P / 32) + ((t * N) >> 5);
    const uint32_t word[2] = {signs[0] >> ((t * N) & 31), N > 32 ? signs[1] : 0u};
#pragma unroll
    for (int s = 0; s < S; ++s) {
      const uint32_t bits = word[s >> 4], f0 = (bits << (31 - 2 * (s & 15))) & 0x80000000u, f1 = (bits << (30 - 2 * (s & 15))) & 0x80000000u;
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const uint32_t f = __float_as_uint(scale[r]);
        x[r][s] = __fmul2_rn(x[r][s], make_float2(__uint_as_float(f ^ f0), __uint_as_float(f ^ f1)));
      }
    }
    if (!vec && a.type != TYPE_F32) {
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        __syncwarp();
#pragma unroll
        for (int s = 0; s < S; ++s) stage[(g * 4 + t) * stage_part<P> + s] = pack2(x[r][s].x, x[r][s].y, a.type);
        __syncwarp();
#pragma unroll 1
        for (int i = 0; i < 8; ++i) {
          const int row = 16 * tile + 8 * r + i;
          if (row >= nt || place[row].page < 0 || !PAGED_CHECK(a.c.status, t0 + row < a.n_tokens && h < heads)) continue;
          uint16_t *to = static_cast<uint16_t *>(dst) + (t0 + row) * dst_token + h * dst_head;
          const uint16_t *from = reinterpret_cast<const uint16_t *>(stage + i * 4 * stage_part<P>);
#pragma unroll 1
          for (int d = lane; d < dim; d += 32) to[d] = from[d + 2 * (d / N)];
        }
      }
      continue;
    }
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int row = 16 * tile + g + 8 * r;
      if (row >= nt || place[row].page < 0 || !PAGED_CHECK(a.c.status, t0 + row < a.n_tokens && h < heads)) continue;
      const long long at = (t0 + row) * dst_token + h * dst_head + t * N;
      if (vec) with_type(a.type, [&](auto type) {
        constexpr int TYPE = decltype(type)::value;
        if (TYPE != TYPE_F32 && vec == 2) {
#pragma unroll
          for (int i = 0; i < N; i += 16)
            if (t * N + i < dim) {
              uint32_t v[8];
#pragma unroll
              for (int j = 0; j < 8; ++j) v[j] = pack2(x[r][i / 2 + j].x, x[r][i / 2 + j].y, TYPE);
              store_32(static_cast<uint16_t *>(dst) + at + i, v);
            }
        } else {
#pragma unroll
          for (int i = 0; i < N; i += 8)
            if (t * N + i < dim) {
              const float v[8] = {x[r][i / 2].x, x[r][i / 2].y, x[r][i / 2 + 1].x, x[r][i / 2 + 1].y, x[r][i / 2 + 2].x, x[r][i / 2 + 2].y, x[r][i / 2 + 3].x, x[r][i / 2 + 3].y};
              store_eight<TYPE>(dst, at + i, v);
            }
        }
      }); else {
#pragma unroll
        for (int i = 0; i < N; ++i)
          if (t * N + i < dim) static_cast<float *>(dst)[at + i] = (i & 1) ? x[r][i >> 1].y : x[r][i >> 1].x;
      }
    }
  }
}

// Grid: block_tokens tokens, side (keys, values), share of their items.
template <int P, int KB, int VB> __global__ void __launch_bounds__(READ_WARPS * 32) paged_read_kernel(const RowsLaunch a) {
  __shared__ uint32_t level[16][32];
  __shared__ TokenPlace place[READ_TOKENS];
  __shared__ uint32_t stage[READ_WARPS * stage_words<P>];
  uint32_t *mine = stage + (threadIdx.x >> 5) * stage_words<P>;
  if (blockIdx.y == 0)
    read_rows<P, KB>(a, a.k, a.k_token, a.k_head, a.k_vec, a.c.k_pages, a.c.k_scales, level, place, mine);
  else
    read_rows<P, VB>(a, a.v, a.v_token, a.v_head, a.v_vec, a.c.v_pages, a.c.v_scales, level, place, mine);
}

} // namespace aq
