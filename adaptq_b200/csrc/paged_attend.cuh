// Attention of one new token per sequence over the pages.
//
// Work.  The tokens of a sequence are cut into units of U tokens; a unit belongs to one
// (sequence, KV head, pass of up to eight of its queries).  All units of the call, in that
// order, are cut into equal runs, one per warp of a persistent grid, wherever the cuts fall;
// the lengths are read on the device.  A warp works alone: it fetches its units into a ring of
// two (16-byte asynchronous copies), keeps its own reference and sums, and meets no barrier
// with other warps until it is done.  A run that starts or ends inside an item leaves a partial
// result; a block joins those of its warps when all are done, and paged_join_kernel those of
// items that span blocks.  (Joining those too in this kernel, by the last block to arrive, saves
// the launch and costs more: 2 us of a short call's 13, 5 of 79.)
// Bulk copies were tried first: issuing one costs its SM 80 clocks, whatever its size, and a unit
// takes four of them, or sixteen with pages of 16 tokens (33 sequences x 14 heads, 64 coordinates:
// 60 us a call against 39 with everything else equal).
//
// Arithmetic.  Codes become float16 values by table look-up: two codes are one index, its
// entry the two values side by side, and every entry lies in shared memory once per lane, so
// that 32 look-ups of any codes meet no bank twice.  Both products run on the tensor cores
// (mma.sync m16n8k16, float32 sums) with the tokens or the coordinates as the 16 rows and
// the queries of the KV head as the 8 columns:
//   scores   S[token][query] = K[token][dim] q[dim][query], a lane's codes of a row being
//            consecutive, since any order of the contracted dimension serves;
//   values   O[dim][query] += V^T[dim][token] w[token][query], where an entry holds the same
//            coordinate of two tokens: their codes are merged into indices by two logic
//            operations per word.
// What bounds it: latency at the eight to twelve warps an SM that the rings leave room for.  The shared-memory pipe
// is 0.7 busy over the call (380 wavefronts a unit of 64 tokens, 128 coordinates at K4/V2: 256 of look-ups, the rest
// copies, rows and norms), the issue slots half, behind 6 us of set-up.  64 sequences of 820 to 8192 tokens x 8 KV heads
// x 4 queries: 79 us, 3.1 TB/s; one of 131072 tokens at K4/V4: 50 us, 2.8 TB/s.
// tcgen05 would take its operands from shared or tensor memory: the expanded rows (512 bytes a
// token and head) would have to be stored first, 256 wavefronts a unit more for the pipe that is busiest here;
// mma.sync takes them from the registers in which the look-up leaves them.
//
// Precision.  float16 queries are scaled by their largest coordinate, weights times norms
// relative to the largest of them, so both keep 11 bits whatever their size; scores, sums and
// outputs are float32.  The codebook is scaled by a constant that brings its values close to
// float16 numbers: they are off by 1e-4 (4 bits), 4e-6 (3) and 2e-8 (2) at most.  Up to four
// queries leave columns free: columns 4-7 are then the lower float16 parts of queries and
// weights, 22 bits in all (SPLIT).  float32 calls also split the codebook (EXACT).
#pragma once
#include "paged_attend_host.h"

namespace aq {

constexpr int ATTEND_SMEM = 232448; // 227 KB
extern __shared__ __align__(128) uint8_t attend_smem[];

template <int KB, int VB, int P, int MODE> struct AttendShape {
  static constexpr int KEY_BITS = KB, VALUE_BITS = VB, DIM = P;
  static constexpr int KIND = MODE;
  static constexpr bool SPLIT = MODE >= 1, EXACT = MODE == 2;
  static constexpr int U = P == 256 ? 32 : 64;
  static constexpr int K_ROW = P * KB / 8, V_ROW = P * VB / 8;
  static constexpr int STAGE = U * (K_ROW + V_ROW + 8);
  static constexpr int COLS = SPLIT ? 4 : 8; // queries of a pass
  static constexpr int SUMS = 8 * P + 128; // floats of the workspace for the sums of a warp under way
  static constexpr int table_bytes(int bits) { return bits == 2 && !EXACT ? 32768 : 128 << (2 * bits); }
  static constexpr int K_TABLE = 0, V_TABLE = KB == VB ? 0 : table_bytes(KB);
  static constexpr int TABLES = table_bytes(KB) + (KB == VB ? 0 : table_bytes(VB));
  static constexpr int PER_WARP = 2 * STAGE + 48;
  static constexpr int FIXED = 512;
  static constexpr int FIT = (ATTEND_SMEM - FIXED - TABLES) / PER_WARP;
  static constexpr int CAP = P == 256 ? 8 : EXACT ? 12 : 16;
  static constexpr int WARPS = FIT >= CAP ? CAP : FIT / 4 * 4;
  static constexpr int THREADS = WARPS * 32;
  static constexpr int RING = TABLES;                         // [WARPS][2] stages
  static constexpr int DESC = RING + WARPS * 2 * STAGE;       // [WARPS][2] int4
  static constexpr int HEADERS = DESC + WARPS * 32;           // [WARPS] int4
  static constexpr int BLOCK = HEADERS + WARPS * 16;          // the chains of the join
  static constexpr int SMEM = BLOCK + FIXED;
  static_assert(WARPS >= 4 && SMEM <= ATTEND_SMEM, "shared memory");
  static_assert(STAGE >= 16 * P, "finish() puts four columns there");
};

// Length of sequence b as far as its table has room.
__device__ __forceinline__ int clipped_length(const AttendLaunch &a, int b, bool report) {
  const int n = a.lengths[b];
  const long long room = (long long)a.table.width << a.c.page_shift;
  if (n >= 0 && n <= room) return n;
  if (report) atomicOr(a.c.status, PAGED_BAD_POSITION);
  return n < 0 ? 0 : (int)room;
}

// n floats at p lie within the workspace (checked build).
__device__ __forceinline__ bool in_workspace(const AttendLaunch &a, const void *p, size_t n) {
  return p >= a.operands && static_cast<const float *>(p) + n <= a.workspace_end;
}

__device__ __forceinline__ int slot_floats(int cols, int P) { return cols * (P + 4); }

// The factor by which the tables' values are larger than the codebook's: of all factors from 1 to 2, the one
// whose largest rounding error to float16 is smallest (1.7e-8, 3.7e-6 and 1.0e-4 of a value; without it 2.3e-4 to
// 4.3e-4).
__host__ __device__ constexpr float table_scale(int bits) { return bits == 2 ? 1.2207031f : bits == 3 ? 1.1793699f : 1.57108554f; }

enum { SEG_FROM_BEFORE = 1, SEG_ENDS = 2, SEG_OPEN = 4 }; // header flags: slot 0 in use, its item ends here, slot 1 in use

__device__ __forceinline__ uint32_t transpose_8x8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t half2_bits(float a, float b) { return pack2(a, b, TYPE_F16); }

// Tables.  BITS bits a code; the index is (first code << BITS) | second code.
//   narrow, one part:   4 bytes {first, second} x 32 lanes
//   narrow, two parts:  8 bytes {first, second upper; first, second lower} x 16 lanes (a 64-bit read serves half a warp
//                       at a time)
//   wide (2 bits):      index = 4 codes of a byte, 8 bytes x 16 lanes
template <int BITS, bool EXACT> __device__ __forceinline__ void fill_table(uint8_t *table, int tid, int threads) {
  const float *c = c_cb[BITS - 2];
  constexpr float F = table_scale(BITS);
  if constexpr (EXACT) {
    for (int i = tid; i < (16 << (2 * BITS)); i += threads) {
      const int index = i >> 4;
      const float a = c[index >> BITS], b = c[index & ((1 << BITS) - 1)];
      const uint32_t upper = half2_bits(a * F, b * F);
      const float2 u = unpack2(upper, TYPE_F16);
      reinterpret_cast<uint2 *>(table)[i] = make_uint2(upper, half2_bits(fmaf(a, F, -u.x), fmaf(b, F, -u.y))); // from the unrounded products
    }
  } else if constexpr (BITS == 2) {
    for (int i = tid; i < 256 * 16; i += threads) {
      const int index = i >> 4;
      reinterpret_cast<uint2 *>(table)[i] = make_uint2(half2_bits(c[index >> 6] * F, c[(index >> 4) & 3] * F), half2_bits(c[(index >> 2) & 3] * F, c[index & 3] * F));
    }
  } else {
    for (int i = tid; i < (32 << (2 * BITS)); i += threads) {
      const int index = i >> 5;
      reinterpret_cast<uint32_t *>(table)[i] = half2_bits(c[index >> BITS] * F, c[index & ((1 << BITS) - 1)] * F);
    }
  }
}

// Entry of a table whose place for this lane is `base` (a shared-memory address): the index are the WIDTH bits of w
// from pos on, entries are 2^SHIFT bytes apart.  Whole bytes take one instruction, a dot product that picks the byte
// and scales it.  The tables do not change once filled, so the loads may move freely.
template <int WIDTH, int SHIFT> __device__ __forceinline__ uint32_t entry_address(uint32_t base, uint32_t w, int pos) {
  if constexpr (WIDTH == 8 && SHIFT == 7) return __dp4a(w, 0x80u << pos, base);
  else if constexpr (WIDTH == 6 && SHIFT == 7) return __dp4a(w, 0x80u << pos, base); // fields spread to bytes
  else return ((pos >= SHIFT ? w >> (pos - SHIFT) : w << (SHIFT - pos)) & (((1u << WIDTH) - 1) << SHIFT)) + base;
}
__device__ __forceinline__ uint2 table_two(uint32_t at) {
  uint2 v;
  asm("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(at));
  return v;
}

// One query's sum of weighted values (coordinates lane*P/32 .. of the transformed domain) and of weights -> its output row.
template <int P> __device__ __forceinline__ void store_column(const AttendLaunch &a, int b, int h, int query, int lane, float (&v)[P / 32], float sum) {
  constexpr int E = P / 32;
  warp_butterflies<E>(v, lane);
  const float inv = sum == 0.f ? 0.f : 1.f / (sum * P);
  if (!PAGED_CHECK(a.c.status, b >= 0 && b < a.n_seqs && h >= 0 && h < a.c.heads && query >= 0 && query < a.group)) return;
  const uint32_t signs = a.c.signs[h * E + lane / (32 / E)] >> (lane * E & 31);
  const long long at = (long long)b * a.out_seq + (long long)(h * a.group + query) * a.out_head + lane * E;
#pragma unroll
  for (int i = 0; i < E; ++i) v[i] *= ((signs >> i) & 1u) ? -inv : inv;
  if (a.out_vec && a.type != TYPE_F32) {
#pragma unroll
    for (int i = 0; i < E; i += 2)
      if (lane * E + i < a.c.dim) *reinterpret_cast<uint32_t *>(static_cast<uint16_t *>(a.out) + at + i) = pack2(v[i], v[i + 1], a.type);
  } else {
#pragma unroll
    for (int i = 0; i < E; ++i)
      if (lane * E + i < a.c.dim) store_one(a.out, at + i, a.type, v[i]);
  }
}

template <int KB, int VB, int P, int MODE> struct AttendWarp {
  using S = AttendShape<KB, VB, P, MODE>;
  static constexpr int U = S::U, TILES = U / 16, DIM_TILES = P / 16;
  static constexpr int K_PART = S::K_ROW / 4, V_PART = S::V_ROW / 8; // bytes of a row that a lane reads
  static constexpr int K_WORDS = (K_PART + 3) / 4, V_WORDS = (V_PART + 3) / 4;

  static constexpr bool SPLIT = S::SPLIT, EXACT = S::EXACT;

  int lane, g, t, phi;         // row of a tile -> token of a tile: row 2t is token t, row 2t+1 token 7-t (and 8 more), see below
  uint32_t k_table, v_table;   // this lane's places in the tables
  uint32_t qb[P / 8];          // the queries, as the second operand
  float acc[DIM_TILES][4];
  float ref[2], l[2], fq[2]; // of the queries 2t, 2t+1 (SPLIT: modulo 4): weights are 2^(fq * score - ref)

  __device__ __forceinline__ void init(int ln) {
    lane = ln; g = ln >> 2; t = ln & 3;
    // Tokens are assigned to rows so that neither the reads of key rows (rows g, g+8) nor those of value
    // rows (rows 2t, 2t+1, 2t+8, 2t+9) of 32 or 64 bytes meet in a bank more often than their size makes them.
    phi = (g & 1) ? 7 - (g >> 1) : g >> 1;
    k_table = smem_u32(attend_smem) + S::K_TABLE + (EXACT || KB == 2 ? (ln & 15) * 8 : ln * 4);
    v_table = smem_u32(attend_smem) + S::V_TABLE + (EXACT || VB == 2 ? (ln & 15) * 8 : ln * 4);
  }

  // Codes 2p, 2p+1 of this lane's part of a key row.
  __device__ __forceinline__ static uint32_t key_word(const uint32_t (&w)[K_WORDS], const uint32_t *g24, int p, int &pos) {
    if constexpr (KB == 4) { pos = 8 * (p & 3); return w[p >> 2]; }
    else if constexpr (KB == 2) { pos = 8 * ((p >> 1) & 3) + ((p & 1) ? 0 : 4); return w[p >> 3]; }
    else { pos = 24 - 8 * (p & 3); return g24[p >> 2]; }
  }

  __device__ __forceinline__ void load_queries(const AttendLaunch &a, size_t item) {
    if (!PAGED_CHECK(a.c.status, item < (size_t)a.n_seqs * a.c.heads * a.passes)) item = 0;
#pragma unroll
    for (int i = 0; i < P / 8; ++i) qb[i] = a.operands[(item * (P / 8) + i) * 32 + lane];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      fq[e] = a.query_scales[item * 8 + (SPLIT ? (2 * t + e) & 3 : 2 * t + e)];
      ref[e] = -1e30f; l[e] = 0.f;
    }
#pragma unroll
    for (int j = 0; j < DIM_TILES; ++j) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.f;
  }

  // One unit: n of its U tokens count.
  __device__ __forceinline__ void unit(int stage, int n) {
    const uint8_t *keys = attend_smem + stage, *vals = keys + U * S::K_ROW;
    const float *ks = reinterpret_cast<const float *>(attend_smem + stage + U * (S::K_ROW + S::V_ROW)), *vs = ks + U;
    float s[TILES][4];
    // two tiles a round; with the codebook in two parts unrolled rounds would not stay in the instruction cache (rolled, and
    // with tables half the size, 20 x 6 heads of 96 coordinates went from 49 to 37 us)
#pragma unroll (EXACT ? 1 : TILES / 2)
    for (int round = 0; round < TILES / 2; ++round) {
#pragma unroll
      for (int i = 0; i + 2 < TILES; ++i) {
#pragma unroll
        for (int j = 0; j < 4; ++j) s[i][j] = s[i + 2][j];
      }
#pragma unroll
      for (int i = TILES - 2; i < TILES; ++i) {
        const uint8_t *tile = keys + (32 * round + 16 * (i - TILES + 2) + phi) * S::K_ROW + t * K_PART;
        s[i][0] = s[i][1] = s[i][2] = s[i][3] = 0.f;
        uint32_t w[2][K_WORDS], g24[2][KB == 3 ? P / 32 : 1];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          load_packed<K_PART>(tile + 8 * r * S::K_ROW, w[r]);
          if constexpr (KB == 3) {
#pragma unroll
            for (int k = 0; k < P / 32; ++k) g24[r][k] = spread6(group24<K_WORDS>(w[r], k));
          }
        }
        if constexpr (KB == 2 && !EXACT) {
          // a byte: two codes of one row and two of the other, an entry: the operands of both
#pragma unroll
          for (int k = 0; k < K_WORDS; ++k) {
            const uint32_t x = (w[0][k] & 0xf0f0f0f0u) | ((w[1][k] >> 4) & 0x0f0f0f0fu), y = ((w[0][k] << 4) & 0xf0f0f0f0u) | (w[1][k] & 0x0f0f0f0fu);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const uint2 u = table_two(entry_address<8, 7>(k_table, x, 8 * j)), v = table_two(entry_address<8, 7>(k_table, y, 8 * j));
              mma_16816(s[i], u.x, u.y, v.x, v.y, qb[8 * k + 2 * j], qb[8 * k + 2 * j + 1]);
            }
          }
        } else {
          float odd[4] = {}, low[4] = {}; // EXACT
#pragma unroll
          for (int k = 0; k < DIM_TILES; ++k) {
            uint32_t word[2][2];
            int pos[2];
#pragma unroll
            for (int r = 0; r < 2; ++r)
#pragma unroll
              for (int p = 0; p < 2; ++p) word[r][p] = key_word(w[r], g24[r], 2 * k + p, pos[p]);
            if constexpr (EXACT) {
              uint2 v[2][2];
#pragma unroll
              for (int r = 0; r < 2; ++r)
#pragma unroll
                for (int p = 0; p < 2; ++p) v[r][p] = table_two(entry_address<2 * KB, 7>(k_table, word[r][p], pos[p]));
              // The tensor cores cut sums off instead of rounding them: short chains, added up in float32.
              if (k & 1) mma_16816(odd, v[0][0].x, v[1][0].x, v[0][1].x, v[1][1].x, qb[2 * k], qb[2 * k + 1]);
              else mma_16816(s[i], v[0][0].x, v[1][0].x, v[0][1].x, v[1][1].x, qb[2 * k], qb[2 * k + 1]);
              mma_16816(low, v[0][0].y, v[1][0].y, v[0][1].y, v[1][1].y, qb[2 * k], qb[2 * k + 1]);
            } else {
              uint32_t v[2][2];
#pragma unroll
              for (int r = 0; r < 2; ++r)
#pragma unroll
                for (int p = 0; p < 2; ++p) v[r][p] = table_one(entry_address<2 * KB, 7>(k_table, word[r][p], pos[p]));
              mma_16816(s[i], v[0][0], v[1][0], v[0][1], v[1][1], qb[2 * k], qb[2 * k + 1]);
            }
          }
          if constexpr (EXACT) {
#pragma unroll
            for (int j = 0; j < 4; ++j) s[i][j] += odd[j] + low[j];
          }
        }
      }
    }
    // softmax: s becomes the logit over fq, then weight times the value's norm
    float top[2] = {-1e30f, -1e30f}, norm[TILES][2], largest = 0.f; // largest: norm of this lane's values
#pragma unroll
    for (int i = 0; i < TILES; ++i)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const float scale = ks[16 * i + 8 * r + phi];
        norm[i][r] = vs[16 * i + 8 * r + phi];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float &z = s[i][2 * r + e];
          if constexpr (SPLIT) z += __shfl_xor_sync(0xffffffffu, z, 2);
          z *= scale;
        }
      }
    if (n < U) { // what lies behind the sequence's end may be anything
#pragma unroll
      for (int i = 0; i < TILES; ++i)
#pragma unroll
        for (int r = 0; r < 2; ++r)
          if (16 * i + 8 * r + phi >= n) { s[i][2 * r] = s[i][2 * r + 1] = -INFINITY; norm[i][r] = 0.f; }
    }
#pragma unroll
    for (int i = 0; i < TILES; ++i) {
      largest = fmaxf(largest, fmaxf(norm[i][0], norm[i][1]));
#pragma unroll
      for (int e = 0; e < 2; ++e) top[e] = fmaxf(top[e], fmaxf(s[i][e], s[i][2 + e]));
    }
    // The reference stays as long as no weight exceeds 2^100 and no weight times norm 2^15.  Where it is set, the largest
    // weight times norm becomes 2^9: float16 then holds everything down to 2^-33 of that one, so that very many tokens
    // far below a single one still add up.
    const float room = fminf(100.f, 15.f - __log2f(largest));
    if (__any_sync(0xffffffffu, fmaf(top[0], fq[0], -ref[0]) > room || fmaf(top[1], fq[1], -ref[1]) > room)) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float high = top[e], product = -100.f;
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) high = fmaxf(high, __shfl_xor_sync(0xffffffffu, high, o));
        high *= fq[e];
#pragma unroll
        for (int i = 0; i < TILES; ++i)
#pragma unroll
          for (int r = 0; r < 2; ++r) product = fmaxf(product, fmaf(s[i][2 * r + e], fq[e], -high) + __log2f(norm[i][r]));
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) product = fmaxf(product, __shfl_xor_sync(0xffffffffu, product, o));
        const float next = fmaxf(ref[e], high + product - 9.f), ratio = exp2_approx(ref[e] - next);
        ref[e] = next;
        l[e] *= ratio;
#pragma unroll
        for (int j = 0; j < DIM_TILES; ++j) { acc[j][e] *= ratio; acc[j][2 + e] *= ratio; }
      }
    }
#pragma unroll
    for (int i = 0; i < TILES; ++i)
#pragma unroll
      for (int r = 0; r < 2; ++r)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float &z = s[i][2 * r + e];
          const float p = exp2_approx(fmaf(z, fq[e], -ref[e]));
          l[e] += p;
          z = p * norm[i][r];
        }
#pragma unroll (EXACT ? 1 : TILES / 2)
    for (int round = 0; round < TILES / 2; ++round) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint8_t *tile = vals + (32 * round + 16 * i) * S::V_ROW + g * V_PART;
        uint32_t wt[2];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const float x = s[i][2 * r], y = s[i][2 * r + 1];
          uint32_t w = half2_bits(x, y);
          if constexpr (SPLIT) {
            const float2 upper = unpack2(w, TYPE_F16);
            const uint32_t lower = half2_bits(x - upper.x, y - upper.y);
            w = t >= 2 ? lower : w;
          }
          wt[r] = transpose_8x8(w);
        }
        // the codes of one coordinate of two tokens side by side: even coordinates in x, odd ones in y
        uint32_t x[2][VB == 3 ? P / 64 : V_WORDS], y[2][VB == 3 ? P / 64 : V_WORDS];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          uint32_t wa[V_WORDS], wb[V_WORDS];
          load_packed<V_PART>(tile + (8 * r + t) * S::V_ROW, wa);
          load_packed<V_PART>(tile + (8 * r + 7 - t) * S::V_ROW, wb);
          if constexpr (VB == 3) {
#pragma unroll
            for (int k = 0; k < P / 64; ++k) {
              const uint32_t va = group24<V_WORDS>(wa, k), vb = group24<V_WORDS>(wb, k);
              x[r][k] = spread6((va & 070707070) | ((vb >> 3) & 007070707));
              y[r][k] = spread6(((va << 3) & 070707070) | (vb & 007070707));
            }
          } else {
            constexpr uint32_t HI = VB == 4 ? 0xf0f0f0f0u : 0xccccccccu;
#pragma unroll
            for (int k = 0; k < V_WORDS; ++k) {
              x[r][k] = (wa[k] & HI) | ((wb[k] >> VB) & ~HI);
              y[r][k] = ((wa[k] << VB) & HI) | (wb[k] & ~HI);
            }
          }
        }
        if constexpr (VB == 2 && !EXACT) {
#pragma unroll
          for (int j = 0; j < DIM_TILES; j += 2) { // a byte: coordinates 2j and 2j+2, or 2j+1 and 2j+3 (rows g and g+8)
            const uint2 a = table_two(entry_address<8, 7>(v_table, x[0][j >> 3], 8 * ((j >> 1) & 3))), b = table_two(entry_address<8, 7>(v_table, x[1][j >> 3], 8 * ((j >> 1) & 3)));
            mma_16816(acc[j], a.x, a.y, b.x, b.y, wt[0], wt[1]);
            const uint2 c = table_two(entry_address<8, 7>(v_table, y[0][j >> 3], 8 * ((j >> 1) & 3))), d = table_two(entry_address<8, 7>(v_table, y[1][j >> 3], 8 * ((j >> 1) & 3)));
            mma_16816(acc[j + 1], c.x, c.y, d.x, d.y, wt[0], wt[1]);
          }
        } else {
#pragma unroll
          for (int j = 0; j < DIM_TILES; ++j) {
            const int k = VB == 4 || VB == 3 ? j >> 2 : j >> 3;
            const int pos = VB == 4 ? 8 * (j & 3) : VB == 3 ? 24 - 8 * (j & 3) : 8 * ((j >> 1) & 3) + ((j & 1) ? 0 : 4);
            const uint32_t src[4] = {x[0][k], y[0][k], x[1][k], y[1][k]};
            if constexpr (EXACT) {
              uint2 v[4];
#pragma unroll
              for (int q = 0; q < 4; ++q) v[q] = table_two(entry_address<2 * VB, 7>(v_table, src[q], pos));
              // Short chains here as well: acc lives as long as the run, and being cut off thousands of times takes
              // more off it than rounding does (32768 tokens of one direction a warp: 2e-4 of the sum instead of
              // 6e-7; the additions cost 0.5 us of the 36.5 of 20 x 6 heads).
              float d[4];
              mma_16816_zero(d, v[0].x, v[1].x, v[2].x, v[3].x, wt[0], wt[1]);
              mma_16816(d, v[0].y, v[1].y, v[2].y, v[3].y, wt[0], wt[1]);
#pragma unroll
              for (int q = 0; q < 4; q += 2) {
                const float2 sum = __fadd2_rn(make_float2(acc[j][q], acc[j][q + 1]), make_float2(d[q], d[q + 1]));
                acc[j][q] = sum.x; acc[j][q + 1] = sum.y;
              }
            } else {
              uint32_t v[4];
#pragma unroll
              for (int q = 0; q < 4; ++q) v[q] = table_one(entry_address<2 * VB, 7>(v_table, src[q], pos));
              mma_16816(acc[j], v[0], v[1], v[2], v[3], wt[0], wt[1]);
            }
          }
        }
      }
#pragma unroll
      for (int i = 0; i + 2 < TILES; ++i) {
#pragma unroll
        for (int j = 0; j < 4; ++j) s[i][j] = s[i + 2][j];
      }
    }
  }

  // The tensor cores cut sums off instead of rounding them, 2^-23 of the sum a product, all to one side, and a float32 sum
  // that holds one large term loses what is added to it in small pieces.  So a long run hands its sums over every KEEP
  // units: to `place` (a lane's own words in the workspace, with the references they are relative to), which is added up
  // in float32 and comes back at the end.  131072 tokens of one direction a warp: 9e-4 of the sum before, 2e-5 now; as
  // many of 2^-27 of one before them, float32: 2e-4, 7e-6 now; 64 x 8 heads x 8192 tokens: 78.4 us, 79.2 now, through the
  // registers that the code takes.
  static constexpr int KEEP = 64;
  __device__ __forceinline__ void hand_over(float *place, bool more) {
    float4 *mine = reinterpret_cast<float4 *>(place) + lane;
    float4 *sums = reinterpret_cast<float4 *>(place + 8 * P) + lane; // references and sums of weights
    float ratio[2] = {0.f, 0.f};
    if (more) {
      const float4 old = *sums;
      ratio[0] = exp2_approx(old.x - ref[0]);
      ratio[1] = exp2_approx(old.y - ref[1]);
      l[0] = fmaf(old.z, ratio[0], l[0]);
      l[1] = fmaf(old.w, ratio[1], l[1]);
    }
    *sums = make_float4(ref[0], ref[1], l[0], l[1]);
    l[0] = l[1] = 0.f;
#pragma unroll
    for (int j = 0; j < DIM_TILES; ++j) {
      const float4 old = more ? mine[32 * j] : make_float4(0.f, 0.f, 0.f, 0.f);
      mine[32 * j] = make_float4(fmaf(old.x, ratio[0], acc[j][0]), fmaf(old.y, ratio[1], acc[j][1]), fmaf(old.z, ratio[0], acc[j][2]),
                                 fmaf(old.w, ratio[1], acc[j][3]));
      acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.f;
    }
  }
  __device__ __forceinline__ void take_back(const float *place) {
    const float4 *mine = reinterpret_cast<const float4 *>(place) + lane;
    const float4 old = reinterpret_cast<const float4 *>(place + 8 * P)[lane];
    const float ratio[2] = {exp2_approx(old.x - ref[0]), exp2_approx(old.y - ref[1])};
    l[0] = fmaf(old.z, ratio[0], l[0]);
    l[1] = fmaf(old.w, ratio[1], l[1]);
#pragma unroll
    for (int j = 0; j < DIM_TILES; ++j) {
      const float4 v = mine[32 * j];
      acc[j][0] = fmaf(v.x, ratio[0], acc[j][0]); acc[j][1] = fmaf(v.y, ratio[1], acc[j][1]);
      acc[j][2] = fmaf(v.z, ratio[0], acc[j][2]); acc[j][3] = fmaf(v.w, ratio[1], acc[j][3]);
    }
  }

  // The item ends here, or this warp's run does: its result goes out, or into a slot of the workspace.  Four columns
  // at a time pass through `scratch` (16 P bytes of shared memory), after which a column lies across the warp.
  __device__ __forceinline__ void finish(const AttendLaunch &a, int b, int h, int pass, int ncols, bool whole, float *slot, float *scratch) {
    constexpr int N = P / 8, E = P / 32;
#pragma unroll
    for (int e = 0; e < 2; ++e)
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) l[e] += __shfl_xor_sync(0xffffffffu, l[e], o);
#pragma unroll 1
    for (int e = 0; e < 2; ++e) {
      __syncwarp();
      float x[N];
#pragma unroll
      for (int j = 0; j < DIM_TILES; ++j) {
        // the coordinates of rows g and g+8 of this tile
        const int lo = VB == 2 && !EXACT ? 4 * (j >> 1) + (j & 1) : 2 * j, hi = VB == 2 && !EXACT ? lo + 2 : lo + 1;
        x[lo] = e ? acc[j][1] : acc[j][0];
        x[hi] = e ? acc[j][3] : acc[j][2];
      }
#pragma unroll
      for (int i = 0; i < N; i += 4) *reinterpret_cast<float4 *>(scratch + t * P + g * N + i) = make_float4(x[i], x[i + 1], x[i + 2], x[i + 3]);
      __syncwarp();
      const float le = e ? l[1] : l[0], re = e ? ref[1] : ref[0];
#pragma unroll 1
      for (int k = 0; 2 * k + e < ncols; ++k) { // lane k (row 0) holds the column's sums
        const float sum = __shfl_sync(0xffffffffu, le, k), top = __shfl_sync(0xffffffffu, re, k);
        float v[E];
#pragma unroll
        for (int i = 0; i < E; ++i) v[i] = (scratch[k * P + lane * E + i] + (SPLIT ? scratch[(k + 2) * P + lane * E + i] : 0.f)) * (1.f / table_scale(VB));
        const int col = 2 * k + e;
        if (whole) store_column<P>(a, b, h, pass * S::COLS + col, lane, v, sum);
        else if (PAGED_CHECK(a.c.status, col < a.slot_cols && in_workspace(a, slot, slot_floats(a.slot_cols, P)))) {
#pragma unroll
          for (int i = 0; i < E; ++i) slot[col * P + lane * E + i] = v[i];
          if (lane == 0) *reinterpret_cast<float2 *>(slot + a.slot_cols * P + 2 * col) = make_float2(top, sum);
        }
      }
    }
  }
};

// Sum of `pieces` partial results of one query: v[P/32] a lane (coordinates lane*P/32 ..), relative to the largest
// maximum.  piece(i) is the slot of the i-th, first <= i < pieces in steps of `step`.
template <int P, typename F>
__device__ __forceinline__ void join_pieces(F piece, int pieces, int first, int step, int cols, int col, int lane, float (&v)[P / 32], float &M, float &L) {
  constexpr int E = P / 32;
  M = -INFINITY; L = 0.f;
#pragma unroll
  for (int i = 0; i < E; ++i) v[i] = 0.f;
  for (int i = lane; i < pieces; i += 32) M = fmaxf(M, piece(i)[cols * P + 2 * col]);
  M = warp_max(M);
#pragma unroll 4
  for (int i = first; i < pieces; i += step) {
    const float *s = piece(i);
    const float2 stat = *reinterpret_cast<const float2 *>(s + cols * P + 2 * col);
    const float w = exp2_approx(stat.x - M);
    L = fmaf(w, stat.y, L);
    const float *x = s + col * P + lane * E;
    if constexpr (E == 2) {
      const float2 u = *reinterpret_cast<const float2 *>(x);
      v[0] = fmaf(w, u.x, v[0]); v[1] = fmaf(w, u.y, v[1]);
    } else {
#pragma unroll
      for (int j = 0; j < E; j += 4) {
        const float4 u = *reinterpret_cast<const float4 *>(x + j);
        v[j] = fmaf(w, u.x, v[j]); v[j + 1] = fmaf(w, u.y, v[j + 1]); v[j + 2] = fmaf(w, u.z, v[j + 2]); v[j + 3] = fmaf(w, u.w, v[j + 3]);
      }
    }
  }
}

__device__ __forceinline__ int live_cols(const AttendLaunch &a, int item, int cols) {
  const int pass = item % a.passes;
  return min(cols, a.group - pass * cols);
}

struct JoinChain { int first, slot, count, item, kind; }; // kind 0: complete, 1: to block slot 0, 2: to block slot 1

// The queries as operands of the scores: rotated, transformed, in float16 relative to their largest coordinate (in two
// parts, if COLS is 4), in the order in which the lanes of paged_attend_kernel hold them.  A block per (sequence, KV
// head, pass), a warp per query; runs beside the set-up of paged_attend_kernel.
constexpr int QUERY_WARPS = 4;
template <int P> __global__ void __launch_bounds__(QUERY_WARPS * 32) paged_query_kernel(const AttendLaunch a, int cols, float unit) {
  constexpr int E = P / 32;
  __shared__ float raw[QUERY_WARPS][P], turned[QUERY_WARPS][P];
  griddep_launch_dependents();
  const int item = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int per_seq = a.c.heads * a.passes, b = item / per_seq, hp = item - b * per_seq, h = hp / a.passes, pass = hp - h * a.passes;
  const long long pos = (long long)clipped_length(a, b, false) - 1;
  if (pos < 0) return;
  const int ncols = min(cols, a.group - pass * cols), half = a.r.dim >> 1;
  for (int col = warp; col < cols; col += QUERY_WARPS) {
    float v[E], scale = 1e-37f;
#pragma unroll
    for (int i = 0; i < E; ++i) v[i] = 0.f;
    if (col < ncols) {
      const long long at = (long long)b * a.q_seq + (long long)(h * a.group + pass * cols + col) * a.q_head;
      __syncwarp();
      for (int d = lane; d < P; d += 32) turned[warp][d] = raw[warp][d] = d < a.c.dim ? load_one(a.q, at + d, a.type) : 0.f;
      __syncwarp();
      for (int pair = lane; pair < half; pair += 32) {
        const int d = a.r.interleaved ? 2 * pair : pair, e = a.r.interleaved ? d + 1 : d + half;
        const float2 k = rotary_turn(a.r, pair, pos);
        turned[warp][d] = rotary_first(raw[warp][d], raw[warp][e], k);
        turned[warp][e] = rotary_second(raw[warp][e], raw[warp][d], k);
      }
      __syncwarp();
      const uint32_t signs = a.c.signs[h * E + lane / (32 / E)] >> (lane * E & 31);
#pragma unroll
      for (int i = 0; i < E; ++i) v[i] = ((signs >> i) & 1u) ? -turned[warp][lane * E + i] : turned[warp][lane * E + i];
      warp_butterflies<E>(v, lane);
      float top = 1e-30f;
#pragma unroll
      for (int i = 0; i < E; ++i) top = fmaxf(top, fabsf(v[i]));
      top = warp_max(top);
      scale = fmaxf(top * (a.scale * unit), 1e-37f);
      const float inv = 1.f / top;
#pragma unroll
      for (int i = 0; i < E; ++i) v[i] *= inv;
    }
    // coordinates d .. d+3 of column g: operands (d % (P/4)) / 2 and the next, of lane 4 g + d / (P/4)
#pragma unroll
    for (int i = 0; i < E; i += 2) {
      const int d = lane * E + i;
      if (!PAGED_CHECK(a.c.status, (size_t)item < (size_t)a.n_seqs * per_seq && col < cols)) continue;
      uint32_t *to = a.operands + ((size_t)item * (P / 8) + (d % (P / 4)) / 2) * 32 + 4 * col + d / (P / 4);
      const uint32_t upper = pack2(v[i], v[i + 1], TYPE_F16);
      *to = upper;
      if (cols == 4) {
        const float2 u = unpack2(upper, TYPE_F16);
        to[16] = pack2(v[i] - u.x, v[i + 1] - u.y, TYPE_F16);
      }
    }
    if (lane == 0) a.query_scales[(size_t)item * 8 + col] = scale;
  }
}

__device__ __forceinline__ void copy_16(uint32_t to, const void *from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}
__device__ __forceinline__ void copies_done() { asm volatile("cp.async.wait_all;" ::: "memory"); }

// A warp's walk over its run of units, and the fetch of them.
template <typename S> struct AttendWalk {
  static constexpr int U = S::U;
  int b, h, pass, u, nu, len; // the unit to be fetched next
  int page;                   // lane i: the page that holds its i-th part (0 where there is none), read one unit ahead
  int lane;

  // The run of warp `warp` of this block; returns its number of units.
  __device__ __forceinline__ int start(const AttendLaunch &a, int warp, int ln) {
    lane = ln;
    b = h = pass = u = len = page = 0;
    nu = 1;
    const int per_seq = a.c.heads * a.passes;
    // units before every lane's share of the sequences (the host refuses calls whose units 31 bits would not count)
    const int chunk = (a.n_seqs + 31) / 32, b0 = min(a.n_seqs, lane * chunk), b1 = min(a.n_seqs, b0 + chunk);
    int sum = 0;
#pragma unroll 4
    for (int i = b0; i < b1; ++i) sum += (clipped_length(a, i, blockIdx.x == 0 && warp == 0) + U - 1) / U;
    sum *= per_seq;
    const int own = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += v;
    }
    const int total = __shfl_sync(0xffffffffu, sum, 31), before = sum - own;
    // blocks share the units evenly, and so do the warps of a block; no block is without any as long as there are some
    const int blocks = min((int)gridDim.x, total), block = blockIdx.x;
    if (block >= blocks) return 0;
    const int even = total / blocks, more = total - even * blocks;
    const int first = even * block + min(block, more), share = even + (block < more);
    const int per_warp = share / S::WARPS, rest_warps = share - per_warp * S::WARPS;
    const int units = per_warp + (warp < rest_warps);
    if (units == 0) return 0;
    // the last lane whose share begins at or before the run, then along that share
    int rest = first + per_warp * warp + min(warp, rest_warps);
    const int at = 31 - __clz(__ballot_sync(0xffffffffu, before <= rest));
    rest -= __shfl_sync(0xffffffffu, before, at);
    for (b = at * chunk;; ++b) {
      if (b >= a.n_seqs) { b = 0; return 0; } // lengths that someone changed meanwhile must not lead out of them
      len = clipped_length(a, b, false);
      nu = (len + U - 1) / U;
      if (rest < nu * per_seq) break;
      rest -= nu * per_seq;
    }
    const int hp = rest / nu;
    u = rest - hp * nu;
    h = hp / a.passes;
    pass = hp - h * a.passes;
    find_pages(a);
    return units;
  }
  __device__ __forceinline__ void find_pages(const AttendLaunch &a) {
    page = 0;
    if (lane << a.c.page_shift < min(U, len - u * U) && PAGED_CHECK(a.c.status, b >= 0 && b < a.n_seqs && u >= 0 && ((u * U) >> a.c.page_shift) + lane < a.table.width))
      page = a.table.entries[(long long)b * a.table.stride + ((u * U) >> a.c.page_shift) + lane];
  }
  // Start the copies of the next unit into `stage` and describe it; then, if there are more, find the one behind it.
  __device__ __forceinline__ void fetch(const AttendLaunch &a, int stage, int4 *desc, bool more) {
    const int tok0 = u * U, n = min(U, len - tok0);
    const bool bad = __any_sync(0xffffffffu, page < 0 || page >= a.c.n_pages);
    if (lane == 0) {
      *desc = make_int4(b, h | pass << 16, u | (u + 1 == nu ? 0x40000000 : 0), bad ? 0 : n);
      if (bad) atomicOr(a.c.status, PAGED_BAD_PAGE);
    }
    if (!bad) {
      const uint32_t to = smem_u32(attend_smem) + stage + lane * 16;
      const uint8_t *norms = reinterpret_cast<const uint8_t *>(lane * 16 < 4 * U ? a.c.k_scales : a.c.v_scales);
      const int norm_at = lane * 16 < 4 * U ? lane * 16 : lane * 16 - 4 * U; // both kinds of norms are 8 U bytes of the stage
      if (a.c.page_size >= U) {
        const long long row = (((long long)__shfl_sync(0xffffffffu, page, 0) * a.c.heads + h) << a.c.page_shift) + (tok0 & (a.c.page_size - 1));
        const uint8_t *k = a.c.k_pages + row * S::K_ROW + lane * 16, *v = a.c.v_pages + row * S::V_ROW + lane * 16;
        if (!PAGED_CHECK(a.c.status, h >= 0 && h < a.c.heads && rows_exist(a.c, row, U))) return;
#pragma unroll
        for (int i = 0; i < U * S::K_ROW / 512; ++i) copy_16(to + i * 512, k + i * 512);
#pragma unroll
        for (int i = 0; i < U * S::V_ROW / 512; ++i) copy_16(to + U * S::K_ROW + i * 512, v + i * 512);
        if (lane * 16 < 8 * U) copy_16(to + U * (S::K_ROW + S::V_ROW), norms + row * 4 + norm_at);
      } else {
        // the pages of the unit one after another
#pragma unroll 1
        for (int p = 0; p << a.c.page_shift < n; ++p) {
          const int per = a.c.page_size, at = p << a.c.page_shift;
          const long long row = ((long long)__shfl_sync(0xffffffffu, page, p) * a.c.heads + h) << a.c.page_shift;
          const uint8_t *k = a.c.k_pages + row * S::K_ROW, *v = a.c.v_pages + row * S::V_ROW;
          if (!PAGED_CHECK(a.c.status, h >= 0 && h < a.c.heads && at + per <= U && rows_exist(a.c, row, per))) continue;
#pragma unroll 1
          for (int i = lane * 16; i < per * S::K_ROW; i += 512) copy_16(to + at * S::K_ROW + i - lane * 16, k + i);
#pragma unroll 1
          for (int i = lane * 16; i < per * S::V_ROW; i += 512) copy_16(to + U * S::K_ROW + at * S::V_ROW + i - lane * 16, v + i);
          if (norm_at < per * 4 && lane * 16 < 8 * U) copy_16(to + U * (S::K_ROW + S::V_ROW) + at * 4, norms + row * 4 + norm_at);
        }
      }
    }
    if (!more) return;
    if (++u == nu) {
      u = 0;
      if (++pass == a.passes) {
        pass = 0;
        if (++h == a.c.heads) {
          h = 0;
          do len = ++b < a.n_seqs ? clipped_length(a, b, false) : 0; while (len == 0 && b < a.n_seqs);
          b = min(b, a.n_seqs - 1); // see start()
          nu = (len + U - 1) / U;
        }
      }
    }
    find_pages(a);
  }
};

template <int KB, int VB, int P, int MODE>
__global__ void __launch_bounds__(AttendShape<KB, VB, P, MODE>::THREADS, 1) paged_attend_kernel(const AttendLaunch a) {
  using S = AttendShape<KB, VB, P, MODE>;
  uint8_t *smem = attend_smem;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  int4 *desc = reinterpret_cast<int4 *>(smem + S::DESC) + 2 * warp;
  int4 *headers = reinterpret_cast<int4 *>(smem + S::HEADERS);
  const int per_seq = a.c.heads * a.passes, ring = S::RING + warp * 2 * S::STAGE;
  griddep_launch_dependents(); // paged_join_kernel waits for this grid's end itself

  AttendWalk<S> walk;
  const int units = walk.start(a, warp, lane);
  if (units > 0) walk.fetch(a, ring, desc, units > 1);
  fill_table<KB, S::EXACT>(smem + S::K_TABLE, tid, S::THREADS);
  if constexpr (KB != VB) fill_table<VB, S::EXACT>(smem + S::V_TABLE, tid, S::THREADS);
  AttendWarp<KB, VB, P, MODE> w;
  w.init(lane);
  __syncthreads();
  griddep_wait(); // for paged_query_kernel
  float *slots = a.warp_slots + (size_t)(blockIdx.x * S::WARPS + warp) * 2 * slot_floats(a.slot_cols, P);
  int flags = 0, item0 = 0, item1 = 0;
  bool from_start = true, fresh = true, handed = false;
  for (int i = 0; i < units; ++i) {
    const int stage = ring + (i & 1) * S::STAGE;
    copies_done();
    __syncwarp();
    if (i + 1 < units) walk.fetch(a, ring + (~i & 1) * S::STAGE, desc + (~i & 1), i + 2 < units);
    const int4 d = desc[i & 1];
    const int h = d.y & 0xffff, pass = d.y >> 16, item = d.x * per_seq + h * a.passes + pass;
    if (fresh) {
      from_start = (d.z & 0x3fffffff) == 0;
      fresh = handed = false;
      w.load_queries(a, item);
    }
    if (d.w > 0) w.unit(stage, d.w);
    const bool ends = d.z & 0x40000000;
    const bool stops = ends || i + 1 == units;
    if (__builtin_expect(!stops && d.z % w.KEEP == w.KEEP - 1, 0)) {
      float *place = a.warp_sums + (size_t)(blockIdx.x * S::WARPS + warp) * S::SUMS;
      if (PAGED_CHECK(a.c.status, in_workspace(a, place, S::SUMS))) {
        w.hand_over(place, handed);
        handed = true;
      }
    } else if (stops) {
      if (handed) w.take_back(a.warp_sums + (size_t)(blockIdx.x * S::WARPS + warp) * S::SUMS);
      const bool whole = ends && from_start;
      const int slot = from_start ? 1 : 0;
      w.finish(a, d.x, h, pass, min(S::COLS, a.group - pass * S::COLS), whole, slots + slot * slot_floats(a.slot_cols, P),
               reinterpret_cast<float *>(smem + stage));
      if (!whole) {
        if (slot == 0) { flags |= SEG_FROM_BEFORE | (ends ? SEG_ENDS : 0); item0 = item; }
        else { flags |= SEG_OPEN; item1 = item; }
      }
      fresh = true;
    }
    __syncwarp(); // the stage is free
  }
  if (lane == 0) headers[warp] = make_int4(flags, item0, item1, 0);
  __syncthreads();

  // join what this block's warps left
  int *n_chains = reinterpret_cast<int *>(smem + S::BLOCK);
  JoinChain *chains = reinterpret_cast<JoinChain *>(smem + S::BLOCK + 16);
  if (tid == 0) {
    int n = 0, open = -1, bflags = 0, bitem0 = 0, bitem1 = 0;
    for (int k = 0; k < S::WARPS; ++k) {
      const int4 hd = headers[k];
      if (hd.x & SEG_FROM_BEFORE) {
        if (open < 0) { open = n++; chains[open] = JoinChain{k, 0, 0, hd.y, 1}; bflags |= SEG_FROM_BEFORE; bitem0 = hd.y; }
        chains[open].count = k - chains[open].first + 1;
        if (hd.x & SEG_ENDS) {
          if (chains[open].kind == 1) bflags |= SEG_ENDS; else chains[open].kind = 0;
          open = -1;
        }
      }
      if (hd.x & SEG_OPEN) { open = n++; chains[open] = JoinChain{k, 1, 1, hd.z, 2}; }
    }
    if (open >= 0 && chains[open].kind == 2) { bflags |= SEG_OPEN; bitem1 = chains[open].item; }
    *n_chains = n;
    if (PAGED_CHECK(a.c.status, n <= S::WARPS + 1 && in_workspace(a, a.block_headers + blockIdx.x, 4))) a.block_headers[blockIdx.x] = make_int4(bflags, bitem0, bitem1, 0);
  }
  __syncthreads();
  const int n = *n_chains, sf = slot_floats(a.slot_cols, P);
  const float *first_slot = a.warp_slots + (size_t)blockIdx.x * S::WARPS * 2 * sf;
  for (int k = warp; k < n * a.slot_cols; k += S::WARPS) {
    const JoinChain ch = chains[k / a.slot_cols];
    const int col = k % a.slot_cols;
    if (col >= live_cols(a, ch.item, S::COLS)) continue;
    float v[P / 32], M, L;
    // its first piece lies in slot `slot`, the others in slot 0 of the warps behind; warps without units have none
    int count = 0;
    unsigned have = 0;
    for (int j = 0; j < ch.count; ++j)
      if (j == 0 || (headers[ch.first + j].x & SEG_FROM_BEFORE)) { have |= 1u << j; ++count; }
    auto piece = [&](int i) {
      unsigned left = have;
      for (int j = 0; j < i; ++j) left &= left - 1;
      const int j = __ffs(left) - 1;
      return first_slot + (size_t)(2 * (ch.first + j) + (j == 0 ? ch.slot : 0)) * sf;
    };
    join_pieces<P>(piece, count, 0, 1, a.slot_cols, col, lane, v, M, L);
    const int b = ch.item / per_seq, hp = ch.item - b * per_seq, h = hp / a.passes;
    if (ch.kind == 0) store_column<P>(a, b, h, (hp - h * a.passes) * S::COLS + col, lane, v, L);
    else {
      float *to = a.block_slots + (size_t)(2 * blockIdx.x + ch.kind - 1) * sf;
      if (!PAGED_CHECK(a.c.status, in_workspace(a, to, sf) && to + sf <= a.warp_slots)) continue;
#pragma unroll
      for (int i = 0; i < P / 32; ++i) to[col * P + lane * (P / 32) + i] = v[i];
      if (lane == 0) *reinterpret_cast<float2 *>(to + a.slot_cols * P + 2 * col) = make_float2(M, L);
    }
  }
}

// Items that span blocks: block (j, col) joins the item that block j of the grid above opened and left.
constexpr int JOIN_WARPS = 4;
template <int P> __global__ void __launch_bounds__(JOIN_WARPS * 32) paged_join_kernel(const AttendLaunch a, int blocks, int cols) {
  __shared__ float part[JOIN_WARPS][P + 1];
  for (int b = blockIdx.y * gridDim.x + blockIdx.x; b < a.n_seqs; b += gridDim.x * gridDim.y)
    if (clipped_length(a, b, false) == 0) { // nothing to attend to: zeros
      const int dim = a.c.dim;
      for (int i = threadIdx.x; i < a.c.heads * a.group * dim; i += JOIN_WARPS * 32)
        store_one(a.out, (long long)b * a.out_seq + (long long)(i / dim) * a.out_head + i % dim, a.type, 0.f);
    }
  griddep_wait();
  const int j = blockIdx.x, col = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int4 mine = a.block_headers[j];
  if (!(mine.x & SEG_OPEN) || col >= live_cols(a, mine.z, cols)) return;
  // pieces: block j's, then those of the blocks behind it up to the one in which the item ends
  int last = j;
  for (int k = j + 1; k < blocks; k += 32) {
    const int f = k + lane < blocks ? a.block_headers[k + lane].x : 0;
    const unsigned ends = __ballot_sync(0xffffffffu, f & SEG_ENDS);
    if (ends) { last = k + __ffs(ends) - 1; break; }
  }
  const int sf = slot_floats(a.slot_cols, P);
  const int pieces = last - j + 1;
  auto piece = [&](int i) { return a.block_slots + (size_t)(2 * (j + i) + (i == 0)) * sf; };
  if (!PAGED_CHECK(a.c.status, last < blocks && mine.z >= 0 && mine.z < a.n_seqs * a.c.heads * a.passes)) return;
  constexpr int E = P / 32;
  float v[E], M, L;
  join_pieces<P>(piece, pieces, warp, JOIN_WARPS, a.slot_cols, col, lane, v, M, L);
#pragma unroll
  for (int i = 0; i < E; ++i) part[warp][lane * E + i] = v[i];
  if (lane == 0) part[warp][P] = L;
  __syncthreads();
  if (warp) return;
#pragma unroll
  for (int i = 0; i < E; ++i)
    for (int k = 1; k < JOIN_WARPS; ++k) v[i] += part[k][lane * E + i];
  for (int k = 1; k < JOIN_WARPS; ++k) L += part[k][P];
  const int per_seq = a.c.heads * a.passes, b = mine.z / per_seq, hp = mine.z - b * per_seq, h = hp / a.passes;
  store_column<P>(a, b, h, (hp - h * a.passes) * cols + col, lane, v, L);
}

} // namespace aq
