// A paged KV cache held in 4 bits (`int4.cuh`): new tokens are quantised into it, and one new token a sequence attends to it.
//
// Pools: codes [pages, Nkv, page_size, H / 2], pairs (s, m) [pages, Nkv, page_size, H / 32, 2] in bf16, for K and for V, so
// that a head's rows of a page are one run of memory; page table [B, max_pages], H 64 or 128.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <float.h>
#include <math.h>
#include <stdint.h>

#include "cache_rows.cuh"
#include "chain.cuh"
#include "cluster.cuh"
#include "int4.cuh"
#include "mma_sync.cuh"
#include "status.cuh"

namespace axb {

struct Int4Pool {
  uint8_t* codes;
  uint32_t* pairs;
};

struct Int4AppendParams {
  HeadRows q, k, v;
  __nv_bfloat16 *q_out, *k_out, *v_out;  // where the rotated q and the values of k and v go; null: not wanted
  int64_t out_b, out_t, out_h;
  Int4Pool k_pool, v_pool;
  const int* page_table;
  const int* start;     // null: 0
  const int* live;      // null: all tokens
  const float2* angle;  // (sin, cos) of [position][H / 2] for positions 0 to T - 1 (`start` is null); null: nothing is rotated
  int* status;
  FastDiv heads, tokens, page;  // units of a token, tokens of a sequence, positions of a page
  uint32_t units;
  int kv_units;                 // of a token
  int num_q_heads, num_kv_heads, max_pages, num_pages;
};

// The eight dims 8 l .. 8 l + 7 of a lane, groups of 32 dims are four neighbouring lanes: codes (dim i in bits 4 i), pair and the
// codes as floats.
//
// Level d / s to the nearest, ties to even.  A product with the reciprocal is within 2^-22 of the quotient, so its rounding is
// right unless it ends next to a half; there (one warp in forty on normal values) d - c s, which is exact (c s has 12 bits),
// tells whether a neighbour is nearer.  That is the rounding of the 32-bit quotient, too: a d that is not (k + 1/2) s is off
// it by more than half a unit of the quotient.  No level passes 15: s is at least 1 - 2^-8 of a fifteenth of the range.
__device__ __forceinline__ uint32_t quantize8(const uint4& x, uint32_t& pair, float (&level)[8]) {
  const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&x);
  __nv_bfloat162 lo2 = __hmin2_nan(__hmin2_nan(h[0], h[1]), __hmin2_nan(h[2], h[3]));
  __nv_bfloat162 hi2 = __hmax2_nan(__hmax2_nan(h[0], h[1]), __hmax2_nan(h[2], h[3]));
#pragma unroll
  for (int off = 1; off <= 2; off <<= 1) {
    lo2 = __hmin2_nan(lo2, __shfl_xor_sync(0xffffffffu, lo2, off));
    hi2 = __hmax2_nan(hi2, __shfl_xor_sync(0xffffffffu, hi2, off));
  }
  const float lo = __bfloat162float(__hmin_nan(lo2.x, lo2.y)), hi = __bfloat162float(__hmax_nan(hi2.x, hi2.y));
  const float range = hi - lo;
  const bool good = range <= FLT_MAX;  // neither NaN nor an infinity nor an overflow
  float s = __bfloat162float(__float2bfloat16(range * (1.f / 15.f)));
  if (!good || s < FLT_MIN) s = 0.f;
  pair = (__float_as_uint(s) >> 16) | (good ? __float_as_uint(lo) : 0x7fff0000u);
  const float inverse = s == 0.f ? 0.f : __frcp_rn(s);
  constexpr float kWhole = 12582912.f;  // 1.5 * 2^23: whole numbers are the last bits
  float off_by = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float2 f = __bfloat1622float2(h[i >> 1]);
    const float t = ((i & 1 ? f.y : f.x) - lo) * inverse;
    level[i] = (t + kWhole) - kWhole;
    off_by = fmaxf(off_by, fabsf(t - level[i]));
  }
  if (__any_sync(0xffffffffu, off_by > 0.5f - 0x1p-16f)) {
    const float half = 0.5f * s;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float2 f = __bfloat1622float2(h[i >> 1]);
      const float rest = fmaf(-level[i], s, (i & 1 ? f.y : f.x) - lo);
      const bool odd = static_cast<int>(level[i]) & 1;
      if (rest > half || (rest == half && odd)) level[i] += 1.f;
      if (rest < -half || (rest == -half && odd)) level[i] -= 1.f;
    }
  }
  if (s == 0.f) {  // (a NaN among the values is one among the levels)
#pragma unroll
    for (int i = 0; i < 8; ++i) level[i] = 0.f;
  }
  const float a = fmaf(level[3], 4096.f, fmaf(level[2], 256.f, fmaf(level[1], 16.f, level[0])));
  const float b = fmaf(level[7], 4096.f, fmaf(level[6], 256.f, fmaf(level[5], 16.f, level[4])));
  return __byte_perm(__float_as_uint(a + kWhole), __float_as_uint(b + kWhole), 0x5410);
}

__device__ __forceinline__ uint4 values8(const float (&level)[8], uint32_t pair) {
  const float s = pair_s(pair), m = pair_m(pair);
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = pack2(fmaf(s, level[2 * i], m), fmaf(s, level[2 * i + 1], m));
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// The four bytes that a lane stores of a row, and where: lanes of neighbouring groups swap halves, so that each has the
// same chunk of two groups.  `lane`: within the row (H / 8 lanes).
template <int H>
__device__ __forceinline__ uint32_t row_word(uint32_t codes, int lane, int& byte) {
  constexpr int G = H / kInt4Group;
  const int g = lane >> 2, sub = lane & 3;
  const uint32_t other = __shfl_xor_sync(0xffffffffu, codes, 4);
  byte = (2 * sub + (g & 1)) * (2 * G) + (g >> 1) * 4;
  return g & 1 ? __byte_perm(other, codes, 0x7632) : __byte_perm(codes, other, 0x5410);
}

constexpr int kAppendThreads = 256;

// A unit is the key and the value of kHeads KV heads of one token, or twice as many of its query heads to be rotated: H / 8
// lanes with 16 bytes of each row.  Units run over heads (KV, then q), tokens, sequences.  The pass is bound by its
// instructions: where rows go is found once for all of a unit, and nothing is quantised behind `live`.  Measured with the values
// written out as well, heads of 128 (us; at the copy rate): 64 x 1 tokens, 32 KV heads, 3.2 (0.4), a launch; 8 x up to 2048
// tokens, 8 KV heads, 26.4 (17.5; issue 71%, ALU 53%); 28.0 with a head a unit, and 64 with a row a unit, a 64-bit division for
// each of its indexes and an IEEE division for each level.  Prompts with 32 query heads to be rotated beside 8 (32) KV heads, 8 x
// 2048: 71 (65) and 171 (136).
template <int H, int kHeads>
__global__ void __launch_bounds__(kAppendThreads)
int4_append_kernel(Int4AppendParams p) {
  chain_link();
  constexpr int kLanes = H / 8, kUnits = kAppendThreads / kLanes;
  const int lane = threadIdx.x % kLanes;
  const uint4 zeros = make_uint4(0, 0, 0, 0);
  for (uint32_t unit0 = blockIdx.x * kUnits; unit0 < p.units; unit0 += gridDim.x * kUnits) {
    const uint32_t unit = unit0 + threadIdx.x / kLanes;  // (shuffles: all lanes stay)
    const bool inside = unit < p.units;
    const uint32_t token = inside ? p.heads.div(unit) : 0;
    const int group = inside ? static_cast<int>(unit - token * p.heads.d) : 0;
    const int b = static_cast<int>(p.tokens.div(token)), t = static_cast<int>(token - b * p.tokens.d);
    const bool live = inside && (p.live == nullptr || t < p.live[b]);
    const bool is_q = group >= p.kv_units;
    const int head = is_q ? 2 * kHeads * (group - p.kv_units) : kHeads * group;
    const int rows = is_q ? p.num_q_heads - head : 2 * (p.num_kv_heads - head);  // (more than a unit's, too)
    const int64_t out_at = b * p.out_b + t * p.out_t + head * p.out_h + lane * 8;
    if (!__any_sync(0xffffffffu, live)) {
      if (inside && !is_q && p.k_out != nullptr) {
#pragma unroll
        for (int i = 0; i < kHeads; ++i) {
          if (2 * i >= rows) break;
          *reinterpret_cast<uint4*>(p.k_out + out_at + i * p.out_h) = zeros;
          *reinterpret_cast<uint4*>(p.v_out + out_at + i * p.out_h) = zeros;
        }
      }
      continue;
    }
    uint4 x[kHeads][2];
    {
      const HeadRows& first = is_q ? p.q : p.k;
      const HeadRows& second = is_q ? p.q : p.v;
      const __nv_bfloat16* src = first.x + b * first.b + t * first.t + head * first.h + lane * 8;
      const __nv_bfloat16* other = second.x + b * second.b + t * second.t + (head + is_q) * second.h + lane * 8;
#pragma unroll
      for (int i = 0; i < kHeads; ++i) {
        x[i][0] = live && 2 * i < rows ? *reinterpret_cast<const uint4*>(src) : zeros;
        x[i][1] = live && 2 * i + 1 < rows ? *reinterpret_cast<const uint4*>(other) : zeros;
        src += first.h << is_q;
        other += second.h << is_q;
      }
    }
    const int pos = (p.start == nullptr ? 0 : p.start[b]) + t;
    if (live && p.angle != nullptr) {
      const float2* angle = p.angle + static_cast<int64_t>(pos) * (H / 2) + lane * 4;
#pragma unroll
      for (int i = 0; i < kHeads; ++i) {
        x[i][0] = rotate8(x[i][0], angle);
        if (is_q) x[i][1] = rotate8(x[i][1], angle);
      }
    }
    if (is_q && live) {
#pragma unroll
      for (int i = 0; i < 2 * kHeads; ++i)
        if (i < rows) *reinterpret_cast<uint4*>(p.q_out + out_at + i * p.out_h) = x[i >> 1][i & 1];
    }
    const bool quantised = live && !is_q;
    if (!__any_sync(0xffffffffu, quantised)) continue;
    int64_t slot = -1;  // of the first head; the next one's is a page's rows further
    if (quantised) {
      const int col = static_cast<int>(p.page.div(static_cast<uint32_t>(max(pos, 0))));
      const uint32_t page = pos >= 0 && col < p.max_pages
                                ? static_cast<uint32_t>(p.page_table[static_cast<int64_t>(b) * p.max_pages + col]) : 0xffffffffu;
      const int page_size = static_cast<int>(p.page.d);
      if (page < static_cast<uint32_t>(p.num_pages))
        slot = (static_cast<int64_t>(page) * p.num_kv_heads + head) * page_size + (pos - col * page_size);
      else
        report_bad_argument(p.status);
    }
#pragma unroll
    for (int i = 0; i < kHeads; ++i) {
      uint32_t k_pair, v_pair;
      float k_level[8], v_level[8];
      int byte;
      const uint32_t k_word = row_word<H>(quantize8(x[i][0], k_pair, k_level), lane, byte);
      const uint32_t v_word = row_word<H>(quantize8(x[i][1], v_pair, v_level), lane, byte);
      if (2 * i >= rows) continue;
      if (inside && !is_q && p.k_out != nullptr) {
        *reinterpret_cast<uint4*>(p.k_out + out_at + i * p.out_h) = live ? values8(k_level, k_pair) : zeros;
        *reinterpret_cast<uint4*>(p.v_out + out_at + i * p.out_h) = live ? values8(v_level, v_pair) : zeros;
      }
      if (slot < 0) continue;
      const int64_t at = slot + i * static_cast<int64_t>(p.page.d);
      *reinterpret_cast<uint32_t*>(p.k_pool.codes + at * (H / 2) + byte) = k_word;
      *reinterpret_cast<uint32_t*>(p.v_pool.codes + at * (H / 2) + byte) = v_word;
      if ((lane & 3) == 0) {
        p.k_pool.pairs[at * (H / kInt4Group) + (lane >> 2)] = k_pair;
        p.v_pool.pairs[at * (H / kInt4Group) + (lane >> 2)] = v_pair;
      }
    }
  }
}

struct Int4AttnParams {
  const __nv_bfloat16* q;  // [B, Nq, H]; kAppend: the packed projection [B, Nq + 2 Nkv, H] of the new token, not rotated
  const float2* angle;     // kAppend: (sin, cos) of [position][H / 2]
  Int4Pool k_pool, v_pool;
  const int* page_table;
  const int* lengths;
  float* part_out;         // [B, Nq, splits / 8, H]: of each cluster, where there are several
  float* part_ml;          // [B, Nq, splits / 8, 2]
  __nv_bfloat16* out;
  int* status;
  int num_q_heads, num_kv_heads, page_size, page_shift, max_pages, num_pages, splits;  // page_shift: -1 where no power of two
  int angle_rows;
  float scale_log2;      // softmax scale * log2(e) * kInt4Back, > 0
};

constexpr int kAttnThreads = 128, kAttnWarps = kAttnThreads / 32;
constexpr int kAttnRows = 8;   // query heads of a CTA: the columns of the second product
constexpr int kAttnKeys = 32;  // keys of a tile
constexpr int kAttnStages = 2;
constexpr int kAttnCluster = 8;

template <int H>
struct Int4Tile {
  static constexpr int kGroups = H / kInt4Group;
  static constexpr int kRow = H / 2, kPairs = 16;                 // bytes of a key's codes and pairs (8 of 16 where H is 64)
  static constexpr int kK = 0, kV = kAttnKeys * kRow, kKPairs = 2 * kV, kVPairs = kKPairs + kAttnKeys * kPairs;
  static constexpr int kBytes = kVPairs + kAttnKeys * kPairs;
  static constexpr int kSmem(int rows) {
    const int merge = (kAttnWarps + 1) * rows * (H + 2) * 4, tiles = kAttnWarps * kAttnStages * kBytes;
    return merge > tiles ? merge : tiles;
  }
  // 16-byte unit u of V's row `key`: units are swapped so that eight lanes of four keys, every second one, hit all banks.
  __device__ static int v_unit(int key, int u) {
    if constexpr (H == 128) return (key >> 1) * 128 + ((((key & 1) * 4 + u) ^ (((key >> 1) & 3) << 1)) << 4);
    return (key >> 2) * 128 + ((((key & 3) * 2 + u) ^ (((key >> 2) & 1) << 1)) << 4);
  }
};

template <int N>
__device__ __forceinline__ void load_words(uint32_t (&w)[N], const uint8_t* src) {
  static_assert(N == 2 || N == 4, "8 or 16 bytes");
  if constexpr (N == 4) *reinterpret_cast<uint4*>(w) = *reinterpret_cast<const uint4*>(src);
  else *reinterpret_cast<uint2*>(w) = *reinterpret_cast<const uint2*>(src);
}

// d = a b + c.
__device__ __forceinline__ void mma_add(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, const float (&c)[4]) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
}

__device__ __forceinline__ uint32_t times(uint32_t x, __nv_bfloat162 f) {
  const __nv_bfloat162 y = __hmul2(reinterpret_cast<__nv_bfloat162&>(x), f);
  return reinterpret_cast<const uint32_t&>(y);
}

// Three bf16 terms each that add up to (x, y): 24 bits of mantissa, cut off from the top.
__device__ __forceinline__ void split_terms(float x, float y, uint32_t (&t)[3]) {
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    const uint32_t ux = __float_as_uint(x), uy = __float_as_uint(y);
    t[i] = __byte_perm(ux, uy, 0x7632);
    x -= __uint_as_float(ux & 0xffff0000u);
    y -= __uint_as_float(uy & 0xffff0000u);
  }
}

// An 8 x 8 tile of bf16 pairs, lane (r, c) with entries (r, 2c), (r, 2c + 1): its transpose in the same layout.
__device__ __forceinline__ uint32_t turned_round(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool ok) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(ok ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async8(uint32_t dst, const void* src, bool ok) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(dst), "l"(src), "r"(ok ? 8 : 0) : "memory");
}

// S^T = K Q^T: 16 keys are the rows of the m16n8k16 tile, the query heads its columns; a lane takes dims 8c .. 8c + 7 of each
// group of a key, and the sums of a group are multiplied by its s: k.q = sum_g s_g (sum c q) + m_g sum q.
// sum_g m_g sum q is one product of its own: the sums of q are three bf16 terms that add up to their 32 bits.
// O^T = V^T P^T: 16 dims of one group are the rows, the heads the columns.  P is rounded to bf16 as the operand of all
// products, as in the prompts' kernels, and normalised by the sum of what it was rounded to; turned round by `movmatrix` and
// multiplied by s of a key's group, it rounds again.  Values are small sums of large terms p m and p s c, so that this second
// rounding would count double against codes of 0 to 15: it counts against c - 8, since sums of the rounded and of the exact p s
// give back 8 times their difference.  The sums are products with P as the first operand, in registers as it lies, and pairs or
// ones as the second: with the roles of the large products they cost 26 register moves a tile (133 us for 127 below).  Two roundings of half a step, 2^-8 of
// a probability each; against 64 bits an output is off by up to 0.0020 of itself (2-norm; 4 to 64 keys, 0.0018 of 2000), 0.0017 of
// it the output's own rounding; without the shift by 8 up to 0.0029.
// Codes enter as denormal bf16 numbers (`int4.cuh`): scores carry 1 / kInt4Back until the exponential, probabilities and the
// sums of them alone kInt4Scale, and the sums of p c 1 / kInt4Back.
// The maximum that probabilities are relative to moves only when a score passes it by kSlack (a factor of 2^kSlack).
//
// A tile is 32 keys, a warp's own from `cp.async` to its sums: no barrier before the end.  Tiles go round the warps of all
// splits, splits of eight or less are a cluster whose parts meet in distributed shared memory, more are clusters whose
// parts a second launch joins.  Measured (us; at the copy rate): 64 sequences of 2000 tokens, 32 KV heads of 128, 127 (100.3);
// 16 x 2048, 8 KV heads for 32, 14.5 (3.3), of which a CTA's start and end are about 4 and the launch 2; 1 x 130001, 8 KV heads
// for 32, 47.4 (25.4).  Instructions bind the pass (600 a tile and warp, two thirds of the ALU pipe's unpack codes), not the
// copies; the first case without the shift of the codes by 8: 125, without arithmetic 97, without
// copies 106 (issue 59%, ALU 56%, tensor cores 28%), with 96 registers and five CTAs an SM 149, with shifts on the FMA pipe 132.
// Heads of 128 take all 128 registers that four CTAs an SM leave, and spill 4 to 28 bytes; heads of 64 up to 117.
//
// kAppend: a decoding step in one launch.  A warp turns its query heads in registers; the warp whose tile holds the new token
// turns its key, quantises key and value, stores them in their page slot and puts them into the tile itself, so nobody reads
// the slot.  The cases above take 137, 15.6 and 48.4 that way.
constexpr float kSlack = 8.f;

template <int H, bool kCluster, bool kAppend>
__global__ void __launch_bounds__(kAttnThreads, 4)
int4_attn_kernel(Int4AttnParams p) {
  chain_link();
  using Tile = Int4Tile<H>;
  constexpr int G = Tile::kGroups;
  extern __shared__ __align__(128) uint8_t s_ring[];
  const int split = blockIdx.x;
  const int group = p.num_q_heads / p.num_kv_heads;
  const int parts = (group + kAttnRows - 1) / kAttnRows;
  const int kvh = blockIdx.y / parts;
  const int first = blockIdx.y % parts * kAttnRows;
  const int rows = min(kAttnRows, group - first);
  const int qh0 = kvh * group + first;
  const int b = blockIdx.z;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int r = lane >> 2, c = lane & 3;
  int len = p.lengths[b];
  // Tiles go to the warps of all splits in turn, so which pages a warp needs does not depend on the length.
  const int step = kAttnWarps * p.splits;
  int tile = split * kAttnWarps + warp;
  if (len > p.max_pages * static_cast<int64_t>(p.page_size) || (kAppend && len > p.angle_rows)) {
    if (threadIdx.x == 0) report_bad_argument(p.status);
    len = kAppend ? 0 : p.max_pages * p.page_size;  // a new token without a place or a rotation: nothing is appended
  }
  const int hi = (max(len, 0) + kAttnKeys - 1) / kAttnKeys;
  const int* table = p.page_table + static_cast<int64_t>(b) * p.max_pages;

  // Key `lane` of a tile: its page, asked for long before `row_of` makes it the row of the pools; kNone beyond the sequence
  // (the launcher keeps rows below it).
  constexpr uint32_t kNone = 0xffffffffu;
  const int cached = kAppend ? len - 1 : len;
  auto col_of = [&](int t) { return p.page_shift >= 0 ? t >> p.page_shift : t / p.page_size; };
  auto page_of = [&](int tile) -> uint32_t {
    const int col = col_of(tile * kAttnKeys + lane);
    return col < p.max_pages ? static_cast<uint32_t>(table[col]) : 0u;
  };
  auto row_of = [&](int tile, uint32_t page) -> uint32_t {
    const int t = tile * kAttnKeys + lane;
    if (tile >= hi || t >= cached) return kNone;
    if (page >= static_cast<uint32_t>(p.num_pages)) {
      report_bad_argument(p.status);
      return kNone;
    }
    return (page * p.num_kv_heads + kvh) * p.page_size + (t - col_of(t) * p.page_size);
  };
  uint8_t* ring = s_ring + warp * kAttnStages * Tile::kBytes;
  constexpr int kUnits = Tile::kRow / 16, kKeys = 32 / kUnits;  // 16-byte units of a row, keys an instruction
  const uint32_t k_dst = sptr(ring) + Tile::kK + lane * 16;
  const uint32_t v_dst = sptr(ring) + Tile::kV + Tile::v_unit(lane / kUnits, lane % kUnits);
  const uint32_t pair_dst = sptr(ring) + Tile::kKPairs + lane * Tile::kPairs;
  const uint8_t* k_src = p.k_pool.codes + lane % kUnits * 16;
  const uint8_t* v_src = p.v_pool.codes + lane % kUnits * 16;
  auto load_tile = [&](int stage, uint32_t slot) {
    const uint32_t at_stage = stage * Tile::kBytes;
    // Keys that are not there have pairs of zeros; their codes, finite whatever they are, come from the first row.
    const bool ok = slot != kNone;
    const uint32_t row = ok ? slot : 0u;
#pragma unroll
    for (int i = 0; i < kUnits; ++i) {
      const uint64_t off = static_cast<uint64_t>(__shfl_sync(0xffffffffu, row, i * kKeys + lane / kUnits)) * Tile::kRow;
      cp_async16(k_dst + at_stage + i * 512, k_src + off);
      cp_async16(v_dst + at_stage + i * 512, v_src + off);
    }
    const uint64_t off = static_cast<uint64_t>(row) * G;
    if constexpr (G == 4) {
      cp_async16(pair_dst + at_stage, p.k_pool.pairs + off, ok);
      cp_async16(pair_dst + at_stage + kAttnKeys * Tile::kPairs, p.v_pool.pairs + off, ok);
    } else {
      cp_async8(pair_dst + at_stage, p.k_pool.pairs + off, ok);
      cp_async8(pair_dst + at_stage + kAttnKeys * Tile::kPairs, p.v_pool.pairs + off, ok);
    }
  };
  uint32_t pages[kAttnStages + 1];
#pragma unroll
  for (int i = 0; i <= kAttnStages; ++i) pages[i] = page_of(tile + i * step);
#pragma unroll
  for (int i = 0; i < kAttnStages; ++i) {
    if (tile + i * step < hi) load_tile(i, row_of(tile + i * step, pages[i]));
    cp_commit();
  }
  uint32_t page = pages[kAttnStages];
  const int q_heads = kAppend ? p.num_q_heads + 2 * p.num_kv_heads : p.num_q_heads;  // of a row of q
  const int pos = len - 1;
  // The new token: lane l of the first H / 8 has dims 8 l .. 8 l + 7 of its key, the next H / 8 lanes its value.
  const int new_tile = pos / kAttnKeys;
  const bool appends = kAppend && len > 0 && new_tile % step == tile;
  const float2* angle = nullptr;
  uint32_t new_word = 0, new_pair = 0;
  int new_byte = 0;
  constexpr int kRowLanes = H / 8;
  if constexpr (kAppend) {
    angle = p.angle + static_cast<int64_t>(max(0, pos)) * (H / 2);
    if (appends) {
      const int is_v = lane / kRowLanes & 1, l8 = lane % kRowLanes;
      uint4 x = *reinterpret_cast<const uint4*>(
          p.q + (static_cast<int64_t>(b) * q_heads + p.num_q_heads + is_v * p.num_kv_heads + kvh) * H + l8 * 8);
      if (!is_v) x = rotate8(x, angle + l8 * 4);
      float level[8];
      new_word = row_word<H>(quantize8(x, new_pair, level), l8, new_byte);
      const uint32_t to = static_cast<uint32_t>(table[col_of(pos)]);
      if (to >= static_cast<uint32_t>(p.num_pages)) {
        report_bad_argument(p.status);
      } else if (first == 0 && lane < 2 * kRowLanes) {  // (the other parts of a large group have the same)
        const int64_t slot =
            (static_cast<int64_t>(to) * p.num_kv_heads + kvh) * p.page_size + (pos - col_of(pos) * p.page_size);
        const Int4Pool& pool = is_v ? p.v_pool : p.k_pool;
        *reinterpret_cast<uint32_t*>(pool.codes + slot * (H / 2) + new_byte) = new_word;
        if ((l8 & 3) == 0) pool.pairs[slot * G + (l8 >> 2)] = new_pair;
      }
    }
  }

  // Q of head r in the order of K's codes: MMA i of group g takes dims 8c + 2i, 8c + 2i + 4 and the two behind them, whose
  // codes are 16 times as large.
  uint32_t qb[2 * G][2];
  float sums[G];
  const __nv_bfloat162 even = __float2bfloat162_rn(kInt4Scale), odd = __float2bfloat162_rn(kInt4Scale / 16.f);
#pragma unroll
  for (int g = 0; g < G; ++g) {
    uint4 x = make_uint4(0, 0, 0, 0);
    if (r < rows)
      x = *reinterpret_cast<const uint4*>(p.q + (static_cast<int64_t>(b) * q_heads + qh0 + r) * H + g * 32 + c * 8);
    if constexpr (kAppend) x = rotate8(x, angle + g * 16 + c * 4);
    const float2 f0 = unpack2(x.x), f1 = unpack2(x.y), f2 = unpack2(x.z), f3 = unpack2(x.w);
    float sum = ((f0.x + f0.y) + (f1.x + f1.y)) + ((f2.x + f2.y) + (f3.x + f3.y));
    sum += __shfl_xor_sync(0xffffffffu, sum, 1);
    sum += __shfl_xor_sync(0xffffffffu, sum, 2);
    sums[g] = sum * (1.f / kInt4Back);
    qb[2 * g][0] = times(__byte_perm(x.x, x.z, 0x5410), even);
    qb[2 * g][1] = times(__byte_perm(x.x, x.z, 0x7632), odd);
    qb[2 * g + 1][0] = times(__byte_perm(x.y, x.w, 0x5410), even);
    qb[2 * g + 1][1] = times(__byte_perm(x.y, x.w, 0x7632), odd);
  }

  // Column k of that product is term k / G of the sum of group k % G, for two neighbours k = 2c and two k = 8 + 2c.
  uint32_t qm[2];
  {
    uint32_t terms[3][G / 2];
#pragma unroll
    for (int g = 0; g < G; g += 2) {
      uint32_t t[3];
      split_terms(sums[g], sums[g + 1], t);
#pragma unroll
      for (int i = 0; i < 3; ++i) terms[i][g / 2] = t[i];
    }
    if constexpr (G == 4) {
      qm[0] = c == 0 ? terms[0][0] : c == 1 ? terms[0][1] : c == 2 ? terms[1][0] : terms[1][1];
      qm[1] = c == 0 ? terms[2][0] : c == 1 ? terms[2][1] : 0u;
    } else {
      qm[0] = c == 0 ? terms[0][0] : c == 1 ? terms[1][0] : c == 2 ? terms[2][0] : 0u;
      qm[1] = 0u;
    }
  }

  float m[2] = {-INFINITY, -INFINITY};  // heads 2c, 2c + 1
  const float slack = kSlack / p.scale_log2;
  float acc[2 * G][4];  // [group, half][dim 32 g + 4 r + 2 half (+ 1: entries 2, 3)][columns 2c, 2c + 1]
  // P as the first operand: its four registers are keys 0 .. 7 and 16 .. 23 in rows 0 to 7, the other keys in rows 8 to 15.
  float acc_lo[4] = {}, acc_hi[4] = {};  // head r: sums of p s, p m of group c; over the first keys in entries 0, 1 of acc_lo, over
                                         // the others in entries 2, 3 of acc_hi (what is in the rest is not used)
  float acc_r[4] = {};                   // both rows together: sums of the rounded p s of groups 2c, 2c + 1; of p where c is 2
#pragma unroll
  for (int i = 0; i < 2 * G; ++i) acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.f;
  const float zero[4] = {0.f, 0.f, 0.f, 0.f};

  int stage = 0;
  for (; tile < hi; tile += step) {
    cp_wait_group<kAttnStages - 1>();
    __syncwarp();
    uint8_t* st = ring + stage * Tile::kBytes;
    if (appends && tile == new_tile) {
      const int row = pos % kAttnKeys, is_v = lane / kRowLanes & 1, l8 = lane % kRowLanes;
      if (lane < 2 * kRowLanes) {
        const int at = is_v ? Tile::kV + Tile::v_unit(row, new_byte >> 4) + (new_byte & 15) : Tile::kK + row * Tile::kRow + new_byte;
        *reinterpret_cast<uint32_t*>(st + at) = new_word;
        if ((l8 & 3) == 0)
          *reinterpret_cast<uint32_t*>(st + (is_v ? Tile::kVPairs : Tile::kKPairs) + row * Tile::kPairs + (l8 >> 2) * 4) = new_pair;
      }
      __syncwarp();
    }
    float s[4][2];  // keys 8 i + r, heads 2c, 2c + 1
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      uint32_t w[2][G], pairs[2][G], low[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int key = (2 * n + i) * 8 + r;
        load_words<G>(w[i], st + Tile::kK + key * Tile::kRow + c * (Tile::kRow / 4));
        load_words<G>(pairs[i], st + Tile::kKPairs + key * Tile::kPairs);
        uint32_t two[2];  // of groups 2 (c % 2) and the next
        load_words<2>(two, st + Tile::kKPairs + key * Tile::kPairs + (G == 4 ? (c & 1) * 8 : 0));
        low[i] = __byte_perm(two[0], two[1], 0x7632);
      }
      float dm[4];
      const uint32_t am[4] = {low[0], low[1], low[0], low[1]};
      mma_add(dm, am, qm[0], qm[1], zero);
#pragma unroll
      for (int i = 0; i < 4; ++i) s[2 * n + (i >> 1)][i & 1] = dm[i];
#pragma unroll
      for (int g = 0; g < G; ++g) {
        uint32_t x[2], y[2];  // dims 8c, + 1, + 4, + 5 and the two behind each pair
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          x[i] = __byte_perm(w[i][g >> 1], w[i][G / 2 + (g >> 1)], g & 1 ? 0x7632 : 0x5410);
          y[i] = __byte_perm(w[i][g >> 1], w[i][G / 2 + (g >> 1)], g & 1 ? 0x7733 : 0x5511);
        }
        float d[4];
        const uint32_t a0[4] = {int4_low(x[0]), int4_low(x[1]), int4_high(x[0]), int4_high(x[1])};
        const uint32_t a1[4] = {int4_low(y[0]), int4_low(y[1]), int4_high(y[0]), int4_high(y[1])};
        mma_add(d, a0, qb[2 * g][0], qb[2 * g][1], zero);
        mma_add(d, a1, qb[2 * g + 1][0], qb[2 * g + 1][1], d);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float ps = pair_s(pairs[i][g]);
#pragma unroll
          for (int h = 0; h < 2; ++h) s[2 * n + i][h] = fmaf(ps, d[2 * i + h], s[2 * n + i][h]);
        }
      }
    }
    if ((tile + 1) * kAttnKeys > len) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (tile * kAttnKeys + i * 8 + r >= len) s[i][0] = s[i][1] = -INFINITY;
    }
    float top[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) top[h] = fmaxf(fmaxf(s[0][h], s[1][h]), fmaxf(s[2][h], s[3][h]));
    if (__any_sync(0xffffffffu, top[0] > m[0] + slack || top[1] > m[1] + slack)) {
      float corr[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int off = 4; off <= 16; off <<= 1) top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], off));
        const float m_new = fmaxf(m[h], top[h]);
        corr[h] = m[h] == -INFINITY ? 0.f : ex2((m[h] - m_new) * p.scale_log2);  // (nothing is there yet)
        m[h] = m_new;
      }
      const float even = __shfl_sync(0xffffffffu, corr[0], r >> 1), odd = __shfl_sync(0xffffffffu, corr[1], r >> 1);
      const float of_row = r & 1 ? odd : even;
      acc_lo[0] *= of_row, acc_lo[1] *= of_row, acc_hi[2] *= of_row, acc_hi[3] *= of_row;
#pragma unroll
      for (int i = 0; i < 4; ++i) acc_r[i] *= of_row;
#pragma unroll
      for (int i = 0; i < 2 * G; ++i) {
        acc[i][0] *= corr[0];
        acc[i][1] *= corr[1];
        acc[i][2] *= corr[0];
        acc[i][3] *= corr[1];
      }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      // (a row of -inf alone keeps zeros; NaN stays)
      const float base = m[h] == -INFINITY ? 0.f : fmaf(-m[h], p.scale_log2, kInt4Shift);
#pragma unroll
      for (int i = 0; i < 4; ++i) s[i][h] = ex2(fmaf(s[i][h], p.scale_log2, base));
    }
    uint32_t pt[4], vt[4];  // rows: heads / entries of pairs; columns: keys 8 i + 2c, + 1 (vt: in the order 0, 2, 1, 3)
    ldsm4t(vt, st + Tile::kVPairs + (((lane & 8) << 1) + (lane >> 4 << 3) + (lane & 7)) * Tile::kPairs);
#pragma unroll
    for (int i = 0; i < 4; ++i) pt[i] = turned_round(pack2(s[i][0], s[i][1]));
    mma(acc_lo, pt, vt[0], vt[1]);
    mma(acc_hi, pt, vt[2], vt[3]);
    {
      const uint32_t one = r == 4 ? 0x3f803f80u : 0u;
      mma(acc_r, pt, one, one);
    }
    uint32_t w[8][G / 2];  // keys 8 i + 2c, + 1
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int key = (i >> 1) * 8 + 2 * c + (i & 1);
      if constexpr (G == 4)
        load_words<2>(w[i], st + Tile::kV + Tile::v_unit(key, r >> 1) + (r & 1) * 8);
      else
        w[i][0] = *reinterpret_cast<const uint32_t*>(st + Tile::kV + Tile::v_unit(key, r >> 2) + (r & 3) * 4);
    }
#pragma unroll
    for (int g = 0; g < G; ++g) {
      uint32_t pb[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t ps = __shfl_sync(0xffffffffu, vt[i >> 1 | (i & 1) << 1], 8 * g + c);  // row 2 g
        pb[i] = times(pt[i], reinterpret_cast<const __nv_bfloat162&>(ps));
      }
      const uint32_t one = r == g ? 0x3f803f80u : 0u;
      mma(acc_r, pb, one, one);
      uint32_t x[4], y[4];  // dims 4r, 4r + 1 and the two behind them of keys 8 i + 2c, + 1
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[i] = __byte_perm(w[2 * i][g >> 1], w[2 * i + 1][g >> 1], g & 1 ? 0x7632 : 0x5410);
        y[i] = __byte_perm(w[2 * i][g >> 1], w[2 * i + 1][g >> 1], g & 1 ? 0x7733 : 0x5511);
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t(&u)[4] = h ? y : x;
        const uint32_t a0[4] = {int4_low(u[0]), int4_high(u[0]), int4_low(u[1]), int4_high(u[1])};
        const uint32_t a1[4] = {int4_low(u[2]), int4_high(u[2]), int4_low(u[3]), int4_high(u[3])};
        mma(acc[2 * g + h], a0, pb[0], pb[1]);
        mma(acc[2 * g + h], a1, pb[2], pb[3]);
      }
    }
    __syncwarp();  // the stage has been read
    if (tile + kAttnStages * step < hi) load_tile(stage, row_of(tile + kAttnStages * step, page));
    cp_commit();
    page = page_of(tile + (kAttnStages + 1) * step);
    if (++stage == kAttnStages) stage = 0;
  }
  cp_wait_all();
  __syncthreads();  // the merge buffers overlay the tiles
  acc_lo[0] += acc_hi[2], acc_lo[1] += acc_hi[3], acc_r[0] += acc_r[2], acc_r[1] += acc_r[3];
  float* s_part = reinterpret_cast<float*>(s_ring);  // 4 warps and the CTA: [rows][H] sums, then maxima, then weights
  const int per_warp = rows * H;
  float* s_m = s_part + (kAttnWarps + 1) * per_warp;
  float* s_l = s_m + (kAttnWarps + 1) * rows;
#pragma unroll
  for (int n = 0; n < 2; ++n) {
    float* dst = s_part + warp * per_warp + (2 * c + n) * H + r * 4;
#pragma unroll
    for (int g = 0; g < G; ++g) {
      const int at = (2 * c + n) * 4;
      const float exact = __shfl_sync(0xffffffffu, acc_lo[0], at + g);
      const float rounded = __shfl_sync(0xffffffffu, acc_r[g & 1], at + (g >> 1));
      const float low = fmaf(-8.f, rounded - exact, __shfl_sync(0xffffffffu, acc_lo[1], at + g)) * (1.f / kInt4Scale);
      if (2 * c + n >= rows) continue;
#pragma unroll
      for (int h = 0; h < 2; ++h)
        *reinterpret_cast<float2*>(dst + g * 32 + 2 * h) = make_float2(fmaf(acc[2 * g + h][n], kInt4Back, low),
                                                                      fmaf(acc[2 * g + h][2 + n], kInt4Back / 16.f, low));
    }
    const float l = __shfl_sync(0xffffffffu, acc_r[0], (2 * c + n) * 4 + 2);
    if (r == 0 && 2 * c + n < rows) {
      s_m[warp * rows + 2 * c + n] = m[n] * p.scale_log2;
      s_l[warp * rows + 2 * c + n] = l * (1.f / kInt4Scale);
    }
  }
  __syncthreads();
  // Thread (g, d) of H threads a head owns output dim d.
  constexpr int kSets = kAttnThreads / H;
  const int d = threadIdx.x % H;
  for (int g = threadIdx.x / H; g < rows; g += kSets) {
    float mm = -INFINITY;
#pragma unroll
    for (int w = 0; w < kAttnWarps; ++w) mm = fmaxf(mm, s_m[w * rows + g]);
    float ll = 0.f, o = 0.f;
#pragma unroll
    for (int w = 0; w < kAttnWarps; ++w) {
      const float f = mm == -INFINITY ? 1.f : exp2f(s_m[w * rows + g] - mm);
      ll += s_l[w * rows + g] * f;
      o += s_part[w * per_warp + g * H + d] * f;
    }
    const int64_t row = static_cast<int64_t>(b) * p.num_q_heads + qh0 + g;
    if (p.splits == 1) {
      p.out[row * H + d] = __float2bfloat16(ll == 0.f ? 0.f : o / ll);
    } else {
      s_part[kAttnWarps * per_warp + g * H + d] = o;
      if (d == 0) {
        s_m[kAttnWarps * rows + g] = mm;
        s_l[kAttnWarps * rows + g] = ll;
      }
    }
  }
  if constexpr (kCluster) {
    const int cluster = min(p.splits, kAttnCluster), rank = split % cluster, parts = p.splits / cluster;
    cluster_sync_all();
    for (int g = rank * kSets + threadIdx.x / H; g < rows; g += cluster * kSets) {
      float mv[kAttnCluster], lv[kAttnCluster], ov[kAttnCluster];
#pragma unroll
      for (int s = 0; s < kAttnCluster; ++s) {
        const bool have = s < cluster;
        mv[s] = have ? ld_cluster_f32(sptr(s_m + kAttnWarps * rows + g), s) : -INFINITY;
        lv[s] = have ? ld_cluster_f32(sptr(s_l + kAttnWarps * rows + g), s) : 0.f;
        ov[s] = have ? ld_cluster_f32(sptr(s_part + kAttnWarps * per_warp + g * H + d), s) : 0.f;
      }
      float mm = -INFINITY;
#pragma unroll
      for (int s = 0; s < kAttnCluster; ++s) mm = fmaxf(mm, mv[s]);
      float ll = 0.f, o = 0.f;
#pragma unroll
      for (int s = 0; s < kAttnCluster; ++s) {
        const float f = mm == -INFINITY ? 1.f : exp2f(mv[s] - mm);
        ll += lv[s] * f;
        o += ov[s] * f;
      }
      const int64_t row = static_cast<int64_t>(b) * p.num_q_heads + qh0 + g;
      if (parts == 1) {
        p.out[row * H + d] = __float2bfloat16(ll == 0.f ? 0.f : o / ll);
      } else {
        const int64_t part = row * parts + split / cluster;
        p.part_out[part * H + d] = o;
        if (d == 0) *reinterpret_cast<float2*>(p.part_ml + part * 2) = make_float2(mm, ll);
      }
    }
    cluster_sync_all();  // a CTA's shared memory outlives its readers
  }
}

// The clusters' parts of a row, eight at a time on their way.
template <int H>
__global__ void __launch_bounds__(H)
int4_combine_kernel(const float* part_out, const float* part_ml, __nv_bfloat16* out, int parts) {
  chain_link();
  constexpr int kAtOnce = 8;
  const int64_t row = blockIdx.x;
  const int d = threadIdx.x;
  float mm = -INFINITY, ll = 0.f, o = 0.f;
  for (int s0 = 0; s0 < parts; s0 += kAtOnce) {
    float2 ml[kAtOnce];
    float ov[kAtOnce];
#pragma unroll
    for (int s = 0; s < kAtOnce; ++s) {
      const bool have = s0 + s < parts;
      ml[s] = have ? *reinterpret_cast<const float2*>(part_ml + (row * parts + s0 + s) * 2) : make_float2(-INFINITY, 0.f);
      ov[s] = have ? part_out[(row * parts + s0 + s) * H + d] : 0.f;
    }
    float top = mm;
#pragma unroll
    for (int s = 0; s < kAtOnce; ++s) top = fmaxf(top, ml[s].x);
    const float old = top == -INFINITY ? 1.f : exp2f(mm - top);
    ll *= old;
    o *= old;
#pragma unroll
    for (int s = 0; s < kAtOnce; ++s) {
      const float f = top == -INFINITY ? 1.f : exp2f(ml[s].x - top);
      ll += ml[s].y * f;
      o += ov[s] * f;
    }
    mm = top;
  }
  out[row * H + d] = __float2bfloat16(ll == 0.f ? 0.f : o / ll);
}

template <int H, bool kCluster, bool kAppend>
static int launch_int4_attn(const Int4AttnParams& p, dim3 grid, int rows, cudaStream_t stream) {
  constexpr auto kernel = int4_attn_kernel<H, kCluster, kAppend>;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim = {static_cast<unsigned>(p.splits < kAttnCluster ? p.splits : kAttnCluster), 1, 1};
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(kAttnThreads);
  cfg.dynamicSmemBytes = static_cast<size_t>(Int4Tile<H>::kSmem(rows));
  static_assert(Int4Tile<H>::kSmem(kAttnRows) <= 48 * 1024, "no opt-in");
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = static_cast<unsigned>(chain_attribute(attr, kCluster ? 1 : 0));
  return cudaLaunchKernelEx(&cfg, kernel, p) == cudaSuccess ? 0 : -4;
}

template <int H, bool kAppend>
static int int4_attn(const Int4AttnParams& p, int B, cudaStream_t stream) {
  const int g = p.num_q_heads / p.num_kv_heads;
  const bool cluster = p.splits > 1;
  const dim3 grid(p.splits, p.num_kv_heads * ((g + kAttnRows - 1) / kAttnRows), B);
  const int rows = g < kAttnRows ? g : kAttnRows;
  const int rc = cluster ? launch_int4_attn<H, true, kAppend>(p, grid, rows, stream)
                         : launch_int4_attn<H, false, kAppend>(p, grid, rows, stream);
  if (rc != 0) return rc;
  if (p.splits > kAttnCluster)
    launch_chained(int4_combine_kernel<H>, B * p.num_q_heads, H, 0, stream, p.part_out, p.part_ml, p.out,
                   p.splits / kAttnCluster);
  return cudaGetLastError() == cudaSuccess ? 0 : -4;
}

}  // namespace axb

namespace axb {

template <int H, int kHeads>
static int launch_int4_append(Int4AppendParams& p, int64_t tokens, cudaStream_t stream) {
  p.kv_units = (p.num_kv_heads + kHeads - 1) / kHeads;
  const int heads = p.kv_units + (p.num_q_heads + 2 * kHeads - 1) / (2 * kHeads);
  p.heads = FastDiv(heads);
  p.units = static_cast<uint32_t>(tokens * heads);
  constexpr int kPerCta = kAppendThreads / (H / 8);
  int64_t ctas = (tokens * heads + kPerCta - 1) / kPerCta;
  if (ctas > 148 * 32) ctas = 148 * 32;
  launch_chained(int4_append_kernel<H, kHeads>, static_cast<unsigned>(ctas), kAppendThreads, 0, stream, p);
  return cudaGetLastError() == cudaSuccess ? 0 : -4;
}

// Two KV heads a unit where units of one would be two waves or more and few units would be half empty (us with one / two: 8 x 2048
// tokens of 8 heads of 128 41.5 / 38.8, 1 x 2048 8.3 / 8.5, 64 x 1 of 32 3.2 / 3.9).
static int int4_append(Int4AppendParams& p, int B, int T, int page_size, int head_dim, cudaStream_t stream) {
  const int64_t tokens = static_cast<int64_t>(B) * T, rows = tokens * (2 * p.num_kv_heads + p.num_q_heads);
  if (rows >= (int64_t{1} << 31)) return -10;
  p.tokens = FastDiv(T), p.page = FastDiv(page_size);
  const bool two = rows / 2 * head_dim >= int64_t{148} * 4 * 2 * kAppendThreads * 8 &&
                   (p.num_kv_heads % 2 == 0 || p.num_kv_heads > 4);
  if (head_dim == 128) return two ? launch_int4_append<128, 2>(p, tokens, stream) : launch_int4_append<128, 1>(p, tokens, stream);
  return two ? launch_int4_append<64, 2>(p, tokens, stream) : launch_int4_append<64, 1>(p, tokens, stream);
}

}  // namespace axb

// k and v [B, T, Nkv, H] with element strides of (sequence, token, head); k_out and v_out (null: not wanted) are contiguous.
// -10: not supported.
extern "C" int axb_int4_append(const void* k, const void* v, int64_t k_b, int64_t k_t, int64_t k_h, int64_t v_b, int64_t v_t,
                               int64_t v_h, void* k_out, void* v_out, void* k_codes, void* k_pairs, void* v_codes,
                               void* v_pairs, const int* page_table, const int* start, const int* live, int B, int T,
                               int num_kv_heads, int head_dim, int page_size, int max_pages, int num_pages, int* status,
                               cudaStream_t stream) {
  using namespace axb;
  if ((head_dim != 64 && head_dim != 128) || page_size < 1 || num_kv_heads < 1 || B < 0 || T < 0 ||
      (k_b | k_t | k_h | v_b | v_t | v_h) % 8)
    return -10;
  for (const void* x : {k, v, static_cast<const void*>(k_out), static_cast<const void*>(v_out), static_cast<const void*>(k_codes),
                        static_cast<const void*>(k_pairs), static_cast<const void*>(v_codes), static_cast<const void*>(v_pairs)})
    if (!aligned16(x)) return -10;
  if (B == 0 || T == 0) return 0;
  Int4AppendParams p = {};
  p.k = {static_cast<const __nv_bfloat16*>(k), k_b, k_t, k_h};
  p.v = {static_cast<const __nv_bfloat16*>(v), v_b, v_t, v_h};
  p.k_out = static_cast<__nv_bfloat16*>(k_out);
  p.v_out = static_cast<__nv_bfloat16*>(v_out);
  p.out_h = head_dim, p.out_t = static_cast<int64_t>(num_kv_heads) * head_dim, p.out_b = T * p.out_t;
  p.k_pool = {static_cast<uint8_t*>(k_codes), static_cast<uint32_t*>(k_pairs)};
  p.v_pool = {static_cast<uint8_t*>(v_codes), static_cast<uint32_t*>(v_pairs)};
  p.page_table = page_table, p.start = start, p.live = live, p.status = status;
  p.num_kv_heads = num_kv_heads, p.max_pages = max_pages, p.num_pages = num_pages;
  return int4_append(p, B, T, page_size, head_dim, stream);
}

// Whole prompts from position 0: qkv [B, T, (Nq + 2 Nkv) * H] of one projection.  Queries and keys are rotated by `angle`
// ([position][H / 2] of (sin, cos), T positions or more), keys and values go to the cache, and what it then stands for
// replaces them in qkv.
extern "C" int axb_int4_append_prompt(void* qkv, void* k_codes, void* k_pairs, void* v_codes, void* v_pairs,
                                      const int* page_table, const float* angle, int angle_rows, int B, int T,
                                      int num_q_heads, int num_kv_heads, int head_dim, int page_size, int max_pages,
                                      int num_pages, int* status, cudaStream_t stream) {
  using namespace axb;
  if ((head_dim != 64 && head_dim != 128) || page_size < 1 || num_kv_heads < 1 || num_q_heads < 1 || B < 0 || T < 0 || angle_rows < T)
    return -10;
  for (const void* x : {static_cast<const void*>(qkv), static_cast<const void*>(angle), static_cast<const void*>(k_codes),
                        static_cast<const void*>(k_pairs), static_cast<const void*>(v_codes), static_cast<const void*>(v_pairs)})
    if (!aligned16(x)) return -10;
  if (B == 0 || T == 0) return 0;
  Int4AppendParams p = {};
  __nv_bfloat16* q = static_cast<__nv_bfloat16*>(qkv);
  const int64_t t = static_cast<int64_t>(num_q_heads + 2 * num_kv_heads) * head_dim;
  p.out_h = head_dim, p.out_t = t, p.out_b = T * t;
  p.q_out = q;
  p.k_out = q + num_q_heads * head_dim;
  p.v_out = p.k_out + num_kv_heads * head_dim;
  p.q = {p.q_out, p.out_b, t, head_dim};
  p.k = {p.k_out, p.out_b, t, head_dim};
  p.v = {p.v_out, p.out_b, t, head_dim};
  p.k_pool = {static_cast<uint8_t*>(k_codes), static_cast<uint32_t*>(k_pairs)};
  p.v_pool = {static_cast<uint8_t*>(v_codes), static_cast<uint32_t*>(v_pairs)};
  p.page_table = page_table, p.status = status;
  p.angle = reinterpret_cast<const float2*>(angle);
  p.num_q_heads = num_q_heads, p.num_kv_heads = num_kv_heads, p.max_pages = max_pages, p.num_pages = num_pages;
  return int4_append(p, B, T, page_size, head_dim, stream);
}

// Scratch of axb_int4_decode_attn in floats: up to a cluster's splits meet without any.  More are a multiple of a cluster's.
extern "C" int64_t axb_int4_attn_scratch_floats(int B, int num_q_heads, int head_dim, int splits) {
  if (splits <= axb::kAttnCluster) return 0;
  return static_cast<int64_t>(B) * num_q_heads * (splits / axb::kAttnCluster) * (head_dim + 2);
}

// One new token a sequence: q [B, Nq, H] over the cache; with `angle` ([position][H / 2] of (sin, cos)) q is the packed
// projection [B, (Nq + 2 Nkv) * H] of the token at position lengths - 1, which is rotated and appended first.
extern "C" int axb_int4_decode_attn(const void* q, void* k_codes, void* k_pairs, void* v_codes, void* v_pairs,
                                    const int* page_table, const int* lengths, const float* angle, void* out, float* scratch,
                                    int angle_rows, int B, int num_q_heads, int num_kv_heads, int head_dim, int page_size,
                                    int max_pages, int num_pages, int splits, float softmax_scale, int* status,
                                    cudaStream_t stream) {
  using namespace axb;
  if ((head_dim != 64 && head_dim != 128) || page_size < 1 || num_kv_heads < 1 || num_q_heads < 1 ||
      num_q_heads % num_kv_heads || num_pages < 1 || splits < 1 || B < 0 || B > 65535 ||
      !(softmax_scale > 0.f && softmax_scale < 1048576.f) ||
      static_cast<int64_t>(num_pages) * num_kv_heads * page_size >= 0xffffffffll || (angle != nullptr && angle_rows < 1))
    return -10;
  if (B == 0) return 0;
  for (const void* x : {q, static_cast<const void*>(angle), static_cast<const void*>(k_codes), static_cast<const void*>(k_pairs),
                        static_cast<const void*>(v_codes), static_cast<const void*>(v_pairs)})
    if (!aligned16(x)) return -10;
  if (splits > kAttnCluster && (scratch == nullptr || (reinterpret_cast<uintptr_t>(scratch) & 7) || splits % kAttnCluster)) return -10;
  Int4AttnParams p = {};
  p.q = static_cast<const __nv_bfloat16*>(q);
  p.angle = reinterpret_cast<const float2*>(angle);
  p.k_pool = {static_cast<uint8_t*>(k_codes), static_cast<uint32_t*>(k_pairs)};
  p.v_pool = {static_cast<uint8_t*>(v_codes), static_cast<uint32_t*>(v_pairs)};
  p.page_table = page_table, p.lengths = lengths;
  p.part_out = scratch;
  p.part_ml = scratch == nullptr ? nullptr : scratch + static_cast<int64_t>(B) * num_q_heads * (splits / kAttnCluster) * head_dim;
  p.out = static_cast<__nv_bfloat16*>(out);
  p.status = status;
  p.num_q_heads = num_q_heads, p.num_kv_heads = num_kv_heads, p.page_size = page_size;
  p.max_pages = max_pages, p.num_pages = num_pages, p.splits = splits;
  p.angle_rows = angle_rows;
  p.page_shift = -1;
  for (int i = 0; i < 31; ++i)
    if (page_size == 1 << i) p.page_shift = i;
  p.scale_log2 = softmax_scale * 1.4426950408889634f * kInt4Back;
  if (angle == nullptr) return head_dim == 128 ? int4_attn<128, false>(p, B, stream) : int4_attn<64, false>(p, B, stream);
  return head_dim == 128 ? int4_attn<128, true>(p, B, stream) : int4_attn<64, true>(p, B, stream);
}
