// A paged KV cache held in 8 bits (`int8.cuh`): new tokens are quantised into it, and one new token a sequence attends to it.
//
// Pools: codes [pages, Nkv, page_size, H], largest magnitudes [pages, Nkv] in bf16, for K and for V: the tokens of a page of one
// KV head are a block, and one run of memory; page table [B, max_pages], H 64 or 128, page_size a multiple of 16.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include "cache_rows.cuh"
#include "chain.cuh"
#include "cluster.cuh"
#include "int8.cuh"
#include "mma_sync.cuh"
#include "opt_in.cuh"
#include "status.cuh"

namespace axb {

struct Int8Pool {
  uint8_t* codes;
  __nv_bfloat16* tops;
};

struct Int8AppendParams {
  HeadRows q, k, v;
  __nv_bfloat16 *q_out, *k_out, *v_out;  // where the rotated q and the values of k and v go; null: not wanted
  int64_t q_out_b, q_out_t, out_b, out_t, out_h;
  Int8Pool k_pool, v_pool;
  const int* page_table;
  const int* start;     // null: 0
  const int* live;      // null: all tokens
  const int* lengths;   // a decoding step: its token is at lengths - 1, and not there where that is behind `limit`
  const float2* angle;  // (sin, cos) of [position][H / 2]; null: nothing is rotated
  int* status;
  FastDiv heads, blocks, page, q_units, tokens;  // units of a block, blocks of a sequence, positions of a page, ...
  uint32_t kv_units, all_units;
  int T, limit, num_q_heads, num_kv_heads, max_pages, num_pages;
};

constexpr int kInt8AppendThreads = 256;
constexpr int kInt8Held = 8;  // 16-byte units of rows that a thread keeps in shared memory
constexpr int kInt8QRows = 4;

// A unit is what a call brings for one block: up to a page's tokens of the keys, or the values, of a KV head.  Its kWarps warps
// hold them in shared memory while the largest magnitude is found (further rows are read again), and turn the codes that are
// there already, if the magnitude has grown.  Units behind those rotate kInt8QRows times kRows query heads of a token.
//
// Measured: 8 x 2048 tokens of 8 heads of 128 with the cache's values, 23.4 us (18.5 at the copy rate); with rows in registers and a branch
// for ties 26.3.  One token for each of 64 sequences 4.2, where that was 5.8: a launch, and behind it four loads that each wait
// for the one before, of the position, its page, the page's largest magnitude and, where that grows, its codes.
template <int H, int kWarps>
__global__ void __launch_bounds__(kInt8AppendThreads, 4)
int8_append_kernel(Int8AppendParams p) {
  chain_link();
  constexpr int kLanes = H / 8, kThreads = 32 * kWarps, kRows = kThreads / kLanes, kUnits = kInt8AppendThreads / kThreads;
  __shared__ uint32_t s_top[kInt8AppendThreads / 32];
  __shared__ uint4 s_held[kInt8Held][kInt8AppendThreads];  // (a thread's own: no bank conflicts, no barriers)
  const int in = threadIdx.x % kThreads, place = threadIdx.x / kThreads;
  const int l8 = in % kLanes, row_at = in / kLanes;
  uint32_t unit = blockIdx.x * kUnits + place;
  if (unit >= p.all_units) return;
  const uint4 zeros = make_uint4(0, 0, 0, 0);
  const bool is_q = unit >= p.kv_units;
  if (is_q) unit -= p.kv_units;
  const uint32_t outer = is_q ? p.q_units.div(unit) : p.heads.div(unit);
  const uint32_t inner = unit - outer * (is_q ? p.q_units.d : p.heads.d);
  const int b = static_cast<int>(is_q ? p.tokens.div(outer) : p.blocks.div(outer));
  int begin = p.start == nullptr ? 0 : p.start[b];
  int count = p.live == nullptr ? p.T : min(max(p.live[b], 0), p.T);
  if (p.lengths != nullptr) {
    begin = p.lengths[b] - 1;
    count = begin >= 0 && begin < p.limit ? 1 : 0;
  }
  if (is_q) {
    const int t = static_cast<int>(outer) - b * p.T;
    if (p.lengths != nullptr && count == 0) return;
    const float2* angle = p.angle + (static_cast<int64_t>(begin) + t) * (H / 2) + l8 * 4;
    const int head = static_cast<int>(inner) * kInt8QRows * kRows + row_at;
    const __nv_bfloat16* src = p.q.x + b * p.q.b + t * p.q.t + head * p.q.h + l8 * 8;
    __nv_bfloat16* dst = p.q_out + b * p.q_out_b + t * p.q_out_t + head * H + l8 * 8;
    uint4 x[kInt8QRows];
#pragma unroll
    for (int i = 0; i < kInt8QRows; ++i)
      x[i] = head + i * kRows < p.num_q_heads ? *reinterpret_cast<const uint4*>(src + i * kRows * p.q.h) : zeros;
#pragma unroll
    for (int i = 0; i < kInt8QRows; ++i)
      if (head + i * kRows < p.num_q_heads) *reinterpret_cast<uint4*>(dst + i * kRows * H) = rotate8(x[i], angle);
    return;
  }
  const int j = static_cast<int>(outer) - b * static_cast<int>(p.blocks.d);
  const bool is_v = inner >= static_cast<uint32_t>(p.num_kv_heads);
  const int head = static_cast<int>(inner) - (is_v ? p.num_kv_heads : 0);
  const int page_size = static_cast<int>(p.page.d);
  const uint32_t at0 = static_cast<uint32_t>(max(begin, 0)), col0 = p.page.div(at0);
  const int row0 = j == 0 ? static_cast<int>(at0 - col0 * p.page.d) : 0;
  const int64_t first = j == 0 ? 0 : static_cast<int64_t>(j) * page_size - (at0 - col0 * p.page.d);
  if (first >= p.T) return;
  const int t0 = static_cast<int>(first), t1 = min(p.T - t0, page_size - row0) + t0, rows = min(t1, count) - t0;
  __nv_bfloat16* out = is_v ? p.v_out : p.k_out;
  if (out != nullptr) {
    out += b * p.out_b + t0 * p.out_t + head * p.out_h + l8 * 8;
    for (int r = max(rows, 0) + row_at; r < t1 - t0; r += kRows) *reinterpret_cast<uint4*>(out + r * p.out_t) = zeros;
  }
  if (rows <= 0) return;
  const HeadRows& source = is_v ? p.v : p.k;
  const __nv_bfloat16* src = source.x + b * source.b + t0 * source.t + head * source.h + l8 * 8;
  const float2* angle = is_v || p.angle == nullptr
                            ? nullptr : p.angle + (static_cast<int64_t>(begin) + t0) * (H / 2) + l8 * 4;
  src += row_at * source.t;
  if (angle != nullptr) angle += static_cast<int64_t>(row_at) * (H / 2);
  const int64_t src_step = kRows * source.t;
  auto load = [&](int i) {  // row row_at + i kRows
    const uint4 x = *reinterpret_cast<const uint4*>(src + i * src_step);
    return angle == nullptr ? x : rotate8(x, angle + static_cast<int64_t>(i) * (kRows * H / 2));
  };
  auto largest = [](uint32_t m, const uint4& x) {  // of both halves; NaN is the largest of all
    m = __vmaxu2(m, __vmaxu2(x.x & 0x7fff7fffu, x.y & 0x7fff7fffu));
    return __vmaxu2(m, __vmaxu2(x.z & 0x7fff7fffu, x.w & 0x7fff7fffu));
  };
  const int mine = row_at < rows ? (rows - row_at + kRows - 1) / kRows : 0, held = min(mine, kInt8Held);  // rows of this thread
#pragma unroll
  for (int i = 0; i < kInt8Held; ++i)
    if (i < mine) cp16(&s_held[i][threadIdx.x], src + i * src_step);
  cp_commit();
  // The place: a sequence that starts ahead of its first position has none.
  const Int8Pool& pool = is_v ? p.v_pool : p.k_pool;
  const int64_t col = static_cast<int64_t>(col0) + j;
  uint32_t page = 0xffffffffu;
  if (begin >= 0 && col < p.max_pages) page = static_cast<uint32_t>(p.page_table[static_cast<int64_t>(b) * p.max_pages + col]);
  const bool placed = page < static_cast<uint32_t>(p.num_pages);
  if (!placed) report_bad_argument(p.status);
  const int64_t block = placed ? static_cast<int64_t>(page) * p.num_kv_heads + head : 0;
  const uint32_t old = placed && row0 > 0
                           ? static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(pool.tops + block) & 0x7fff) << 16 : 0u;
  uint32_t m = 0;
  cp_wait_all();
#pragma unroll 4
  for (int i = 0; i < held; ++i) {
    uint4& x = s_held[i][threadIdx.x];
    if (angle != nullptr) x = rotate8(x, angle + i * (kRows * H / 2));
    m = largest(m, x);
  }
  for (int i = kInt8Held; i < mine; ++i) m = largest(m, load(i));
  m = __reduce_max_sync(0xffffffffu, max(m & 0xffffu, m >> 16));
  if constexpr (kWarps > 1) {
    if ((threadIdx.x & 31) == 0) s_top[threadIdx.x >> 5] = m;
    asm volatile("bar.sync %0, %1;" ::"r"(1 + place), "r"(kThreads) : "memory");
#pragma unroll
    for (int w = 0; w < kWarps; ++w) m = max(m, s_top[place * kWarps + w]);
  }
  const float top = __uint_as_float(max(m << 16, old));
  const Int8Scale<> s(top);
  uint8_t* codes = pool.codes + (block * page_size + row0) * H + l8 * 8;
  if (placed) {
    if (in == 0) pool.tops[block] = __float2bfloat16(s.top);
    if (row0 > 0 && __float_as_uint(s.top) != old && !s.empty()) {
      // (Codes times an A that has been scaled down with the new one, as A above 2^121 times 127 is infinite.)
      Int8Scale<1> turn(top);
      const float by = __uint_as_float(old) * turn.factor;
      turn.factor = 1.f;
      for (int r = row_at; r < row0; r += kRows) {
        uint2* at = reinterpret_cast<uint2*>(codes + static_cast<int64_t>(r - row0) * H);
        const uint2 was = *at;
        float f[8];
#pragma unroll
        for (int i = 0; i < 8; ++i)
          f[i] = by * static_cast<float>(static_cast<int8_t>((i < 4 ? was.x : was.y) >> (8 * (i & 3))));
        *at = int8_codes(f, turn);
      }
    }
  }
  const float back = s.top * (1.f / 127.f);
  codes += row_at * H;
  if (out != nullptr) out += row_at * p.out_t;
  const int64_t out_step = kRows * p.out_t;
  auto hold = [&](int i, const uint4& v) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    float f[8];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 two = unpack2(w[j]);
      f[2 * j] = two.x, f[2 * j + 1] = two.y;
    }
    uint32_t u[8];
    int8_levels<false>(u, f, s);
    if (placed) *reinterpret_cast<uint2*>(codes + i * (kRows * H)) = int8_bytes(u);
    if (out != nullptr) *reinterpret_cast<uint4*>(out + i * out_step) = int8_values(u, back);
  };
#pragma unroll 1
  for (int i = 0; i < held; ++i) hold(i, s_held[i][threadIdx.x]);
  for (int i = kInt8Held; i < mine; ++i) hold(i, load(i));
}

template <int H, int kWarps>
static int launch_int8_append(Int8AppendParams& p, int64_t sequences, int q_heads, cudaStream_t stream) {
  constexpr int kRows = 32 * kWarps / (H / 8), kUnits = kInt8AppendThreads / (32 * kWarps);
  const int q_units = (q_heads + kRows * kInt8QRows - 1) / (kRows * kInt8QRows);
  const int64_t kv = sequences * p.blocks.d * 2 * p.num_kv_heads, all = kv + sequences * p.T * q_units;
  if (all >= (int64_t{1} << 31)) return -10;
  p.heads = FastDiv(2 * p.num_kv_heads), p.tokens = FastDiv(p.T);
  p.q_units = FastDiv(q_units > 0 ? q_units : 1);
  p.kv_units = static_cast<uint32_t>(kv), p.all_units = static_cast<uint32_t>(all);
  launch_chained(int8_append_kernel<H, kWarps>, static_cast<unsigned>((all + kUnits - 1) / kUnits), kInt8AppendThreads, 0, stream, p);
  return cudaGetLastError() == cudaSuccess ? 0 : -4;
}

static int int8_append(Int8AppendParams& p, int B, int page_size, int head_dim, cudaStream_t stream) {
  p.page = FastDiv(page_size);
  p.blocks = FastDiv(p.start == nullptr ? (p.T + page_size - 1) / page_size : (p.T - 1 + page_size - 1) / page_size + 1);
  // Warps of a unit: one as long as they hold its rows.
  const int rows = p.T < page_size ? p.T : page_size, held = kInt8Held * 32 / (head_dim / 8);
  const bool four = rows > held;
  if (head_dim == 128)
    return four ? launch_int8_append<128, 4>(p, B, p.num_q_heads, stream) : launch_int8_append<128, 1>(p, B, p.num_q_heads, stream);
  return four ? launch_int8_append<64, 4>(p, B, p.num_q_heads, stream) : launch_int8_append<64, 1>(p, B, p.num_q_heads, stream);
}

struct Int8AttnParams {
  const __nv_bfloat16* q;  // [B, Nq, H]
  const uint8_t *k_codes, *v_codes;
  const __nv_bfloat16 *k_tops, *v_tops;
  const int* page_table;
  const int* lengths;
  float* part_out;         // [B, Nq, splits, H]: more than a cluster's
  float* part_ml;          // [B, Nq, splits, 2]
  __nv_bfloat16* out;
  int* status;
  FastDiv page;
  int num_q_heads, num_kv_heads, max_pages, num_pages, splits;
  int limit;               // a decoding step: longer sequences than this had no place or rotation and get zeros; else -1
  float scale_log2;        // softmax scale * log2(e) / 127, > 0
};

constexpr int kI8AttnRows = 8;   // query heads of a CTA: the columns of both products
constexpr int kI8Chunk = 16;     // keys of an MMA, of one page
constexpr int kI8AttnKeys = 2 * kI8Chunk;
constexpr int kI8AttnStages = 2;
constexpr int kI8AttnCluster = 8, kI8MostSplits = 1024;
constexpr float kI8Slack = 8.f;

// Warps of a CTA: four, three CTAs an SM, or, of more splits than a cluster has, twelve that have an SM to themselves: a third of the
// parts (1 x 130001 tokens, 8 KV heads, before scores and sums were two numbers an instruction: 16 splits of twelve 49.5 us, 32 of
// four 51.6, 48 of four 53.8; 46.7 now).
constexpr int kI8FewWarps = 4, kI8ManyWarps = 12;
// Where a CTA's sums go: out, the CTA of its cluster that finishes a head, or scratch for a second launch.
enum Int8Merge { kMergeNone, kMergeCluster, kMergeScratch };

// V's codes as operands: c + 128, a byte in the low half of a bf16 lane, is the number (c + 128) 2^-133 as it lies (a denormal,
// then the first binade of the same spacing).  P carries 2^64, so that products stay in fp32's range.
constexpr float kInt8Up = 0x1p64f, kInt8Back = 0x1p69f;

__device__ __forceinline__ uint32_t int8_even(uint32_t x) { return (x & 0x00ff00ffu) ^ 0x00800080u; }
__device__ __forceinline__ uint32_t int8_odd(uint32_t x) { return ((x >> 8) & 0x00ff00ffu) ^ 0x00800080u; }

__device__ __forceinline__ uint32_t int8_turned_round(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// d = a b + c in bf16.
__device__ __forceinline__ void int8_mma_add(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, const float (&c)[4]) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
}

// Sums of products of codes and a digit of q, from kInt8Sums: whole numbers below 2^22 that are the last bits of a float.
constexpr int kInt8Sums = 0x4b400000;  // 1.5 * 2^23
template <bool kSigned>
__device__ __forceinline__ void int8_mma_sum(int (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, const int* c) {
  if constexpr (kSigned)
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
        : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "r"(c[0]), "r"(c[1]), "r"(c[2]), "r"(c[3]));
  else
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.u8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
        : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "r"(c[0]), "r"(c[1]), "r"(c[2]), "r"(c[3]));
}

__device__ __forceinline__ void int8_copy16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}

// Two matrices of 16 keys x 16 dims, a row a lane (0 .. 15, 16 .. 31): lane (r, c) gets keys 4c .. 4c + 3 of dims r and r + 8 of each.
__device__ __forceinline__ void int8_load_turned(uint32_t (&v)[4], uint32_t row) {
  asm volatile("ldmatrix.sync.aligned.m16n16.x2.trans.shared.b8 {%0,%1,%2,%3}, [%4];"
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(row));
}

template <int H, int kWarps>
struct Int8Tile {
  static constexpr int kChunk = kI8Chunk * H, kBytes = 4 * kChunk;  // two chunks of K, two of V
  static constexpr int kPart = H + 4;                               // floats of a head's part: no bank conflicts
  static constexpr int kSmem(int rows) {
    const int merge = (kWarps + 1) * rows * (kPart + 2) * 4, tiles = kWarps * kI8AttnStages * kBytes;
    return merge > tiles ? merge : tiles;
  }
  // Where 16-byte unit u of a chunk's row lies.
  __device__ static int unit(int row, int u) {
    if constexpr (H == 128) return row * 128 + ((u ^ (row & 7)) << 4);
    return row * 64 + ((u ^ ((row >> 1) & 3)) << 4);
  }
};

// S^T = K Q^T in integers: 16 keys are the rows of the m16n8k32 tile, the query heads its columns, K's codes operands as they lie.
// A head's q is a whole number of 24 bits times a power of two, three digits of 8 bits, so that scores are exact to 2^-23 of its
// largest value.  O^T = V^T P^T in bf16: 16 dims are the rows, `ldmatrix` turns V round and `movmatrix` P, and a word of four
// codes becomes two operand registers.  A chunk of 16 keys is of one page, so A / 127 of K multiplies its scores, and that of V its
// products in fp32; codes of V enter as c + 128, and 128 times the sums of P leave again.  P is rounded to bf16 once and normalised
// by the sum of what it was rounded to.  The maximum that P is relative to moves only when a score passes it by kI8Slack.
//
// A tile is 32 keys, a warp's own from `cp.async` to its sums: no barrier of the CTA before the end.  Tiles go round the warps of all
// splits; splits of eight or less are a cluster whose parts meet in distributed shared memory, those of more are joined by a second
// launch.
//
// Measured (us; at the copy rate): 64 sequences of 2000 tokens, 32 KV heads of 128, 154 in a burst and 161 for as long as one likes
// (160); 16 x up to 2048 tokens, 8 KV heads for 32, 14.3 (5.3); 1 x 130001, 8 KV heads for 32, 46.7 (40.6); 1 x 300, 16 heads, 4.2.
// With bf16 operands in both products (three operations to unpack four codes of K, four of V) the first was 164 and, under the power
// cap, 190; with TMA boxes of 16 rows, whose issue by one or two lanes and whose barriers cost some hundred instructions a tile,
// 160 and 178, and a split of 2048 tokens of one warp in four 20.4 where it is 18 now; without two
// numbers an instruction for scores and sums 4.5, 14.9, 155 and 47.8.  What is left of small calls is a CTA's
// start and end, 4 us, and the 0.75 us that a warp takes for a tile when nothing else runs on its scheduler.
template <int H, int kWarps, Int8Merge kMerge>
__global__ void __launch_bounds__(32 * kWarps, 12 / kWarps)
int8_attn_kernel(Int8AttnParams p) {
  chain_link();
  using Tile = Int8Tile<H, kWarps>;
  constexpr int kSteps = H / 16, kDigitSteps = H / 32;  // MMAs of a chunk in V's product, in K's for a digit
  extern __shared__ __align__(128) uint8_t s_ring[];
  const int split = blockIdx.x;
  const int group = p.num_q_heads / p.num_kv_heads;
  const int parts = (group + kI8AttnRows - 1) / kI8AttnRows;
  const int kvh = blockIdx.y / parts;
  const int first = blockIdx.y % parts * kI8AttnRows;
  const int rows = min(kI8AttnRows, group - first);
  const int qh0 = kvh * group + first;
  const int b = blockIdx.z;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int r = lane >> 2, c = lane & 3;
  const int page_size = static_cast<int>(p.page.d);
  const int64_t capacity = p.max_pages * static_cast<int64_t>(page_size);
  const int step = kWarps * p.splits, tile0 = split * kWarps + warp;
  const int* table = p.page_table + static_cast<int64_t>(b) * p.max_pages;
  // 16-byte units of K's rows that a lane takes: of 128-byte rows two that leave those of the next lanes' rows other banks.
  const int unit0 = H == 128 ? (c & 1) + ((c >> 1) << 2) : c;
  const __nv_bfloat16* q_at = p.q + (static_cast<int64_t>(b) * p.num_q_heads + qh0 + r) * H + unit0 * 16;
  const uint4 zeros = make_uint4(0, 0, 0, 0);

  // Places of a warp's tiles, sixteen at a time: lane l has chunk l % 2 of tile l / 2 of a batch, its page a batch ahead of the
  // row of the pools and the magnitudes that follow from it, and those a batch ahead of their use.
  auto position = [&](int batch) -> int64_t {
    return (static_cast<int64_t>(tile0) + (static_cast<int64_t>(batch) * 16 + (lane >> 1)) * step) * kI8AttnKeys + (lane & 1) * kI8Chunk;
  };
  auto page_of = [&](int batch, int64_t end) -> uint32_t {
    const int64_t pos = position(batch);
    return pos < end ? static_cast<uint32_t>(table[p.page.div(static_cast<uint32_t>(pos))]) : 0u;
  };
  // (The table's first entries and the queries do not wait for the length: 4.5 us where it was 4.7 at 1 x 300 tokens, 14.9 for 15.8
  // at 16 x up to 2048.)
  int len = p.lengths[b];
  uint32_t page = page_of(0, min(capacity, int64_t{0x7fffffff})), page_next = page_of(1, min(capacity, int64_t{0x7fffffff}));
  uint4 q_raw[kDigitSteps];
#pragma unroll
  for (int j = 0; j < kDigitSteps; ++j) q_raw[j] = r < rows ? *reinterpret_cast<const uint4*>(q_at + (j >> 1) * 32 + (j & 1) * 8) : zeros;
  if (len > capacity || (p.limit >= 0 && len > p.limit)) {
    if (threadIdx.x == 0) report_bad_argument(p.status);
    len = p.limit >= 0 ? 0 : static_cast<int>(capacity);
  }
  len = max(len, 0);
  const int hi = len / kI8AttnKeys + (len % kI8AttnKeys != 0);
  struct Places {
    int row;  // of the pools; -1: no keys
    uint16_t k_top, v_top;
  };
  auto places = [&](int batch, uint32_t page) -> Places {
    const int64_t pos = position(batch);
    Places at{-1, 0, 0};
    if (pos >= len) return at;
    if (page >= static_cast<uint32_t>(p.num_pages)) {
      report_bad_argument(p.status);
      return at;
    }
    const uint32_t col = p.page.div(static_cast<uint32_t>(pos));
    const int64_t block = static_cast<int64_t>(page) * p.num_kv_heads + kvh;
    at.row = static_cast<int>(block * page_size + (pos - static_cast<int64_t>(col) * page_size));
    at.k_top = *reinterpret_cast<const uint16_t*>(p.k_tops + block);
    at.v_top = *reinterpret_cast<const uint16_t*>(p.v_tops + block);
    return at;
  };
  Places now = places(0, page), next = places(1, page_next);
  page = page_of(2, len);
  uint32_t none = __ballot_sync(0xffffffffu, now.row < 0);  // chunks of the batch without keys
  uint8_t* ring = s_ring + warp * kI8AttnStages * Tile::kBytes;
  // Tile `n` of the warp, whose batch is `now` or the next one.  A chunk is a run of memory; its 16-byte units are swapped within
  // 128 bytes, so that eight lanes of both products hit all banks.  Chunks that are not there come from the first row, and do not count.
  uint32_t to[2];  // of unit `lane`, and 512 bytes further
#pragma unroll
  for (int i = 0; i < 2; ++i) to[i] = sptr(ring) + Tile::unit(lane / (H / 16) + i * (512 / H), lane % (H / 16));
  const uint8_t* k_src = p.k_codes + lane * 16;
  const uint8_t* v_src = p.v_codes + lane * 16;
  auto load_tile = [&](int n, int stage, bool ahead) {
    const int at = ahead ? next.row : now.row;
#pragma unroll
    for (int ch = 0; ch < 2; ++ch) {
      const int64_t off = static_cast<int64_t>(max(__shfl_sync(0xffffffffu, at, (n & 15) * 2 + ch), 0)) * H;
      const uint32_t dst = stage * Tile::kBytes + ch * Tile::kChunk;
#pragma unroll
      for (int i = 0; i < Tile::kChunk / 512; ++i) {
        int8_copy16(to[i & 1] + dst + (i >> 1) * 1024, k_src + off + i * 512);
        int8_copy16(to[i & 1] + dst + 2 * Tile::kChunk + (i >> 1) * 1024, v_src + off + i * 512);
      }
    }
  };
#pragma unroll
  for (int i = 0; i < kI8AttnStages; ++i) {
    if (tile0 + i * step < hi) load_tile(i, i, false);
    cp_commit();
  }

  // Q of head r in three digits, q = 2^(e - 22) (65536 q2 + 256 q1 + q0), e the exponent of its largest value; step j takes eight
  // dims of a unit.
  uint32_t qd[3][kDigitSteps][2];
  float q_scale[2];
  {
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < kDigitSteps; ++j) {
      top = __vmaxu2(top, __vmaxu2(q_raw[j].x & 0x7fff7fffu, q_raw[j].y & 0x7fff7fffu));
      top = __vmaxu2(top, __vmaxu2(q_raw[j].z & 0x7fff7fffu, q_raw[j].w & 0x7fff7fffu));
    }
    top = max(top & 0xffffu, top >> 16);
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
    // (Queries below 2^-64 are not told apart any further.)
    const int e = max(static_cast<int>(top >> 7) - 127, -64);
    const float up = __int_as_float((22 - e + 127) << 23);  // (of an infinity or NaN: what comes out is not used)
    float back = top >= 0x7f80u ? __int_as_float(0x7fffffff) : __int_as_float((e - 22 + 127) << 23);
    back *= p.scale_log2;
    q_scale[0] = __shfl_sync(0xffffffffu, back, 8 * c);
    q_scale[1] = __shfl_sync(0xffffffffu, back, 8 * c + 4);
#pragma unroll
    for (int j = 0; j < kDigitSteps; ++j) {
      const uint32_t w[4] = {q_raw[j].x, q_raw[j].y, q_raw[j].z, q_raw[j].w};
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float2 f0 = unpack2(w[2 * i]), f1 = unpack2(w[2 * i + 1]);
        const int n0 = __float2int_rn(f0.x * up), n1 = __float2int_rn(f0.y * up), n2 = __float2int_rn(f1.x * up),
                  n3 = __float2int_rn(f1.y * up);
#pragma unroll
        for (int digit = 0; digit < 3; ++digit) {
          const uint32_t pick = digit | (digit + 4) << 4;
          qd[digit][j][i] = __byte_perm(__byte_perm(n0, n1, pick), __byte_perm(n2, n3, pick), 0x5410);
        }
      }
    }
  }

  float m[2] = {-INFINITY, -INFINITY};  // heads 2c, 2c + 1
  uint64_t l = 0, w_sum = 0;            // pairs of them
  uint64_t acc[kSteps][2];  // pairs of heads 2c, 2c + 1 for dims 16 i + r and 16 i + 8 + r
#pragma unroll
  for (int i = 0; i < kSteps; ++i) acc[i][0] = acc[i][1] = 0;
  const uint64_t q_scales = f32x2(q_scale[0], q_scale[1]);
  const float zero[4] = {0.f, 0.f, 0.f, 0.f};
  const int none_yet[4] = {kInt8Sums, kInt8Sums, kInt8Sums, kInt8Sums};
  const uint32_t ones[4] = {0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u};
  // Slots r and r + 8 of a chunk's rows are keys 2r and 2r + 1, so that after `movmatrix` lane c has P of the keys that `ldmatrix` gives
  // it of V.
  const uint8_t* k_at = ring + Tile::unit(2 * r, unit0);
  const uint32_t v_at = sptr(ring) + 2 * Tile::kChunk;

  int stage = 0, n = 0;
  for (int tile = tile0; tile < hi; tile += step, ++n) {
    if (n > 0 && (n & 15) == 0) {
      now = next;
      none = __ballot_sync(0xffffffffu, now.row < 0);
      const int batch = n >> 4;
      next = places(batch + 1, page);
      page = page_of(batch + 2, len);
    }
    cp_wait_group<kI8AttnStages - 1>();
    __syncwarp();
    const int at_stage = stage * Tile::kBytes, lane_a = (n & 15) * 2;
    const uint32_t tops = static_cast<uint32_t>(now.k_top) | static_cast<uint32_t>(now.v_top) << 16;
    uint64_t s[2][2];  // keys 2r and 2r + 1 of a chunk, pairs of heads
    float vt[2];
#pragma unroll
    for (int ch = 0; ch < 2; ++ch) {
      const uint32_t pair = __shfl_sync(0xffffffffu, tops, lane_a + ch);
      const float kt = __uint_as_float(pair << 16);
      vt[ch] = __uint_as_float(pair & 0xffff0000u) * (1.f / 127.f);
      uint32_t w[2][2 * kDigitSteps];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int u = 0; u < kDigitSteps / 2; ++u) {
          // (The next row, the second unit: bits of the swizzled place, and the row's own.)
          const uint8_t* at = H == 128 ? ring + Tile::unit(2 * r + i, unit0 + 2 * u) : k_at + i * H;
          *reinterpret_cast<uint4*>(&w[i][4 * u]) = *reinterpret_cast<const uint4*>(at + at_stage + ch * Tile::kChunk);
        }
      }
      int d[3][4];
#pragma unroll
      for (int j = 0; j < kDigitSteps; ++j) {
        const uint32_t a[4] = {w[0][2 * j], w[1][2 * j], w[0][2 * j + 1], w[1][2 * j + 1]};
        int8_mma_sum<false>(d[0], a, qd[0][j][0], qd[0][j][1], j == 0 ? none_yet : d[0]);
        int8_mma_sum<false>(d[1], a, qd[1][j][0], qd[1][j][1], j == 0 ? none_yet : d[1]);
        int8_mma_sum<true>(d[2], a, qd[2][j][0], qd[2][j][1], j == 0 ? none_yet : d[2]);
      }
      const float start = -__int_as_float(kInt8Sums);
      const uint64_t by = mul2(q_scales, f32x2(kt, kt));
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        uint64_t f[3];
#pragma unroll
        for (int digit = 0; digit < 3; ++digit)
          f[digit] = add2(f32x2(__int_as_float(d[digit][2 * i]), __int_as_float(d[digit][2 * i + 1])), f32x2(start, start));
        s[ch][i] = mul2(fma2(f[2], f32x2(65536.f, 65536.f), fma2(f[1], f32x2(256.f, 256.f), f[0])), by);
      }
    }
    const uint32_t empty = none >> lane_a & 3;  // chunks behind the sequence, or of a page that is not in the pool
    if (empty != 0 || (tile + 1) * static_cast<int64_t>(kI8AttnKeys) > len) {
#pragma unroll
      for (int ch = 0; ch < 2; ++ch) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
          if ((empty >> ch & 1) || tile * kI8AttnKeys + ch * kI8Chunk + 2 * r + i >= len) s[ch][i] = f32x2(-INFINITY, -INFINITY);
      }
    }
    float top[2];
    {
      float x[4][2];
#pragma unroll
      for (int i = 0; i < 4; ++i) f32x2_split(s[i >> 1][i & 1], x[i][0], x[i][1]);
#pragma unroll
      for (int h = 0; h < 2; ++h) top[h] = fmaxf(fmaxf(x[0][h], x[1][h]), fmaxf(x[2][h], x[3][h]));
    }
    if (__any_sync(0xffffffffu, top[0] > m[0] + kI8Slack || top[1] > m[1] + kI8Slack)) {
      float by[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int off = 4; off <= 16; off <<= 1) top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], off));
        const float m_new = fmaxf(m[h], top[h]);
        by[h] = m[h] == -INFINITY ? 0.f : ex2(m[h] - m_new);  // (nothing is there yet)
        m[h] = m_new;
      }
      const uint64_t both = f32x2(by[0], by[1]);
      l = mul2(l, both), w_sum = mul2(w_sum, both);
#pragma unroll
      for (int i = 0; i < kSteps; ++i) acc[i][0] = mul2(acc[i][0], both), acc[i][1] = mul2(acc[i][1], both);
    }
    const uint64_t base = f32x2(m[0] == -INFINITY ? 0.f : 64.f - m[0], m[1] == -INFINITY ? 0.f : 64.f - m[1]);
#pragma unroll
    for (int ch = 0; ch < 2; ++ch) {
      uint32_t pt[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {  // (NaN stays)
        float x, y;
        f32x2_split(add2(s[ch][i], base), x, y);
        pt[i] = int8_turned_round(pack2(ex2(x), ex2(y)));
      }
      float sums[4];  // of P, in every lane of a column
      int8_mma_add(sums, ones, pt[0], pt[1], zero);
      const uint64_t both = f32x2(sums[0], sums[1]);
      l = add2(l, both);
      w_sum = fma2(f32x2(vt[ch], vt[ch]), mul2(both, f32x2(1.f / kInt8Up, 1.f / kInt8Up)), w_sum);
      const uint64_t back = f32x2(vt[ch] * kInt8Back, vt[ch] * kInt8Back);
#pragma unroll
      for (int i = 0; i < kSteps; i += 2) {
        uint32_t v[4];
        int8_load_turned(v, v_at + at_stage + ch * Tile::kChunk + Tile::unit(lane & 15, i + (lane >> 4)));
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const uint32_t a[4] = {int8_even(v[2 * t]), int8_even(v[2 * t + 1]), int8_odd(v[2 * t]), int8_odd(v[2 * t + 1])};
          float d[4];
          int8_mma_add(d, a, pt[0], pt[1], zero);
#pragma unroll
          for (int e = 0; e < 2; ++e) acc[i + t][e] = fma2(back, f32x2(d[2 * e], d[2 * e + 1]), acc[i + t][e]);
        }
      }
    }
    __syncwarp();  // the stage has been read
    if (tile + kI8AttnStages * static_cast<int64_t>(step) < hi)
      load_tile(n + kI8AttnStages, stage, (n >> 4) != ((n + kI8AttnStages) >> 4));
    cp_commit();
    if (++stage == kI8AttnStages) stage = 0;
  }
  cp_wait_all();
  __syncthreads();  // the merge buffers overlay the tiles
  constexpr int kPart = Tile::kPart;
  float* s_part = reinterpret_cast<float*>(s_ring);  // the warps and the CTA: [rows][kPart] sums, then maxima, then weights
  const int per_warp = rows * kPart;
  float* s_m = s_part + (kWarps + 1) * per_warp;
  float* s_l = s_m + (kWarps + 1) * rows;
  float l_of[2], w_of[2];
  f32x2_split(l, l_of[0], l_of[1]);
  f32x2_split(w_sum, w_of[0], w_of[1]);
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    if (2 * c + h >= rows) continue;
    float* dst = s_part + warp * per_warp + (2 * c + h) * kPart + r;
    const float low = -128.f * w_of[h];
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float x[2];
        f32x2_split(acc[i][e], x[0], x[1]);
        dst[16 * i + 8 * e] = x[h] + low;
      }
    }
    if (r == 0) {
      s_m[warp * rows + 2 * c + h] = m[h];
      s_l[warp * rows + 2 * c + h] = l_of[h] * (1.f / kInt8Up);
    }
  }
  __syncthreads();
  // Thread (g, d) of H threads a head owns output dim d.
  constexpr int kSets = 32 * kWarps / H;
  const int d = threadIdx.x % H;
  for (int g = threadIdx.x / H; g < rows; g += kSets) {
    float mm = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) mm = fmaxf(mm, s_m[w * rows + g]);
    float ll = 0.f, o = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float f = mm == -INFINITY ? 1.f : exp2f(s_m[w * rows + g] - mm);
      ll += s_l[w * rows + g] * f;
      o += s_part[w * per_warp + g * kPart + d] * f;
    }
    const int64_t row = static_cast<int64_t>(b) * p.num_q_heads + qh0 + g;
    if constexpr (kMerge == kMergeNone) {
      p.out[row * H + d] = __float2bfloat16(ll == 0.f ? 0.f : o / ll);
    } else if constexpr (kMerge == kMergeScratch) {
      const int64_t part = row * p.splits + split;
      p.part_out[part * H + d] = o;
      if (d == 0) *reinterpret_cast<float2*>(p.part_ml + part * 2) = make_float2(mm, ll);
    } else {
      s_part[kWarps * per_warp + g * kPart + d] = o;
      if (d == 0) {
        s_m[kWarps * rows + g] = mm;
        s_l[kWarps * rows + g] = ll;
      }
    }
  }
  if constexpr (kMerge == kMergeCluster) {
    const int cluster = p.splits, rank = split;
    cluster_sync_all();
    for (int g = rank * kSets + threadIdx.x / H; g < rows; g += cluster * kSets) {
      float mv[kI8AttnCluster], lv[kI8AttnCluster], ov[kI8AttnCluster];
#pragma unroll
      for (int s = 0; s < kI8AttnCluster; ++s) {
        const bool have = s < cluster;
        mv[s] = have ? ld_cluster_f32(sptr(s_m + kWarps * rows + g), s) : -INFINITY;
        lv[s] = have ? ld_cluster_f32(sptr(s_l + kWarps * rows + g), s) : 0.f;
        ov[s] = have ? ld_cluster_f32(sptr(s_part + kWarps * per_warp + g * kPart + d), s) : 0.f;
      }
      float mm = -INFINITY;
#pragma unroll
      for (int s = 0; s < kI8AttnCluster; ++s) mm = fmaxf(mm, mv[s]);
      float ll = 0.f, o = 0.f;
#pragma unroll
      for (int s = 0; s < kI8AttnCluster; ++s) {
        const float f = mm == -INFINITY ? 1.f : exp2f(mv[s] - mm);
        ll += lv[s] * f;
        o += ov[s] * f;
      }
      const int64_t row = static_cast<int64_t>(b) * p.num_q_heads + qh0 + g;
      p.out[row * H + d] = __float2bfloat16(ll == 0.f ? 0.f : o / ll);
    }
    cluster_sync_all();  // a CTA's shared memory outlives its readers
  }
}

// The splits' parts of a row, eight at a time on their way.
template <int H>
__global__ void __launch_bounds__(H)
int8_combine_kernel(const float* part_out, const float* part_ml, __nv_bfloat16* out, int parts) {
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

template <int H, int kWarps, Int8Merge kMerge>
static int launch_int8_attn(const Int8AttnParams& p, dim3 grid, cudaStream_t stream) {
  constexpr auto kernel = int8_attn_kernel<H, kWarps, kMerge>;
  constexpr int kSmem = Int8Tile<H, kWarps>::kSmem(kI8AttnRows);
  static_assert(12 / kWarps * (kSmem + 1024 + 512) <= 228 * 1024, "resident CTAs");
  static OptIn opt_in;
  if (!opt_in.done(kernel, kSmem)) return -3;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim = {static_cast<unsigned>(p.splits), 1, 1};
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(32 * kWarps);
  cfg.dynamicSmemBytes = static_cast<size_t>(kSmem);
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = static_cast<unsigned>(chain_attribute(attr, kMerge == kMergeCluster ? 1 : 0));
  return cudaLaunchKernelEx(&cfg, kernel, p) == cudaSuccess ? 0 : -4;
}

template <int H>
static int int8_attn(const Int8AttnParams& p, int B, cudaStream_t stream) {
  const int g = p.num_q_heads / p.num_kv_heads;
  const dim3 grid(p.splits, p.num_kv_heads * ((g + kI8AttnRows - 1) / kI8AttnRows), B);
  const int rc = p.splits == 1                ? launch_int8_attn<H, kI8FewWarps, kMergeNone>(p, grid, stream)
                 : p.splits <= kI8AttnCluster ? launch_int8_attn<H, kI8FewWarps, kMergeCluster>(p, grid, stream)
                                              : launch_int8_attn<H, kI8ManyWarps, kMergeScratch>(p, grid, stream);
  if (rc != 0) return rc;
  if (p.splits > kI8AttnCluster) {
    ChainedBehind chained;
    launch_chained(int8_combine_kernel<H>, B * p.num_q_heads, H, 0, stream, p.part_out, p.part_ml, p.out, p.splits);
  }
  return cudaGetLastError() == cudaSuccess ? 0 : -4;
}

// What the entry points below ask of a cache.
static bool int8_cache_fits(int64_t head_dim, int64_t page_size, int64_t num_kv_heads, int64_t num_pages, const void* k_codes,
                            const void* v_codes) {
  return (head_dim == 64 || head_dim == 128) && page_size >= 16 && page_size % 16 == 0 && num_kv_heads >= 1 && num_pages >= 1 &&
         int8_ints({page_size, num_kv_heads, num_pages}) && num_pages * num_kv_heads < 0x7fffffffll / page_size &&
         aligned16(k_codes) && aligned16(v_codes);
}

}  // namespace axb

// k and v [B, T, Nkv, H] with element strides of (sequence, token, head); k_out and v_out (null: not wanted) are contiguous.
// -10: not supported.
extern "C" int axb_int8_append(const axb::Int8AppendCall* call, cudaStream_t stream) {
  using namespace axb;
  const Int8AppendCall& a = *call;
  if (!int8_cache_fits(a.head_dim, a.page_size, a.num_kv_heads, a.num_pages, a.k_codes, a.v_codes) || a.B < 0 || a.T < 0 ||
      !int8_ints({a.B, a.T, a.max_pages}) || (a.k_b | a.k_t | a.k_h | a.v_b | a.v_t | a.v_h) % 8)
    return -10;
  if (a.B == 0 || a.T == 0) return 0;
  for (const void* x : {a.k, a.v, static_cast<const void*>(a.k_out), static_cast<const void*>(a.v_out)})
    if (!aligned16(x)) return -10;
  Int8AppendParams p = {};
  p.k = {static_cast<const __nv_bfloat16*>(a.k), a.k_b, a.k_t, a.k_h};
  p.v = {static_cast<const __nv_bfloat16*>(a.v), a.v_b, a.v_t, a.v_h};
  p.k_out = static_cast<__nv_bfloat16*>(a.k_out);
  p.v_out = static_cast<__nv_bfloat16*>(a.v_out);
  p.out_h = a.head_dim, p.out_t = a.num_kv_heads * a.head_dim, p.out_b = a.T * p.out_t;
  p.k_pool = {static_cast<uint8_t*>(a.k_codes), static_cast<__nv_bfloat16*>(a.k_tops)};
  p.v_pool = {static_cast<uint8_t*>(a.v_codes), static_cast<__nv_bfloat16*>(a.v_tops)};
  p.page_table = a.page_table, p.start = a.start, p.live = a.live, p.status = a.status;
  p.T = static_cast<int>(a.T), p.num_kv_heads = static_cast<int>(a.num_kv_heads);
  p.max_pages = static_cast<int>(a.max_pages), p.num_pages = static_cast<int>(a.num_pages);
  return int8_append(p, static_cast<int>(a.B), static_cast<int>(a.page_size), static_cast<int>(a.head_dim), stream);
}

// qkv [B, T, (Nq + 2 Nkv) * H] of one projection, queries and keys to be rotated by `angle` ([position][H / 2] of (sin, cos)).
// Whole prompts (`lengths` null) start at position 0 and have `live` tokens (null: T): rotated queries and what the cache then
// stands for replace queries, keys and values (zeros behind `live`).  A decoding step has T = 1 token at position lengths - 1;
// its rotated queries go to q_out [B, Nq, H], and sequences of length 0 or behind the table or the rotations append nothing.
extern "C" int axb_int8_rope_append(const axb::Int8RopeAppendCall* call, cudaStream_t stream) {
  using namespace axb;
  const Int8RopeAppendCall& a = *call;
  const bool step = a.lengths != nullptr;
  if (!int8_cache_fits(a.head_dim, a.page_size, a.num_kv_heads, a.num_pages, a.k_codes, a.v_codes) || a.num_q_heads < 1 || a.B < 0 ||
      a.T < 0 || !int8_ints({a.B, a.T, a.max_pages, a.num_q_heads}) || (step ? a.T != 1 || a.angle_rows < 1 : a.angle_rows < a.T))
    return -10;
  if (a.B == 0 || a.T == 0) return 0;
  if (step && a.q_out == nullptr) return -10;
  for (const void* x : {static_cast<const void*>(a.qkv), static_cast<const void*>(a.q_out), static_cast<const void*>(a.angle)})
    if (!aligned16(x)) return -10;
  Int8AppendParams p = {};
  __nv_bfloat16* q = static_cast<__nv_bfloat16*>(a.qkv);
  const int64_t t = (a.num_q_heads + 2 * a.num_kv_heads) * a.head_dim, h = a.head_dim;
  p.q = {q, a.T * t, t, h};
  p.k = {q + a.num_q_heads * h, a.T * t, t, h};
  p.v = {p.k.x + a.num_kv_heads * h, a.T * t, t, h};
  if (step) {
    p.q_out = static_cast<__nv_bfloat16*>(a.q_out);
    p.q_out_b = p.q_out_t = a.num_q_heads * h;
    const int64_t capacity = a.max_pages * a.page_size, most = capacity < a.angle_rows ? capacity : a.angle_rows;
    p.limit = static_cast<int>(most < 0x7fffffff ? most : 0x7fffffff);
  } else {
    p.q_out = q, p.q_out_b = a.T * t, p.q_out_t = t;
    p.k_out = q + a.num_q_heads * h;
    p.v_out = p.k_out + a.num_kv_heads * h;
    p.out_b = a.T * t, p.out_t = t, p.out_h = h;
  }
  p.k_pool = {static_cast<uint8_t*>(a.k_codes), static_cast<__nv_bfloat16*>(a.k_tops)};
  p.v_pool = {static_cast<uint8_t*>(a.v_codes), static_cast<__nv_bfloat16*>(a.v_tops)};
  p.page_table = a.page_table, p.lengths = a.lengths, p.live = a.live, p.status = a.status;
  p.angle = reinterpret_cast<const float2*>(a.angle);
  p.T = static_cast<int>(a.T), p.num_q_heads = static_cast<int>(a.num_q_heads), p.num_kv_heads = static_cast<int>(a.num_kv_heads);
  p.max_pages = static_cast<int>(a.max_pages), p.num_pages = static_cast<int>(a.num_pages);
  return int8_append(p, static_cast<int>(a.B), static_cast<int>(a.page_size), static_cast<int>(a.head_dim), stream);
}

// Scratch of axb_int8_decode_attn in floats: up to a cluster's splits meet without any.
extern "C" int64_t axb_int8_attn_scratch_floats(int B, int num_q_heads, int head_dim, int splits) {
  if (splits <= axb::kI8AttnCluster) return 0;
  return static_cast<int64_t>(B) * num_q_heads * splits * (head_dim + 2);
}

// One new token a sequence: q [B, Nq, H] over the cache, into out [B, Nq, H] (which may be q).  `limit` (-1: none): sequences
// behind it get zeros.
extern "C" int axb_int8_decode_attn(const axb::Int8AttnCall* call, cudaStream_t stream) {
  using namespace axb;
  const Int8AttnCall& a = *call;
  if (!int8_cache_fits(a.head_dim, a.page_size, a.num_kv_heads, a.num_pages, a.k_codes, a.v_codes) || a.num_q_heads < 1 ||
      a.num_q_heads % a.num_kv_heads || a.splits < 1 || a.splits > kI8MostSplits || a.B < 0 || a.B > 65535 ||
      !int8_ints({a.num_q_heads, a.max_pages}) || !(a.softmax_scale > 0. && a.softmax_scale < 1048576.) || !aligned16(a.q) ||
      a.num_kv_heads * ((a.num_q_heads / a.num_kv_heads + kI8AttnRows - 1) / kI8AttnRows) > 65535)
    return -10;
  if (a.B == 0) return 0;
  if (a.splits > kI8AttnCluster && (a.scratch == nullptr || (reinterpret_cast<uintptr_t>(a.scratch) & 7))) return -10;
  Int8AttnParams p = {};
  p.q = static_cast<const __nv_bfloat16*>(a.q);
  p.k_codes = static_cast<const uint8_t*>(a.k_codes), p.v_codes = static_cast<const uint8_t*>(a.v_codes);
  p.k_tops = static_cast<const __nv_bfloat16*>(a.k_tops), p.v_tops = static_cast<const __nv_bfloat16*>(a.v_tops);
  p.page_table = a.page_table, p.lengths = a.lengths;
  p.part_out = a.scratch;
  p.part_ml = a.scratch == nullptr ? nullptr : a.scratch + a.B * a.num_q_heads * a.splits * a.head_dim;
  p.out = static_cast<__nv_bfloat16*>(a.out);
  p.status = a.status;
  p.page = FastDiv(static_cast<int>(a.page_size));
  p.num_q_heads = static_cast<int>(a.num_q_heads), p.num_kv_heads = static_cast<int>(a.num_kv_heads);
  p.max_pages = static_cast<int>(a.max_pages), p.num_pages = static_cast<int>(a.num_pages);
  p.splits = static_cast<int>(a.splits);
  p.limit = static_cast<int>(a.limit < 0 ? -1 : a.limit < 0x7fffffff ? a.limit : 0x7fffffff);
  p.scale_log2 = static_cast<float>(a.softmax_scale) * (1.4426950408889634f / 127.f);
  const int B = static_cast<int>(a.B);
  return a.head_dim == 128 ? int8_attn<128>(p, B, stream) : int8_attn<64>(p, B, stream);
}
