// Attention of one new token per sequence over a paged key/value cache.
//
// For query head h of sequence b, with n = lengths[b] tokens in the cache and k_t, v_t the rows of
// its key/value head (times their scales where the pool holds 8 bits):
//     s_t = scale * q . k_t,   o = sum_t softmax(s)_t v_t,   lse = log sum_t exp(s_t).
// A sequence without tokens gives o = 0 and lse = -inf.  Tokens in pages that lie outside the pool
// count as masked, lengths beyond the table are cut to it.
//
// Bound: memory.  Every cached byte is needed once and meets 2 * (heads per key/value head) flops per
// element, so the kernel is built around keeping loads in flight:
//
// * Work.  A *row* is one sequence and one key/value head with up to 8 of its query heads (a larger
//   group makes further rows, which read the same keys and values again).  All rows' tiles of TOK tokens
//   form one line, cut into equal ranges per block and, inside a block, per warp, whatever the lengths:
//   one persistent block per SM, no idle SM for ragged batches, long rows split without a plan on the
//   host.  Every warp streams its range through a ring of its own in shared memory with 16-byte
//   cp.async; warps never wait for one another before their range is done.
// * Matrix instructions.  S = Q K^T and O += P V have the 8 heads as rows 0-7 of a tile of 16 rows, the smallest
//   there is: at these intensities the tensor pipe is far from its limit.  Rows 8-15 are not wasted; they carry
//   what rounding left over of the same heads' operand.  P enters with the 24 bits of an fp32 weight, as three bf16 terms or
//   four digits of 8 bits, since two of either would move one bf16 output in 600 (bf16) or 60 (int8) to its neighbour.  Where a row
//   has at most 4 heads the third (and fourth) go to rows 4-7 (and 12-15), whose lanes repeat the scores of rows 0-3: no
//   further instruction (10 warps, 32 x 4096 bf16 at 32/8 heads 92.2 us, with two terms 91.8; 48 ragged GPT-2 rows 23.8 and 23.4).
//   With 5 to 8 heads they take a second instruction (32 x 4096 at 32/4 heads: bf16 53.0 and 51.9 us, int8 41.2 and 37.1).
//   The dimensions of q and k are summed in the order in which 16-byte loads deliver them, and the tokens of a tile in
//   the order in which score accumulators and the second product's operand agree: no data is moved for either.
// * 8 bits.  Keys enter the instructions (m16n8k32) as they are held, so q has to be in 8 bits too, as digits, worked
//   out once per row.  int8: q of a head, scaled by a power of two and rounded to 22 bits, is three signed digits, and
//   the sums are exact integers (below 2^22, read as floats by starting the accumulators at the bits of 1.5 2^23).  The
//   third digit has rows 4-7 of at most 4 heads, or a second instruction, which took 128 x 4097..8192 at 32/8 heads from
//   272 us to 293.
//   e4m3: q is two terms of 4 bits each, which hold all 8 bits of a bf16.  int8 values are used as they are as well,
//   with floor(2^31 p) as four unsigned digits: p is taken relative to the tile's own maximum, so that its
//   digits always start at the tile's largest weight, and the tile's product is added to the output in fp32.  e4m3 values are
//   converted to fp16 pairs (one conversion costs what a byte permute does; three e4m3 terms of p per token
//   cost more: 82 us against 71 on 32 rows of 4096).
//   A token's key scale multiplies its score.  Of its value scale sv = 2^n f, 1 <= f < 2, the power of two joins the
//   exponent: with s'_t = s_t + n_t, m the maximum of s' rounded up and x_t = 2^(s'_t - m) <= 1, the output is
//   sum (x_t f_t) v_t / sum (x_t 2^-n_t): what is rounded for it is s' alone, like the score itself.  n is held within 60 of the
//   largest so far (with a smaller f), so that weights stay in range whatever the scales are, of rows of zeros next to values
//   of 2^64 and more, too.
// * References m are whole numbers, in all formats: factors between them are powers of two and round nothing.
// * Joining.  A row inside one warp's range is finished by that warp.  Otherwise warps leave (o, m, sum)
//   in shared memory, the block merges neighbours, and rows that cross blocks go through a workspace:
//   the block that arrives last merges the pieces in the order of the tokens, so results do not depend
//   on timing.  One launch, no second kernel.
#include <algorithm>

#include "generation.cuh"

namespace ht {
namespace paged {

constexpr float LN2 = 0.6931471805599453f;
constexpr int HEADS = 8;  // query heads of one row

template <int F, int D>
struct Shape {
  static constexpr int ROW = D * (F == kv::kBf16 ? 2 : 1);  // bytes of one key
  static constexpr int TOK = ROW == 256 ? 16 : ROW == 64 ? 64 : 32;  // tokens of one tile: 8 KB of keys and values
  // Warps of a block.  Heads of 64 leave registers for more than 8, which pays as long as loads are what a warp waits for: bf16
  // 12 (48 ragged GPT-2 rows 23.8 us, with 10 25.0, with 8 25.3; 32 x 4096 at 32/8 heads 50.0, 50.7, 51.1), int8 10 (48 ragged rows
  // 24.0 us, with 8 24.7, with 6 28.6; 32 x 4096 43.3, 43.2, 51.4), but e4m3 8 (32 x 4096 47.4 us, with 10 51.5, with 6 59.3).
  // Heads of 128 take 8: 32 x 4096 at 32/8 and at 32/4 heads bf16 91.0 and 52.0 us (with 10 92.2 and 53.0), int8 61 and 43.1 (10,
  // where 8 heads spill registers, 62 and 47.8; 6: 70.6 and 51.4), e4m3 70 and 43.2 (10, spilling, 78 and 49.0; 6: 86 and 52).
  static constexpr int WARPS = D == 128 ? 8 : F == kv::kBf16 ? 12 : F == kv::kInt8 ? 10 : 8;
  static constexpr int DATA = TOK * ROW, SCALES = F == kv::kBf16 ? 0 : TOK * 4;
  static constexpr int STAGE = 2 * (DATA + SCALES);
  static constexpr int STAGES = 2;  // one tile under way while the other is used
  static constexpr int PIECE = HEADS * (D + 2) * 4;  // o, m and sum of one row's piece
  static constexpr int THREADS = WARPS * 32;
  static constexpr int FACTORS = F == kv::kBf16 ? 0 : TOK * 16;  // per token: what its scales do to score and weight
  static constexpr int BOOK = 224;  // bookkeeping per warp
  static constexpr int SMEM = WARPS * (STAGES * STAGE + PIECE + FACTORS + BOOK);
};

__device__ __forceinline__ uint32_t smem_addr(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }

// 16 bytes, or zeros without reading `src`.
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool real, uint64_t policy) {
  asm volatile("cp.async.cg.shared.global.L2::cache_hint [%0], [%1], 16, %2, %3;" ::"r"(dst), "l"(src), "r"(real ? 16 : 0), "l"(policy) : "memory");
}
// Keys and values are read once per call: they should leave the L2 before what is needed again (code, tables, pieces).
__device__ __forceinline__ uint64_t stream_policy() {
  uint64_t p;
  asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(p));
  return p;
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ uint4 lds128(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ uint2 lds64(uint32_t a) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ void ldmatrix4t(uint32_t* r, uint32_t a) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(a)
               : "memory");
}

__device__ __forceinline__ void mma_bf16(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_f16(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_e4m3(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <bool SIGNED>
__device__ __forceinline__ void mma_int8(int* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if constexpr (SIGNED)
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// An integer accumulator that starts at these bits is, read as a float, 1.5 2^23 plus the sum (below 2^22 in magnitude).
constexpr int ZERO_BITS = 0x4b400000;
__device__ __forceinline__ float sum_of(int bits) { return __fadd_rn(__int_as_float(bits), -12582912.f); }

// Byte `BYTE` of four words as one word.
template <int BYTE>
__device__ __forceinline__ uint32_t gather_bytes(uint32_t x0, uint32_t x1, uint32_t x2, uint32_t x3) {
  constexpr uint32_t pick = BYTE | ((BYTE + 4) << 4);
  return __byte_perm(__byte_perm(x0, x1, pick), __byte_perm(x2, x3, pick), 0x5410);
}

// Four floats rounded to e4m3, and 16 times what the rounding left of each.
__device__ __forceinline__ uint32_t take_digit(float* x) {
  uint32_t word = 0;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const __nv_fp8x2_storage_t two = __nv_cvt_float2_to_fp8x2(make_float2(x[2 * h], x[2 * h + 1]), __NV_SATFINITE, __NV_E4M3);
    const float2 back = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2(two, __NV_E4M3)));
    x[2 * h] = 16.f * (x[2 * h] - back.x);
    x[2 * h + 1] = 16.f * (x[2 * h + 1] - back.y);
    word |= (uint32_t)two << (16 * h);
  }
  return word;
}

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t pack_half(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ float2 unpack_half(uint32_t x) { return __half22float2(*reinterpret_cast<const __half2*>(&x)); }
// Two e4m3 values (the first or the second two bytes) as fp16.
template <int PAIR>
__device__ __forceinline__ uint32_t half_pair(uint32_t x) {
  const __half2_raw v = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(PAIR == 0 ? x & 0xffffu : x >> 16), __NV_E4M3);
  return (uint32_t)v.x | ((uint32_t)v.y << 16);
}
__device__ __forceinline__ float2 unpack_bf16(uint32_t x) { return make_float2(__uint_as_float(x << 16), __uint_as_float(x & 0xffff0000u)); }

// A product that takes numbers below 2^-126 as they are, which the build's fast arithmetic does not.
__device__ __forceinline__ float times(float x, float y) {
  float z;
  asm("mul.rn.f32 %0, %1, %2;" : "=f"(z) : "f"(x), "f"(y));
  return z;
}
__device__ __forceinline__ float fast_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float fast_log2(float x) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// 2^d, d <= 0.  References of 8-bit caches contain value scales, which may lie 2^185 apart, and the sums their inverses: a
// sum takes the factor in two steps (WIDE), since it may be large where the factor alone is too small for fp32.
template <bool WIDE>
struct Factor {
  float first, second, all;
  __device__ explicit Factor(float d) {
    const float part = WIDE ? fmaxf(d, -100.f) : d;
    first = fast_exp2(part);
    second = WIDE ? fast_exp2(d - part) : 1.f;
    all = WIDE ? first * second : first;
  }
  __device__ __forceinline__ float operator()(float sum) const { return WIDE ? sum * first * second : sum * first; }
};

// log(2^m sum).  The power of two of the sum joins m, so that the logarithm is that of a number between 1 and 2.  Without a
// token m is -inf; a sum that is NaN stays so.
__device__ __forceinline__ float lse_of(float m, float sum) {
  const uint32_t u = __float_as_uint(sum);
  const float mantissa = __uint_as_float((u & 0x007fffffu) | 0x3f800000u);
  return fmaf(sum, 0.f, m + (float)((int)(u >> 23) - 127) + fast_log2(mantissa)) * LN2;
}

// A place on the line of tiles.  `rows` counts the rows of one sequence.
struct Cursor {
  int b, row, tile, tiles, n;
};

// Tokens of sequence b that the kernel attends to.
__device__ __forceinline__ int tokens_of(const Args& a, int b) {
  const long long most = (long long)a.width << a.pool.page_shift;
  const int n = max(a.lengths[b], 0);
  return n < most ? n : (int)most;
}

template <int TOK>
__device__ __forceinline__ void open_row(const Args& a, Cursor& c) {
  c.n = tokens_of(a, c.b);
  c.tiles = (c.n + TOK - 1) / TOK;
}

template <int TOK>
__device__ __forceinline__ void advance(const Args& a, Cursor& c, int rows) {
  if (++c.tile < c.tiles) return;
  c.tile = 0;
  if (++c.row < rows) return;
  c.row = 0;
  do {
    if (++c.b >= a.B) return;
    open_row<TOK>(a, c);
  } while (c.tiles == 0);
}

// Counts one more and returns the count before.  Releases what the block wrote before its last barrier, and acquires what the
// blocks that arrived earlier had written.
__device__ __forceinline__ unsigned arrive(unsigned* counter) {
  unsigned before;
  asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;" : "=r"(before) : "l"(counter) : "memory");
  return before;
}

// Of this block's shared memory, or of what other blocks wrote before they arrived.
__device__ __forceinline__ float load(const float* p) {
  float v;
  asm volatile("ld.relaxed.gpu.f32 %0, [%1];" : "=f"(v) : "l"(p) : "memory");
  return v;
}

// TWIN: rows of at most 4 heads (not of e4m3).
template <int F, int D, bool TWIN>
__global__ void __launch_bounds__(Shape<F, D>::THREADS, 1) decode_kernel(const __grid_constant__ Args a) {
  using S = Shape<F, D>;
  constexpr int TOK = S::TOK, GROUPS = TOK / 16, NT = D / 8, WARPS = S::WARPS;
  // Scores are in units of 2^SHIFT times the key's scale (at most 2^128 / 127) until that multiplies them: digits of the largest
  // queries are sums up to 2^37 before it does.
  constexpr int SHIFT = 6;
  constexpr uint32_t UNIT = F == kv::kInt8 ? 0x4f000000u : 0x3f800000u;  // what a weight of 1 is held as, 2^31 or 1, in bits
  // Value scales more than 2^RANGE below a bound of those of the row so far count as that, with a smaller f.  The bound
  // leaves room above the largest, so that it seldom moves.
  constexpr uint32_t RANGE = 60, SPARE = 4;
  extern __shared__ __align__(16) unsigned char smem[];
  struct Meta {
    int item;  // first tile of the row on the line
    int b, row, tile, count, tiles;
  };
  struct Job {      // pieces of one row to bring together
    int from, to;   // of the list of pieces
    int b, row;
    int item, tiles;
    bool begins, whole;  // whether they start with the row's first token, and whether they are all of the row
  };
  struct Shared {
    Meta meta[2 * WARPS];
    Job jobs[WARPS + 1];
    int count;
    bool shared_rows;  // whether a row of this block goes on in another one
  };
  static_assert(sizeof(Shared) <= WARPS * S::BOOK, "shared bookkeeping");
  unsigned char* const rings = smem;
  unsigned char* const pieces = smem + WARPS * S::STAGES * S::STAGE;
  Shared& sh = *reinterpret_cast<Shared*>(pieces + WARPS * (S::PIECE + S::FACTORS));

  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  const int g = lane / 4, c4 = lane % 4;
  const int group = a.H / a.pool.Hkv;               // query heads per key/value head
  const int chunks = (group + HEADS - 1) / HEADS;  // rows per key/value head
  const int rows = a.pool.Hkv * chunks;
  const auto kv_head_of = [&](int row) { return chunks == 1 ? row : row / chunks; };

  // ---- this warp's range of the line.  Every warp works it out for itself: sums of the tiles of 32 sequences at a time, a
  // lane for each sum, then the 32 sequences among which the range starts.  Nobody waits for another warp.
  const auto tiles_of = [&](int n) { return (n + TOK - 1) / TOK * rows; };
  const auto scan = [&](int v) {  // inclusive, over the lanes
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int other = __shfl_up_sync(0xffffffffu, v, o);
      if (lane >= o) v += other;
    }
    return v;
  };
  if (warp == 0) {  // sequences without tokens have no tiles: their results are written here
    for (int b = blockIdx.x; b < a.B; b += gridDim.x) {
      if (tokens_of(a, b) > 0) continue;
      for (int i = lane * 8; i < a.H * D; i += 256) *reinterpret_cast<uint4*>(a.out + (long long)b * a.H * D + i) = make_uint4(0, 0, 0, 0);
      if (a.lse != nullptr)
        for (int i = lane; i < a.H; i += 32) a.lse[(long long)b * a.H + i] = -INFINITY;
    }
  }
  int line = 0, base = 0, b0 = 0, mine, upto;
  int per_block = 0, block_from = 0, from = 0, count = 0;
  for (bool counted = false;;) {
    mine = 0;  // lane k: the tiles of sequences b0 + 32 k ... + 31
#pragma unroll 4
    for (int k = 0; k < 32; ++k) {
      if (b0 + 32 * k >= a.B) break;
      const int b = b0 + 32 * k + lane;
      const int sum = (int)__reduce_add_sync(0xffffffffu, b < a.B ? (uint32_t)tiles_of(tokens_of(a, b)) : 0u);
      if (lane == k) mine = sum;
    }
    upto = scan(mine);
    const int total = __shfl_sync(0xffffffffu, upto, 31);
    if (!counted) {
      line += total;
      b0 += 1024;
      if (b0 < a.B) continue;
      counted = true;
      // at least 8 tiles, a tile a warp: fewer, fuller blocks have fewer pieces to join, and rows of a power of two of tiles end
      // with a block
      per_block = max((int)((line + gridDim.x - 1) / gridDim.x), 8);
      block_from = (int)min((long long)line, (long long)per_block * blockIdx.x);
      const int block_to = min(line - block_from, per_block) + block_from;
      if (block_from >= block_to) return;
      const int per_warp = (block_to - block_from + WARPS - 1) / WARPS;
      from = block_from + warp * per_warp;
      count = max(0, min(per_warp, block_to - from));
      b0 = 0;
      if (a.B > 1024) continue;  // again from the first 1024, which are no longer at hand
    }
    if (count == 0 || from < base + total) break;
    base += total;
    b0 += 1024;
  }
  if (lane < 2) sh.meta[2 * warp + lane].count = 0;
  Cursor start{0, 0, 0, 1, 0};
  if (count > 0) {
    const int chunk = __popc(__ballot_sync(0xffffffffu, base + upto <= from));
    base += __shfl_sync(0xffffffffu, upto - mine, chunk);
    b0 += 32 * chunk;
    const int n = b0 + lane < a.B ? tokens_of(a, b0 + lane) : 0;
    const int reach = scan(tiles_of(n)), at = __popc(__ballot_sync(0xffffffffu, base + reach <= from));
    start.b = b0 + at;
    start.n = __shfl_sync(0xffffffffu, n, at);
    start.tiles = (start.n + TOK - 1) / TOK;
    const int in = from - (base + __shfl_sync(0xffffffffu, reach - tiles_of(n), at));
    start.row = in / start.tiles;
    start.tile = in - start.row * start.tiles;
  }
  unsigned char* const ring = rings + warp * S::STAGES * S::STAGE;
  const uint32_t ring_addr = smem_addr(ring);
  // Lanes g >= 4 work out head g - 4 once more, and their rows of the second product's operand take the last of the weights'
  // three terms.
  const bool last_term = TWIN && g >= HEADS / 2;  // (of int8: the last two of four)
  [[maybe_unused]] float4* const factors = reinterpret_cast<float4*>(pieces + WARPS * S::PIECE + warp * S::FACTORS);

  if (count > 0) {
    const uint64_t policy = stream_policy();
    Cursor load = start;
    Cursor use = load;
    int to_load = count;
    uint32_t held = 0;  // per stage: which groups of 16 tokens are in the pool
    // Pages are looked up 32 groups at a time, a window ahead of their use.
    constexpr int WINDOW = 32 / GROUPS;  // tiles
    const auto look_up = [&](const Cursor& c) {
      const int token = c.tile * TOK + lane * 16;
      return c.b < a.B && token < c.n ? a.table[c.b * a.table_row + (token >> a.pool.page_shift)] : -1;
    };
    const auto next_window = [&](Cursor c) {
      c.tile = min(c.tile + WINDOW, c.tiles) - 1;
      advance<TOK>(a, c, rows);
      return c;
    };
    int page = look_up(load), next_page = -1, window = load.tile;
    bool turn = false;  // the next tile opens a window
    const auto issue = [&](int stage) {
      if (to_load > 0) {
        const bool opens = turn;
        if (opens) {
          page = next_page;
          window = load.tile;
        }
        const uint32_t base = ring_addr + stage * S::STAGE;
        uint32_t bits = 0;
#pragma unroll
        for (int i = 0; i < GROUPS; ++i) {
          const int p = __shfl_sync(0xffffffffu, page, (load.tile - window) * GROUPS + i);
          const int token = load.tile * TOK + i * 16;
          const bool in_pool = p >= 0 && p < a.pool.pages;
          bits |= (uint32_t)in_pool << i;
          const long long first =
              in_pool ? (((long long)p * a.pool.Hkv + kv_head_of(load.row)) << a.pool.page_shift) + (token & ((1 << a.pool.page_shift) - 1)) : 0;
          const int real = in_pool ? load.n - token : 0;  // rows behind the sequence become zeros: 0 * NaN would not be 0
          const unsigned char* ks = static_cast<const unsigned char*>(a.pool.k) + first * S::ROW;
          const unsigned char* vs = static_cast<const unsigned char*>(a.pool.v) + first * S::ROW;
#pragma unroll
          for (int j = 0; j < S::ROW / 32; ++j) {
            constexpr int PER = S::ROW / 16;  // 16-byte pieces of a row
            const int q = j * 32 + lane, r = q / PER, ch = q % PER;
            const int kch = PER >= 8 ? ch ^ ((r & 1) << 2) : ch;
            const int vch = F == kv::kBf16 ? ch ^ (r & 7) : PER >= 8 ? ch ^ (((r >> 2) & 3) << 1) : ch ^ ((r >> 2) & 3);
            copy16(base + (i * 16 + r) * S::ROW + kch * 16, ks + q * 16, r < real, policy);
            copy16(base + S::DATA + (i * 16 + r) * S::ROW + vch * 16, vs + q * 16, r < real, policy);
          }
          if (F != kv::kBf16 && lane < 8) {
            const float* scales = (lane < 4 ? a.pool.k_scale : a.pool.v_scale) + first;
            copy16(base + 2 * S::DATA + (lane < 4 ? 0 : S::SCALES) + i * 64 + (lane & 3) * 16, scales + (lane & 3) * 4, in_pool, policy);
          }
        }
        held = (held & ~(0xfu << (4 * stage))) | (bits << (4 * stage));
        if (opens) next_page = look_up(next_window(load));
        advance<TOK>(a, load, rows);
        --to_load;
        turn = load.tile == 0 || load.tile == window + WINDOW;
      }
      copies_commit();
    };

    const Cursor ahead = next_window(load);

    // Per row: q as fragments of the first operand, the output's accumulators, and the softmax's state.
    constexpr int DIGITS = F == kv::kInt8 && !TWIN ? 3 : 2;  // 8 bits: of q, in one lane
    constexpr int QR = F == kv::kBf16 ? D / 8 : DIGITS * (D / 16);
    uint32_t q[QR];
    constexpr int PLACES = F == kv::kInt8 ? 2 : 4;  // of an accumulator; int8 adds up tiles in fp32 itself
    float o[NT][PLACES], m = -INFINITY, sum = 0.f, up = 1.f;  // up: what scores are multiplied by, also for the digits of q
    [[maybe_unused]] uint32_t least = 0;  // power of two that value scales count as at least, as bits of an exponent
    int row_tile = 0;          // the row's first tile in this warp
    bool opened = false, first_row = true;
    int row_start = from - use.tile;  // first tile of the row on the line

    // Turn i uses tile i; turn -1 starts the first tile's copies (from the same code as all others: what is fetched once is
    // slow) and opens its row meanwhile.
    static_assert(S::STAGES == 2, "one tile ahead");
    for (int i = -1; i < count; ++i) {
      if (i >= 0) {
        copies_wait<0>();
        __syncwarp();
      }
      issue((i + 1) & 1);
      if (!opened) {
        opened = true;
        row_tile = use.tile;
        m = -INFINITY;
        sum = 0.f;
        least = 0;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          o[t][0] = o[t][1] = 0.f;
          if constexpr (PLACES == 4) o[t][2] = o[t][3] = 0.f;
        }
        const int kv_head = kv_head_of(use.row), in_group = (use.row - kv_head * chunks) * HEADS + (last_term ? g - HEADS / 2 : g);
        const bool real = in_group < group;
        const __nv_bfloat16* src = a.q + use.b * a.q_seq + ((long long)kv_head * group + in_group) * a.q_head;
        // lane (g, c4) holds, of head g, the 16-byte pieces of a key row that it will load: piece 4 j + c4
        if constexpr (F == kv::kBf16) {
#pragma unroll
          for (int j = 0; j < D / 32; ++j) {
            const uint4 x = real ? *reinterpret_cast<const uint4*>(src + (j * 4 + c4) * 8) : make_uint4(0, 0, 0, 0);
            q[4 * j] = x.x, q[4 * j + 1] = x.y, q[4 * j + 2] = x.z, q[4 * j + 3] = x.w;
          }
        } else {
          float x[D / 4];
          uint32_t largest = 0;  // magnitude as bits: infinities and NaN above all numbers
#pragma unroll
          for (int j = 0; j < D / 64; ++j)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const uint4 raw = real ? *reinterpret_cast<const uint4*>(src + (j * 4 + c4) * 16 + h * 8) : make_uint4(0, 0, 0, 0);
              const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
              for (int r = 0; r < 4; ++r) {
                const float2 f = unpack_bf16(w[r]);
                x[16 * j + 8 * h + 2 * r] = f.x;
                x[16 * j + 8 * h + 2 * r + 1] = f.y;
                largest = max(largest, max(__float_as_uint(f.x) & 0x7fffffffu, __float_as_uint(f.y) & 0x7fffffffu));
              }
            }
          largest = max(largest, __shfl_xor_sync(0xffffffffu, largest, 1));
          largest = max(largest, __shfl_xor_sync(0xffffffffu, largest, 2));
          // the power of two that brings the largest magnitude into [1, 2): exact both ways, in two steps, since neither it nor
          // its reciprocal need be a float of its own
          const auto power = [](int e) { return __uint_as_float((uint32_t)(127 + e) << 23); };
          constexpr int BITS = F == kv::kInt8 ? 21 : 7;
          const int exponent = max(-126, (int)(largest >> 23) - 127), half = exponent / 2;
          const float down = power(BITS - half), rest = power(half - exponent);
          up = largest < 0x7f800000u ? a.scale_log2 * power(half) * power(exponent - half - BITS - SHIFT) : __int_as_float(0x7fc00000);
#pragma unroll
          for (int r = 0; r < D / 4; ++r) x[r] = times(x[r], rest);
#pragma unroll
          for (int r = 0; r < D / 16; ++r) {
            if constexpr (F == kv::kInt8) {
              // bytes of y + 0x808080, less 128 each, are its signed digits
              uint32_t y[4];
#pragma unroll
              for (int e = 0; e < 4; ++e) y[e] = (uint32_t)(__float2int_rn(x[4 * r + e] * down) + 0x808080);
              const uint32_t d0 = gather_bytes<2>(y[0], y[1], y[2], y[3]) ^ 0x80808080u;
              const uint32_t d1 = gather_bytes<1>(y[0], y[1], y[2], y[3]) ^ 0x80808080u;
              const uint32_t d2 = gather_bytes<0>(y[0], y[1], y[2], y[3]) ^ 0x80808080u;
              if constexpr (TWIN) {
                q[2 * r] = last_term ? d2 : d0;
                q[2 * r + 1] = last_term ? 0u : d1;
              } else {
                q[3 * r] = d0, q[3 * r + 1] = d1, q[3 * r + 2] = d2;
              }
            } else {
              float y[4] = {x[4 * r] * down, x[4 * r + 1] * down, x[4 * r + 2] * down, x[4 * r + 3] * down};
              q[2 * r] = take_digit(y);
              q[2 * r + 1] = take_digit(y);
            }
          }
        }
      }

      if (i < 0) {
        next_page = look_up(ahead);
        continue;
      }
      const int stage = i & 1;
      const uint32_t kb = ring_addr + stage * S::STAGE, vb = kb + S::DATA;
      const uint32_t in_pool = held >> (4 * stage);
      [[maybe_unused]] const float* const stage_scales = reinterpret_cast<const float*>(ring + stage * S::STAGE + 2 * S::DATA);

      // 8 bits: one lane per token works out what its scales do.  A value scale below the smallest that kv_cache_write leaves
      // counts as that one; one of 2^127 or more (it leaves at most 2^128 / 127) counts as NaN, which NaN and infinities stay.
      // Masked tokens get a finite score factor and an exponent of -inf.
      if constexpr (F != kv::kBf16) {
        bool fits = true;
#pragma unroll
        for (int i = lane; i < TOK; i += 32) {
          const bool real = ((in_pool >> (i / 16)) & 1u) && use.tile * TOK + i < use.n;
          const float ks = stage_scales[i], raw = stage_scales[TOK + i];
          const float vs = raw < kv::kMinScale ? kv::kMinScale : raw;
          const uint32_t u = __float_as_uint(vs), n = u >> 23;  // 2^(n - 127) f
          const float power = vs < 0x1p127f ? __uint_as_float(0x4b000000u | n) - (8388608.f + 127.f) : __int_as_float(0x7fc00000);
          factors[i] = make_float4(real ? ks * (float)(1 << SHIFT) : 0.f, real ? power : -INFINITY,
                                   real ? __uint_as_float(0x7f000000u - (u & 0x7f800000u)) : 0.f, __uint_as_float((u & 0x007fffffu) | UNIT));
          fits = fits && (!real || n - least <= RANGE);
        }
        // With a row's first tile, and then hardly ever: a value scale out of range moves the bound, or is brought within it.
        // (Asking costs 128 x 4097..8192 int8 8 us of 283; a reduction in every tile 15, exponents with room to spare their
        // last bits.)
        if (!__all_sync(0xffffffffu, fits)) {
          uint32_t largest = 0;
#pragma unroll
          for (int i = lane; i < TOK; i += 32) {
            const float power = factors[i].y;
            if (power > -127.f) largest = max(largest, (uint32_t)(power + 127.f));  // not masked, not NaN
          }
          largest = __reduce_max_sync(0xffffffffu, largest) + SPARE;
          if (largest > least + RANGE) least = largest - RANGE;
#pragma unroll
          for (int i = lane; i < TOK; i += 32) {
            float4& f = factors[i];
            const float bound = (float)((int)least - 127);
            if (f.y > -127.f && f.y < bound) {
              f.w *= fast_exp2(f.y - bound);
              f.y = bound;
              f.z = __uint_as_float((254u - least) << 23);
            }
          }
        }
        __syncwarp();
      }
      if constexpr (F == kv::kBf16) {
        // scores, in the accumulator's layout: head g, tokens 8 t + 2 c4 and + 1
        float acc[TOK / 8][4], s[TOK / 8][2];
#pragma unroll
        for (int t = 0; t < TOK / 8; ++t) acc[t][0] = acc[t][1] = acc[t][2] = acc[t][3] = 0.f;
#pragma unroll
        for (int j = 0; j < D / 32; ++j)
#pragma unroll
          for (int t = 0; t < TOK / 8; ++t) {
            const uint4 k = lds128(kb + (t * 8 + g) * S::ROW + (((j * 4 + c4) ^ ((g & 1) << 2)) * 16));
            mma_bf16(acc[t], q[4 * j], 0u, q[4 * j + 1], 0u, k.x, k.y);
            mma_bf16(acc[t], q[4 * j + 2], 0u, q[4 * j + 3], 0u, k.z, k.w);
          }
        float top = -INFINITY;
#pragma unroll
        for (int t = 0; t < TOK / 8; ++t) {
          const int token = use.tile * TOK + t * 8 + 2 * c4;
          const bool pool_ok = (in_pool >> (t / 2)) & 1u;
          s[t][0] = pool_ok && token < use.n ? times(acc[t][0], a.scale_log2) : -INFINITY;
          s[t][1] = pool_ok && token + 1 < use.n ? times(acc[t][1], a.scale_log2) : -INFINITY;
          top = fmaxf(top, fmaxf(s[t][0], s[t][1]));
        }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const float higher = fmaxf(m, ceilf(top));
        const float at = higher == -INFINITY ? 0.f : higher;  // nothing but masked tokens so far
        if (__any_sync(0xffffffffu, higher > m)) {
          const float keep = fast_exp2(m - at);
          sum *= keep;
#pragma unroll
          for (int t = 0; t < NT; ++t) o[t][0] *= keep, o[t][1] *= keep, o[t][2] *= keep, o[t][3] *= keep;
          m = higher;
        }
#pragma unroll
        for (int t = 0; t < TOK / 8; ++t)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            s[t][e] = fast_exp2(s[t][e] - at);
            sum += s[t][e];
          }
        // o += p v, the rounding's remainder of p in rows 8 to 15, what its rounding left in rows 4 to 7 or in a second product
#pragma unroll
        for (int kk = 0; kk < GROUPS; ++kk) {
          uint32_t hi[2], lo[2], rest[2];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float x = s[2 * kk + h][0], y = s[2 * kk + h][1];
            hi[h] = pack_bf16(x, y);
            const float2 back = unpack_bf16(hi[h]);
            lo[h] = pack_bf16(x - back.x, y - back.y);
            const float2 more = unpack_bf16(lo[h]);
            rest[h] = pack_bf16(x - back.x - more.x, y - back.y - more.y);
            if (last_term) hi[h] = rest[h], lo[h] = 0u;
          }
          const int mat = lane / 8, r = kk * 16 + (mat & 1) * 8 + (lane & 7);
          const uint32_t row = vb + r * S::ROW;
#pragma unroll
          for (int np = 0; np < NT / 2; ++np) {
            uint32_t v[4];
            ldmatrix4t(v, row + (((2 * np + (mat >> 1)) ^ (r & 7)) * 16));
            mma_bf16(o[2 * np], hi[0], lo[0], hi[1], lo[1], v[0], v[1]);
            mma_bf16(o[2 * np + 1], hi[0], lo[0], hi[1], lo[1], v[2], v[3]);
            if constexpr (!TWIN) {
              mma_bf16(o[2 * np], rest[0], 0u, rest[1], 0u, v[0], v[1]);
              mma_bf16(o[2 * np + 1], rest[0], 0u, rest[1], 0u, v[2], v[3]);
            }
          }
        }
      } else {
        // Column n of score tile i is the token place(i) + 4 (n / 2) + n % 2: the lane's scores of four tiles are then tokens
        // 4 c4 ... + 3 and 16 + 4 c4 ... + 3 of a block of 32, in the order of the second product's operand.
        constexpr int BLOCKS = TOK / 32;
        const auto place = [](int i) { return i / 4 * 32 + i % 4 / 2 * 16 + i % 2 * 2; };
        float s[TOK / 8][2];
#pragma unroll
        for (int i = 0; i < TOK / 8; ++i) {
          const uint32_t row = kb + (place(i) + 4 * (g >> 1) + (g & 1)) * S::ROW;
          if constexpr (F == kv::kInt8 && TWIN) {
            int x[4] = {ZERO_BITS, ZERO_BITS, ZERO_BITS, ZERO_BITS};
            const float first = last_term ? up : 65536.f * up;
#pragma unroll
            for (int j = 0; j < D / 64; ++j) {
              const uint4 k = lds128(row + ((D == 128 ? (j * 4 + c4) ^ ((g & 1) << 2) : c4) * 16));
              const uint32_t* d = q + 8 * j;
              mma_int8<true>(x, d[0], d[1], d[2], d[3], k.x, k.y);
              mma_int8<true>(x, d[4], d[5], d[6], d[7], k.z, k.w);
            }
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const float part = fmaf(sum_of(x[e]), first, 256.f * up * sum_of(x[e + 2]));  // (no second digit in the last lanes)
              s[i][e] = part + __shfl_xor_sync(0xffffffffu, part, 16);
            }
          } else if constexpr (F == kv::kInt8) {
            int x[4] = {ZERO_BITS, ZERO_BITS, ZERO_BITS, ZERO_BITS}, y[4] = {ZERO_BITS, ZERO_BITS, ZERO_BITS, ZERO_BITS};
#pragma unroll
            for (int j = 0; j < D / 64; ++j) {
              const uint4 k = lds128(row + ((D == 128 ? (j * 4 + c4) ^ ((g & 1) << 2) : c4) * 16));
              const uint32_t* d = q + 12 * j;
              mma_int8<true>(x, d[0], d[1], d[3], d[4], k.x, k.y);
              mma_int8<true>(y, d[2], 0u, d[5], 0u, k.x, k.y);
              mma_int8<true>(x, d[6], d[7], d[9], d[10], k.z, k.w);
              mma_int8<true>(y, d[8], 0u, d[11], 0u, k.z, k.w);
            }
#pragma unroll
            for (int e = 0; e < 2; ++e) s[i][e] = fmaf(sum_of(x[e]), 65536.f * up, fmaf(sum_of(x[e + 2]), 256.f * up, sum_of(y[e]) * up));
          } else {
            float x[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int j = 0; j < D / 64; ++j) {
              const uint4 k = lds128(row + ((D == 128 ? (j * 4 + c4) ^ ((g & 1) << 2) : c4) * 16));
              const uint32_t* d = q + 8 * j;
              mma_e4m3(x, d[0], d[1], d[2], d[3], k.x, k.y);
              mma_e4m3(x, d[4], d[5], d[6], d[7], k.z, k.w);
            }
#pragma unroll
            for (int e = 0; e < 2; ++e) s[i][e] = fmaf(x[e + 2], 0.0625f * up, x[e] * up);
          }
        }
        float inv[TOK / 8][2], rest[TOK / 8][2], top = -INFINITY;
#pragma unroll
        for (int i = 0; i < TOK / 8; ++i)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float4 f = factors[place(i) + 4 * c4 + e];
            s[i][e] = fmaf(s[i][e], f.x, f.y);
            inv[i][e] = f.z;
            rest[i][e] = f.w;
            top = fmaxf(top, s[i][e]);
          }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = ceilf(fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2)));
        const float higher = fmaxf(m, top), now = higher == -INFINITY ? 0.f : higher;  // nothing but masked tokens so far
        if (__any_sync(0xffffffffu, higher > m)) {
          const Factor<true> keep(m - now);
          sum = keep(sum);
#pragma unroll
          for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int e = 0; e < PLACES; ++e) o[t][e] *= keep.all;
          m = higher;
        }
        // lane (g, c4) takes dimensions g NT ... + NT - 1 of the tokens whose weights it has
        constexpr int WORDS = NT / 4;
        uint32_t w[BLOCKS][8][WORDS];
#pragma unroll
        for (int b = 0; b < BLOCKS; ++b)
#pragma unroll
          for (int x = 0; x < 8; ++x) {
            const int r = b * 32 + x / 4 * 16 + 4 * c4 + x % 4;
            if constexpr (D == 128) {
              const uint4 v = lds128(vb + r * S::ROW + ((g ^ (c4 << 1)) * 16));
              w[b][x][0] = v.x, w[b][x][1] = v.y, w[b][x][2] = v.z, w[b][x][3] = v.w;
            } else {
              const uint2 v = lds64(vb + r * S::ROW + ((g / 2 ^ c4) * 16) + (g & 1) * 8);
              w[b][x][0] = v.x, w[b][x][1] = v.y;
            }
          }
        if constexpr (F == kv::kInt8) {
          const float at = top == -INFINITY ? 0.f : top;  // of this tile
          const float share = fast_exp2(top - now);       // of the tile's weights
          float tile_sum = 0.f;
          uint32_t p[BLOCKS][2][4];  // digits of the weights of tokens 4 c4 ... and 16 + 4 c4 ..., which a TWIN lane has two of
#pragma unroll
          for (int b = 0; b < BLOCKS; ++b)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              uint32_t y[4];  // bytes are the digits
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const int i = 4 * b + 2 * h + e / 2;
                const float x = fast_exp2(s[i][e % 2] - at);
                tile_sum = fmaf(x, inv[i][e % 2], tile_sum);
                y[e] = __float2uint_rz(x * rest[i][e % 2]);
              }
              const auto take = [&](uint32_t pick, uint32_t& higher, uint32_t& lower) {  // two neighbouring bytes of each
                const uint32_t y01 = __byte_perm(y[0], y[1], pick), y23 = __byte_perm(y[2], y[3], pick);
                higher = __byte_perm(y01, y23, 0x7632);
                lower = __byte_perm(y01, y23, 0x5410);
              };
              take(last_term ? 0x5140 : 0x7362, p[b][h][0], p[b][h][1]);
              if constexpr (!TWIN) take(0x5140, p[b][h][2], p[b][h][3]);
            }
          sum = fmaf(share, tile_sum, sum);
          const float unit = share * 0x1p-31f, second = last_term ? unit : 65536.f * unit, first = 256.f * second;
#pragma unroll
          for (int y = 0; y < WORDS; ++y) {
            uint32_t v[BLOCKS][2][4];  // four tokens' bytes of each of four dimensions
#pragma unroll
            for (int b = 0; b < BLOCKS; ++b)
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const uint32_t t0 = w[b][4 * h][y], t1 = w[b][4 * h + 1][y], t2 = w[b][4 * h + 2][y], t3 = w[b][4 * h + 3][y];
                const uint32_t a01 = __byte_perm(t0, t1, 0x5140), a23 = __byte_perm(t0, t1, 0x7362);
                const uint32_t b01 = __byte_perm(t2, t3, 0x5140), b23 = __byte_perm(t2, t3, 0x7362);
                v[b][h][0] = __byte_perm(a01, b01, 0x5410);
                v[b][h][1] = __byte_perm(a01, b01, 0x7632);
                v[b][h][2] = __byte_perm(a23, b23, 0x5410);
                v[b][h][3] = __byte_perm(a23, b23, 0x7632);
              }
#pragma unroll
            for (int z = 0; z < 4; ++z) {
              int x[4] = {ZERO_BITS, ZERO_BITS, ZERO_BITS, ZERO_BITS};
#pragma unroll
              for (int b = 0; b < BLOCKS; ++b) mma_int8<false>(x, p[b][0][0], p[b][0][1], p[b][1][0], p[b][1][1], v[b][0][z], v[b][1][z]);
#pragma unroll
              for (int e = 0; e < 2; ++e) o[4 * y + z][e] = fmaf(sum_of(x[e]), first, fmaf(sum_of(x[e + 2]), second, o[4 * y + z][e]));
              if constexpr (!TWIN) {
                x[0] = x[1] = x[2] = x[3] = ZERO_BITS;
#pragma unroll
                for (int b = 0; b < BLOCKS; ++b) mma_int8<false>(x, p[b][0][2], p[b][0][3], p[b][1][2], p[b][1][3], v[b][0][z], v[b][1][z]);
#pragma unroll
                for (int e = 0; e < 2; ++e) o[4 * y + z][e] = fmaf(fmaf(sum_of(x[e]), 256.f, sum_of(x[e + 2])), unit, o[4 * y + z][e]);
              }
            }
          }
        } else {
          // in fp16, which holds e4m3 values exactly: p in rows 0 to 7, what its rounding left in rows 8 to 15
#pragma unroll
          for (int b = 0; b < BLOCKS; ++b)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              uint32_t hi[2], lo[2];
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const int i = 4 * b + 2 * h + e;
                const float x = fast_exp2(s[i][0] - now), y = fast_exp2(s[i][1] - now);
                sum = fmaf(x, inv[i][0], fmaf(y, inv[i][1], sum));
                const float px = x * rest[i][0], py = y * rest[i][1];
                hi[e] = pack_half(px, py);
                const float2 back = unpack_half(hi[e]);
                lo[e] = pack_half(px - back.x, py - back.y);
              }
#pragma unroll
              for (int y = 0; y < WORDS; ++y) {
                const uint32_t t0 = w[b][4 * h][y], t1 = w[b][4 * h + 1][y], t2 = w[b][4 * h + 2][y], t3 = w[b][4 * h + 3][y];
                const uint32_t a01 = __byte_perm(t0, t1, 0x5140), a23 = __byte_perm(t0, t1, 0x7362);
                const uint32_t b01 = __byte_perm(t2, t3, 0x5140), b23 = __byte_perm(t2, t3, 0x7362);
                mma_f16(o[4 * y], hi[0], lo[0], hi[1], lo[1], half_pair<0>(a01), half_pair<0>(b01));
                mma_f16(o[4 * y + 1], hi[0], lo[0], hi[1], lo[1], half_pair<1>(a01), half_pair<1>(b01));
                mma_f16(o[4 * y + 2], hi[0], lo[0], hi[1], lo[1], half_pair<0>(a23), half_pair<0>(b23));
                mma_f16(o[4 * y + 3], hi[0], lo[0], hi[1], lo[1], half_pair<1>(a23), half_pair<1>(b23));
              }
            }
        }
      }
      __syncwarp();  // the stage may be refilled

      const bool row_ends = use.tile + 1 == use.tiles, last = i + 1 == count;
      if (row_ends || last) {
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            if constexpr (PLACES == 4) o[t][e] += o[t][e + 2];
            if constexpr (TWIN) o[t][e] += __shfl_xor_sync(0xffffffffu, o[t][e], 16);
          }
        const auto value = [&](int t, int e) { return o[t][e]; };
        // where accumulator column n of tile t lies in the head's dimensions
        const auto dim = [&](int t, int e) { return F == kv::kBf16 ? t * 8 + 2 * c4 + e : (2 * c4 + e) * NT + t; };
        if (row_ends && row_tile == 0) {
          const int kv_head = kv_head_of(use.row), in_group = (use.row - kv_head * chunks) * HEADS + g;
          if (in_group < group) {
            const long long head = (long long)use.b * a.H + (long long)kv_head * group + in_group;
            const float norm = sum == 0.f ? 0.f : __fdividef(1.f, sum);
            __nv_bfloat16* dst = a.out + head * D;
            if constexpr (F == kv::kBf16) {
#pragma unroll
              for (int t = 0; t < NT; ++t)
                *reinterpret_cast<uint32_t*>(dst + dim(t, 0)) = pack_bf16(value(t, 0) * norm, value(t, 1) * norm);
            } else {
#pragma unroll
              for (int e = 0; e < 2; ++e)
#pragma unroll
                for (int t = 0; t < NT; t += 8) {
                  uint32_t x[4];
#pragma unroll
                  for (int y = 0; y < 4; ++y)
                    x[y] = pack_bf16(value(t + 2 * y, e) * norm, value(t + 2 * y + 1, e) * norm);
                  *reinterpret_cast<uint4*>(dst + dim(t, e)) = make_uint4(x[0], x[1], x[2], x[3]);
                }
            }
            if (a.lse != nullptr && c4 == 0) a.lse[head] = lse_of(m, sum);
          }
        } else {
          // A piece of a row.  One of the warp's first row goes to a place of its own, one of a later row ends the
          // range, so that the ring is free for it.
          const int which = first_row ? 0 : 1;
          if (which == 1) {
            copies_wait<0>();
            __syncwarp();
          }
          float* const piece = reinterpret_cast<float*>(which == 0 ? pieces + warp * S::PIECE : ring);
          // in the order of the accumulators: value (t, e) of every lane next to one another
#pragma unroll
          for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int e = 0; e < 2; ++e) piece[(2 * t + e) * 32 + lane] = value(t, e);
          if (c4 == 0) {
            piece[HEADS * D + g] = m;
            piece[HEADS * D + HEADS + g] = sum;
          }
          if (lane == 0) sh.meta[2 * warp + which] = Meta{row_start, use.b, use.row, row_tile, use.tile + 1 - row_tile, use.tiles};
          __syncwarp();
        }
        opened = first_row = false;
        row_start = from + i + 1;
      }
      advance<TOK>(a, use, rows);
    }
    copies_wait<0>();
  }
  __syncthreads();

  // ---- bring pieces of the same row together: first those of this block, which are neighbours, and then, if this block is the
  // last to arrive, those that other blocks left of its first and its last row.  One loop does both: the code of the
  // end of a block is fetched from afar, so that its length costs more than its steps.
  static_assert(2 * WARPS <= 32, "a lane per piece");
  constexpr int STEP = HEADS * (D + 2);  // floats of a piece
  const float** const list = reinterpret_cast<const float**>(rings + S::PIECE);  // behind the first warp's piece
  if (warp == 0) {
    const Meta mine = sh.meta[lane < 2 * WARPS ? lane : 0];
    const bool some = lane < 2 * WARPS && mine.count > 0;
    const uint32_t have = __ballot_sync(0xffffffffu, some), before = have & ((1u << lane) - 1);
    const int previous = __shfl_sync(0xffffffffu, mine.item, before ? 31 - __clz(before) : 0);
    const bool head = some && (before == 0 || previous != mine.item);
    const uint32_t heads = __ballot_sync(0xffffffffu, head), later = heads & ~((2u << lane) - 1);
    const uint32_t members = have & ~((1u << lane) - 1) & (later ? (1u << (__ffs(later) - 1)) - 1 : 0xffffffffu);
    const int last = members ? 31 - __clz(members) : lane;
    const int end = __shfl_sync(0xffffffffu, mine.tile + mine.count, last);
    const bool whole = mine.tile == 0 && end == mine.tiles;
    if (some) list[__popc(before)] = reinterpret_cast<const float*>(lane % 2 == 0 ? pieces + lane / 2 * S::PIECE : rings + lane / 2 * S::STAGES * S::STAGE);
    if (head)
      sh.jobs[__popc(heads & ((1u << lane) - 1))] =
          Job{__popc(before), __popc(before) + __popc(members), mine.b, mine.row, mine.item, mine.tiles, mine.tile == 0, whole};
    const bool shared_rows = __any_sync(0xffffffffu, head && !whole);
    if (lane == 0) {
      sh.count = __popc(heads);
      sh.shared_rows = shared_rows;
    }
  }
  __syncthreads();
  for (bool joining = false;; joining = true) {
    constexpr int VALUES = 4, UNITS = 2 * NT / VALUES;  // a warp takes this many values a lane, of one row, at a time
    for (int unit = warp; unit < sh.count * UNITS; unit += WARPS) {
      const Job job = sh.jobs[unit / UNITS];
      const int v0 = unit % UNITS * VALUES;
      float top = -INFINITY, total = 0.f, x[VALUES] = {};
      constexpr int BATCH = 4;  // pieces whose loads are under way together
      for (int i = job.from; i < job.to; i += BATCH) {
        float m[BATCH], l[BATCH], v[BATCH][VALUES], higher = top;
#pragma unroll
        for (int k = 0; k < BATCH; ++k) {
          const float* p = list[min(i + k, job.to - 1)];
          m[k] = load(p + HEADS * D + g);
          l[k] = load(p + HEADS * D + HEADS + g);
#pragma unroll
          for (int y = 0; y < VALUES; ++y) v[k][y] = load(p + (v0 + y) * 32 + lane);
        }
#pragma unroll
        for (int k = 0; k < BATCH; ++k) {
          if (i + k >= job.to) m[k] = -INFINITY;
          higher = fmaxf(higher, m[k]);
        }
        const float at = higher == -INFINITY ? 0.f : higher;
        const Factor<F != kv::kBf16> keep(top - at);
        top = higher;
        total = keep(total);
#pragma unroll
        for (int y = 0; y < VALUES; ++y) x[y] *= keep.all;
#pragma unroll
        for (int k = 0; k < BATCH; ++k) {
          const Factor<F != kv::kBf16> w(m[k] - at);
          total += w(l[k]);
#pragma unroll
          for (int y = 0; y < VALUES; ++y) x[y] = fmaf(w.all, v[k][y], x[y]);
        }
      }
      const int kv_head = kv_head_of(job.row), in_group = (job.row - kv_head * chunks) * HEADS + g;
      if (in_group >= group) continue;
      if (job.whole) {
        const long long head = (long long)job.b * a.H + (long long)kv_head * group + in_group;
        const float norm = total == 0.f ? 0.f : __fdividef(1.f, total);
#pragma unroll
        for (int y = 0; y < VALUES; ++y) {
          const int v = v0 + y, d = F == kv::kBf16 ? (v >> 1) * 8 + 2 * c4 + (v & 1) : (2 * c4 + (v & 1)) * NT + (v >> 1);
          a.out[head * D + d] = __float2bfloat16_rn(x[y] * norm);
        }
        if (a.lse != nullptr && v0 == 0 && c4 == 0) a.lse[head] = lse_of(top, total);
      } else {
        float* const out = a.partial + ((long long)blockIdx.x * 2 + (job.begins ? 1 : 0)) * STEP;
#pragma unroll
        for (int y = 0; y < VALUES; ++y) out[(v0 + y) * 32 + lane] = x[y];
        if (v0 == 0 && c4 == 0) {
          out[HEADS * D + g] = top;
          out[HEADS * D + HEADS + g] = total;
        }
      }
    }
    if (joining || !sh.shared_rows) return;
    __syncthreads();
    // A row that goes on behind its first block is that block's last one, so the block's number names the row's counter.
    if (warp == 0) {
      const Job job = sh.jobs[lane == 0 ? 0 : sh.count - 1];
      int first = 0, n = 0;
      bool won = false;
      if (lane < min(2, sh.count) && !job.whole) {
        first = job.item / per_block;
        n = (job.item + job.tiles - 1) / per_block - first + 1;
        won = arrive(a.arrived + first) == (unsigned)(n - 1);
        if (won) a.arrived[first] = 0;
      }
      const uint32_t wins = __ballot_sync(0xffffffffu, won);
      if (won) sh.jobs[lane == 1 && (wins & 1u) ? 1 : 0] = Job{0, n, job.b, job.row, first, n, true, true};
      __syncwarp();
      if (lane == 0) {
        sh.count = __popc(wins);
        if (wins == 3u) {  // the second row's pieces lie behind the first's
          sh.jobs[1].from = sh.jobs[0].to;
          sh.jobs[1].to += sh.jobs[0].to;
        }
      }
    }
    __syncthreads();
    for (int j = 0; j < sh.count; ++j) {
      const Job job = sh.jobs[j];
      // a row's first block left its piece in its second place, the others in their first
      for (int x = tid; x < job.tiles; x += S::THREADS) list[job.from + x] = a.partial + ((long long)(job.item + x) * 2 + (x == 0 ? 1 : 0)) * STEP;
    }
    __syncthreads();
  }
}

long long workspace_floats(int sms) { return (long long)sms * 2 * HEADS * (128 + 2); }
int workspace_counters(int sms) { return sms; }

template <int F, int D, bool TWIN>
static cudaError_t launch_as(const Args& a, int sms, cudaStream_t stream) {
  using S = Shape<F, D>;
  // dynamic shared memory beyond 48 KB is opted into once per device
  static unsigned long long opted = 0;
  int device = 0;
  cudaError_t err = cudaGetDevice(&device);
  if (err != cudaSuccess) return err;
  const unsigned long long bit = 1ull << (device & 63);
  if (!(__atomic_load_n(&opted, __ATOMIC_ACQUIRE) & bit)) {
    err = cudaFuncSetAttribute(decode_kernel<F, D, TWIN>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM);
    if (err != cudaSuccess) return err;
    __atomic_fetch_or(&opted, bit, __ATOMIC_RELEASE);
  }
  decode_kernel<F, D, TWIN><<<sms, S::THREADS, S::SMEM, stream>>>(a);
  return cudaGetLastError();
}

cudaError_t launch(const Args& a, int sms, cudaStream_t stream) {
  cudaError_t err = cudaSuccess;
  kv::by_format(a.pool, [&](auto f, auto d) {
    constexpr int F = decltype(f)::value, D = decltype(d)::value;
    if (F != kv::kFp8 && a.H / a.pool.Hkv <= HEADS / 2) err = launch_as<F, D, F != kv::kFp8>(a, sms, stream);
    else err = launch_as<F, D, false>(a, sms, stream);
  });
  return err;
}

}  // namespace paged
}  // namespace ht
