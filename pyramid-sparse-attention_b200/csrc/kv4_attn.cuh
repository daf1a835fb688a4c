// What the two kernels of the attention over the 4-bit cache (kv4_attn.cu, kv4_attn_rows.cu) share: how the work is laid out, and the arithmetic
// of codes.
#pragma once
#include <type_traits>

#include "kv4.cuh"
#include "kv4_ring.h"
#include "mma_sync.cuh"
#include "tc_common.cuh"

namespace psa {

struct AttnArgs {
  const void* q;
  int64_t q_stride[3], out_stride[3];   // batch, head, token; in elements
  const uint8_t* data;
  const int32_t *table, *lengths, *counts;
  void* out;
  float* lse;
  int32_t* status;
  int64_t pages;
  int batch, tokens, heads, kv_heads, group, width, page;   // group: query heads of a key head
  float scale;
  int unit_cells;      // what a unit's beginning and end cost, in tiles
  int least_cells;     // a block takes at least so many
  int row_tiles;       // of a request that brings all `tokens`
  int blocks;          // of the first kernel
  int2* owners;        // [batch][kv_heads][row_tiles]: first and last block of a unit (rows of a tile x a key head)
  float* parts;        // [blocks][2]: what a block has of a unit that began before it, and of one that goes on behind it
};

template <typename T>
__device__ __forceinline__ void write_row(const AttnArgs& a, int b, int head, int i, int d, float4 o, float top, float sum) {
  const float f = sum == 0.f ? 0.f : 1.f / sum;
  T* to = static_cast<T*>(a.out) + b * a.out_stride[0] + head * a.out_stride[1] + i * a.out_stride[2] + d;
  uint2 w;
  w.x = MmaOp<T>::pack(o.x * f, o.y * f);
  w.y = MmaOp<T>::pack(o.z * f, o.w * f);
  *reinterpret_cast<uint2*>(to) = w;
  if (a.lse && d == 0) a.lse[((int64_t)b * a.heads + head) * a.tokens + i] = sum == 0.f ? -INFINITY : 0.6931471805599453f * (top + log2f(sum));
}

constexpr int kWarps = 4, kTile = 16 * kWarps;   // slices and tokens of a tile
constexpr float kLowest = -3.4028234664e38f;   // reference of a row that has seen nothing: exp2(-inf - kLowest) is 0
// A weight is 2^(score - reference), and meets the steps of its token's values in f16.  A token's need is the largest of its steps; where its groups
// are constant and have none, 2^-64 of its values' size; and kLeastNeed at least.  A row's reference moves when a weight times its token's need
// is above 2^15, to where the largest of these products is 2^kHead: f16 has its full precision from 2^-14 to 2^16, so a product 2^-20 of the
// largest is still rounded to 11 bits.  A row looks at its own tokens alone: what it does not see, and what other rows see, changes no
// bit of it.
// Weights are up to 2^95 (f16 tensors: 2^63), 2^31 of them fit 32 bits, and so do as many of up to 2^79 times a lowest value.  Steps may be up to
// 2^100 (below 2^-126 weights are 0).  Where zeros have nearly all the weight, what is left of an output below 2^-80 of its values' size loses bits.
constexpr float kHead = 7.f, kMostLog2 = 15.f, kMost = 32768.f, kLowestShare = 5.421010862427522e-20f;
// f16: 2^-64 of the largest number; a step is 2^-24 or more.
template <typename T> constexpr float kLeastNeed = std::is_same<T, __half>::value ? 3.552713678800501e-15f : 8.271806125530277e-25f;   // 2^-48, 2^-80
// The smallest power of two that is not below x, or `least` if that is larger.
__device__ __forceinline__ float power_above(float least, float x) {
  return x > least ? __uint_as_float((__float_as_uint(x) + 0x7fffffu) & 0x7f800000u) : least;
}
// Sums of q meet the lowest values in two terms of 11 bits each (22 in all: off by 2^-22 of themselves): tf32 for bf16 tensors - two terms of bf16 would
// be 16 bits, which keys far from zero show - and f16 for f16 ones.  They are kept in units of scores, 2^-24 of q's operands - in f16,
// whose numbers end there, 2^12 times that.
// A weight times a step in one term of 11 bits costs a bf16 output a twentieth of its error: its own rounding is 2^-9, that of the weights 2^-12 of
// what the codes add (0.00175 of the output's norm instead of 0.00166-0.00168; with two terms 8 x 131071 tokens take 157 us instead of 133, 6 drafted
// tokens 71 instead of 58).  An f16 output would show it (0.00041 instead of 0.00021), so there it is two terms: 25 products a slice for 17.
template <typename T> constexpr int kWeightTerms = std::is_same<T, __half>::value ? 2 : 1;
template <typename T> constexpr float kSumScale = std::is_same<T, __half>::value ? 2.44140625e-4f : 1.f;

// A request's part of the line.  A unit - a key head with up to R rows - counts `unit_cells` more than it has tiles: what its rows cost before
// and after the tiles.
struct Span {
  int rows, row_tiles, tiles, cells, work;
  bool bad;   // a length or count out of range, and cut to it (the joining kernel reports it: here an atomic costs the start 0.2 us)
};
__device__ __forceinline__ Span span_of(const AttnArgs& a, int b, int rows_per_tile, int& length, int& count) {
  length = a.lengths[b];
  count = a.counts ? a.counts[b] : a.tokens;
  const int most = a.width * a.page;
  Span s;
  s.bad = length < 0 || length > most || count < 0 || count > a.tokens;
  length = min(max(length, 0), most);
  count = min(max(count, 0), a.tokens);
  s.rows = count * a.group;
  s.row_tiles = (s.rows + rows_per_tile - 1) / rows_per_tile;
  s.tiles = (int)(((uint32_t)length + kTile - 1) / kTile);   // lengths up to 2^31 - 16
  s.cells = s.tiles ? s.tiles + a.unit_cells : 0;
  s.work = s.cells * s.row_tiles * a.kv_heads;   // the entry point sees to it that the sum over all requests fits 32 bits
  return s;
}

// The line is shared out in stretches of `each` cells, the first `longer` of them one longer.
struct Shares {
  int blocks, each, longer;
  __device__ __forceinline__ Shares(int work, int most_blocks, int least) {
    blocks = min(most_blocks, (work + least - 1) / least);
    each = blocks ? work / blocks : 0;
    longer = work - each * blocks;
  }
  __device__ __forceinline__ int first(int i) const { return i * each + min(i, longer); }
  __device__ __forceinline__ int owner(int at) const {
    const int edge = longer * (each + 1);
    return at < edge ? at / (each + 1) : longer + (at - edge) / each;
  }
};

// The whole line's length, and the request that cell `first(block)` lies in with the place where that begins.  scan: THREADS / 32 + 2 words.
template <int THREADS>
__device__ __forceinline__ int line_of(const AttnArgs& a, int rows_per_tile, int* scan, int& request, int& base, Shares& shares) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int length, count, mine = 0;
  for (int b = threadIdx.x; b < a.batch; b += THREADS) mine += span_of(a, b, rows_per_tile, length, count).work;
  const int own0 = mine;   // of request threadIdx.x, where there are no more than threads
  int sum = mine;
#pragma unroll
  for (int d = 1; d < 32; d *= 2) {
    const int y = __shfl_up_sync(~0u, sum, d);
    if (lane >= d) sum += y;
  }
  if (lane == 31) scan[warp] = sum;
  __syncthreads();
  int work = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 32; ++w) work += scan[w];
  shares = Shares(work, gridDim.x, a.least_cells);
  request = base = 0;
  if ((int)blockIdx.x >= shares.blocks || a.batch == 1) return work;
  // whose tile it is: requests in rounds of one a thread
  const int first = shares.first(blockIdx.x);
  int before = 0;
  if (threadIdx.x == 0) scan[THREADS / 32] = scan[THREADS / 32 + 1] = 0;
  __syncthreads();
  for (int b0 = 0;; b0 += THREADS) {
    int own = own0;
    if (a.batch > THREADS) {
      const int b = b0 + threadIdx.x;
      own = b < a.batch ? span_of(a, b, rows_per_tile, length, count).work : 0;
      sum = own;
#pragma unroll
      for (int d = 1; d < 32; d *= 2) {
        const int y = __shfl_up_sync(~0u, sum, d);
        if (lane >= d) sum += y;
      }
      __syncthreads();
      if (lane == 31) scan[warp] = sum;
      __syncthreads();
    }
    int start = before + sum - own;
#pragma unroll
    for (int w = 0; w < THREADS / 32; ++w) {
      start += w < warp ? scan[w] : 0;
      before += scan[w];
    }
    if (first >= start && first < start + own) {
      scan[THREADS / 32] = b0 + threadIdx.x;
      scan[THREADS / 32 + 1] = start;
    }
    if (before > first || b0 + THREADS >= a.batch) break;
  }
  __syncthreads();
  request = scan[THREADS / 32];
  base = scan[THREADS / 32 + 1];
  return work;
}

// Lengths that another stream changes meanwhile give wrong outputs, but no wait without end and no access out of range: one warp reads
// them for those that meet at barriers, requests and blocks are bounded by what there is, waits for tiles run out, and a block ends when
// all that it copied has landed - also tiles that those who compute, with lengths of another moment, did not wait for.
//
// What a block has of a unit: tiles tile0 .. tile0 + tiles - 1 of key head `head` for the rows from row0 on.
struct Piece {
  int b, head, row0, rows, tile0, tiles, all_tiles, length, count;
  int end;    // the cell behind the unit
};
struct Walk {
  int b, base, at, last;   // the next cell, the block's end, the request it lies in and where that begins
  __device__ __forceinline__ bool next(const AttnArgs& a, int rows_per_tile, Piece& p) {
    while (at < last && b < a.batch) {
      const Span span = span_of(a, b, rows_per_tile, p.length, p.count);
      if (at >= base + span.work) {
        base += span.work;
        ++b;
        continue;
      }
      const int unit = (at - base) / span.cells, cell = at - base - unit * span.cells, cells = min(span.cells - cell, last - at);
      p.tile0 = max(cell - a.unit_cells, 0);
      p.tiles = max(cell + cells - a.unit_cells, 0) - p.tile0;
      p.end = at - cell + span.cells;
      at += cells;
      if (p.tiles == 0) continue;
      p.b = b;
      p.all_tiles = span.tiles;
      p.rows = span.rows;
      p.head = unit / span.row_tiles;
      p.row0 = (unit - p.head * span.row_tiles) * rows_per_tile;
      return true;
    }
    return false;
  }
};
// Two 32-bit operations in one instruction: the scheduler's slots are what these kernels run out of.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{.reg .b64 a, b, c, d; mov.b64 a, {%2, %3}; mov.b64 b, {%4, %5}; mov.b64 c, {%6, %7}; fma.rn.f32x2 d, a, b, c; mov.b64 {%0, %1}, d;}"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("{.reg .b64 a, b, d; mov.b64 a, {%2, %3}; mov.b64 b, {%4, %5}; mul.rn.f32x2 d, a, b; mov.b64 {%0, %1}, d;}"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{.reg .b64 a, b, d; mov.b64 a, {%2, %3}; mov.b64 b, {%4, %5}; add.rn.f32x2 d, a, b; mov.b64 {%0, %1}, d;}"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float2 both(float x) { return make_float2(x, x); }

// Codes of nibbles i and i + 4 as two f16 numbers: n 2^-24 for even i, n 2^-20 for odd ones.  (Subnormal numbers: a nibble is a number
// where it stands, with no exponent to add and no offset to take off again.)
__device__ __forceinline__ uint32_t codes(uint32_t w, int i) { return (i < 2 ? w : w >> 8) & (i & 1 ? 0x00f000f0u : 0x000f000fu); }
// The same of 15 - n.
__device__ __forceinline__ uint32_t rest(uint32_t w, int i) { return ~(i < 2 ? w : w >> 8) & (i & 1 ? 0x00f000f0u : 0x000f000fu); }
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// MmaOp<__half>'s product on an accumulator of zeros.
__device__ __forceinline__ void mma_new(float (&c)[4], const uint32_t (&a)[4], const uint32_t (&b)[2]) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
               : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]), "f"(0.f));
}
// What lies between two references of a row may be below the least number of 32 bits while what a weight becomes of it is not (rows of
// zeros, then of 10^15: weights of 2^87 become such of 2^-46), so it is applied in two halves.  The half of 2^x; y times 2^x.
__device__ __forceinline__ float half_of(float x) { return ex2(0.5f * x); }
__device__ __forceinline__ float faded(float y, float half) { return y * half * half; }
// Before parts of a row meet, each takes the size of its sum (a power of two) into its reference: what lies between those is what the parts
// count for, and below the least number of 32 bits is nothing.  2^-100 at least: 2^24 times what shrinks the sum is a number.
__device__ __forceinline__ float size_of(float sum) { return sum > 0.f ? (float)max((int)(__float_as_uint(sum) >> 23) - 127, -100) : 0.f; }
__device__ __forceinline__ uint32_t to_tf32(float x) {
  uint32_t y;
  asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(y) : "f"(x));
  return y;
}
// sum_g lo_g (sum of q over g) is a product too.  w0, w1: the parameters of group c (lane 4 r + c) of the tokens in rows r and r + 8; q: from
// row_operands.  f16: the words themselves are the operand, a group's step against 0; bf16: the lowest value is a word's upper half, a
// number of tf32 as it stands.
template <typename T> __device__ __forceinline__ void lowest_part(float (&x)[4], uint32_t w0, uint32_t w1, const uint32_t (&q)[2]) {
  if constexpr (std::is_same<T, __half>::value) {
    const uint32_t a[4] = {w0, w1, w0, w1};
    mma_new(x, a, q);
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] *= kSumScale<T>;
  } else {
    asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%4,%5}, {%6,%7}, {%8,%8,%8,%8};"
                 : "=f"(x[0]), "=f"(x[1]), "=f"(x[2]), "=f"(x[3]) : "r"(w0 & 0xffff0000u), "r"(w1 & 0xffff0000u), "r"(q[0]), "r"(q[1]), "f"(0.f));
  }
}
// step and lowest value of a group
template <typename T> __device__ __forceinline__ float2 param(uint32_t w);
template <> __device__ __forceinline__ float2 param<__nv_bfloat16>(uint32_t w) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
template <> __device__ __forceinline__ float2 param<__half>(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }

template <int N> struct Words { uint32_t w[N]; };
template <int N> __device__ __forceinline__ Words<N> lds(const uint8_t* p) {
  Words<N> r;
  if constexpr (N == 4) *reinterpret_cast<uint4*>(r.w) = *reinterpret_cast<const uint4*>(p);
  else if constexpr (N == 2) *reinterpret_cast<uint2*>(r.w) = *reinterpret_cast<const uint2*>(p);
  else r.w[0] = *reinterpret_cast<const uint32_t*>(p);
  return r;
}

// The need that parameter words stand for: of a token's groups, or of tokens.
template <typename T, int N> __device__ __forceinline__ float need_of(const Words<N>& p) {
  if constexpr (std::is_same<T, __half>::value) {
    __half2 most = *reinterpret_cast<const __half2*>(&p.w[0]);
#pragma unroll
    for (int g = 1; g < N; ++g) most = __hmax2(most, *reinterpret_cast<const __half2*>(&p.w[g]));
    return fmaxf(__low2float(most), kLeastNeed<T>);
  } else {
    __nv_bfloat162 most = __habs2(*reinterpret_cast<const __nv_bfloat162*>(&p.w[0]));
#pragma unroll
    for (int g = 1; g < N; ++g) most = __hmax2(most, __habs2(*reinterpret_cast<const __nv_bfloat162*>(&p.w[g])));
    const float2 m = param<T>(*reinterpret_cast<const uint32_t*>(&most));
    return fmaxf(fmaxf(m.x, kLeastNeed<T>), m.y * kLowestShare);
  }
}
// log2 of the smallest power of two that is not below a need.
__device__ __forceinline__ float log2_above(float need) { return (float)((int)(__float_as_uint(need) + 0x7fffffu >> 23) - 127); }

// A lane's operands of a row of q (lane 4 r + c: row r of eight), from its row's start plus 8 c channels, or of no row: q as f16, times the
// power of two that brings the row's largest value to 2^14 - exact for all that matters to a score; channels 4 i + 1 and 4 i + 3 meet
// codes of 16 times the unit.  sum: lowest_part's operand, the sum of q over group c in two terms.  Returns the power of two.
template <typename T, int D, int G>
__device__ __forceinline__ float row_operands(const T* from, bool in, uint32_t (&w)[D / 32][2][2], uint32_t (&sum)[2]) {
  constexpr int NG = D / G, NB = D / 32;
  const int c = threadIdx.x & 3;
  float2 e[NB][4];
  float most = 0.f, sums[NG];
#pragma unroll
  for (int i = 0; i < NB; ++i) {
    const uint4 x = in ? *reinterpret_cast<const uint4*>(from + 32 * i) : make_uint4(0, 0, 0, 0);
    e[i][0] = param<T>(x.x), e[i][1] = param<T>(x.y), e[i][2] = param<T>(x.z), e[i][3] = param<T>(x.w);
#pragma unroll
    for (int k = 0; k < 4; ++k) most = fmaxf(most, fmaxf(fabsf(e[i][k].x), fabsf(e[i][k].y)));
  }
  most = fmaxf(most, __shfl_xor_sync(~0u, most, 1));
  most = fmaxf(most, __shfl_xor_sync(~0u, most, 2));
  const int up = most > 0.f && isfinite(most) ? min(max(14 - ilogbf(most), -120), 120) : 0;
  const float grow = __int_as_float((127 + up) << 23);
#pragma unroll
  for (int i = 0; i < NB; ++i) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      w[i][k][0] = MmaOp<__half>::pack(e[i][k].x * grow, e[i][k + 2].x * grow);
      w[i][k][1] = MmaOp<__half>::pack(e[i][k].y * (grow * 0.0625f), e[i][k + 2].y * (grow * 0.0625f));
    }
    const float x = ((e[i][0].x + e[i][0].y) + (e[i][1].x + e[i][1].y)) + ((e[i][2].x + e[i][2].y) + (e[i][3].x + e[i][3].y));
    if (i % (G / 32) == 0) sums[i / (G / 32)] = x;
    else sums[i / (G / 32)] += x;
  }
  float x = 0.f;
#pragma unroll
  for (int g = 0; g < NG; ++g) {
    sums[g] += __shfl_xor_sync(~0u, sums[g], 1);
    sums[g] += __shfl_xor_sync(~0u, sums[g], 2);
    x = c == g ? sums[g] * (grow * 5.9604644775390625e-8f / kSumScale<T>) : x;
  }
  if constexpr (std::is_same<T, __half>::value) {
    const float high = Elem<T>::to_f(Elem<T>::from_f(x));
    sum[0] = MmaOp<T>::pack(0.f, high);
    sum[1] = MmaOp<T>::pack(0.f, x - high);
  } else {
    sum[0] = to_tf32(x);
    sum[1] = to_tf32(x - __uint_as_float(sum[0]));
  }
  return grow;
}

// Copies a tile of a unit into `to`: lanes of one warp.  whole: pages hold whole tiles, a copy each; else one for every slice.  The lanes
// look up the pages of 32 tiles (whole) or 32 slices at a time.
struct Lookup {
  int from;   // the slice in the cache that this lane is to copy from, -1: none
  __device__ __forceinline__ void look(const AttnArgs& a, const Piece& p, int tile, bool whole, int last_slice) {
    const int s = (p.tile0 + tile) * kWarps + (threadIdx.x & 31) * (whole ? kWarps : 1), per_page = a.page / 16;
    from = -1;
    if (s < last_slice) {
      const int in_page = s / per_page, page = a.table[(int64_t)p.b * a.width + in_page];
      if (page >= 0 && page < a.pages) from = (page * a.kv_heads + p.head) * per_page + s - in_page * per_page;
      else report(a.status, PSA_ERR_ARG);
    }
  }
  // Tile `tile` of the piece, of which `slices` slices are there, to `to`; valid: a bit for every slice that is.
  template <int SLICE, typename V>
  __device__ __forceinline__ void copy(const AttnArgs& a, int tile, bool whole, int slices, uint8_t* to, uint64_t* full, volatile V* valid) const {
    const int lane = threadIdx.x & 31, n = min(kWarps, slices);
    if (whole) {   // the lane that looked the page up does it all
      if (lane == (tile & 31)) {
        const int bytes = from >= 0 ? n * SLICE : 0;
        *valid = (V)(from >= 0 ? (1u << n) - 1 : 0u);
        tc::mbar_arrive_expect_tx(full, bytes);
        if (bytes) tc::bulk_load_a(tc::smem_u32(to), a.data + (int64_t)from * SLICE, bytes, tc::smem_u32(full));
      }
      return;
    }
    const int k = (tile & 7) * kWarps;
    const uint32_t bits = __ballot_sync(~0u, from >= 0) >> k & ((1u << n) - 1);
    if (lane == k) {
      *valid = (V)bits;
      tc::mbar_arrive_expect_tx(full, __popc(bits) * SLICE);
    }
    __syncwarp();
    if (lane >= k && lane < k + n && from >= 0)
      tc::bulk_load_a(tc::smem_u32(to + (lane - k) * SLICE), a.data + (int64_t)from * SLICE, SLICE, tc::smem_u32(full));
  }
};

// The kernel for more than 16 rows a key head (kv4_attn_rows.cu), launched.
template <typename T, int D, int G> int launch_rows(const AttnArgs& a, int rows_per_tile, cudaStream_t st);
__host__ __device__ constexpr int blocks_of(int rows) { return rows <= 8 ? 3 : rows == 24 ? 4 : rows == 32 ? 3 : 2; }   // of an SM, by the registers that rows take

}  // namespace psa
