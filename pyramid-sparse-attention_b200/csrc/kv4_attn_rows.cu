// Attention over the 4-bit cache for more than 16 query rows a key head (kv4_attn.cu has the arithmetic, and the kernel for fewer): drafted
// tokens, pieces of a prompt.
//
// A code is decoded once for 24 or 32 rows, in a warp that carries few outputs.  Four warps share a tile of 64 tokens twice: first a slice's 16
// tokens each, for the scores; then 32 channels each (at head_dim 64: 32 channels of two slices), for the outputs.  The weights times the
// steps pass through shared memory.  So a warp carries outputs of 32 channels instead of 128: 16 warps with 24 rows each fit on an SM, or
// 12 with 32; for 48 rows eight warps take half of them each.  All references of a row are one for the block, and move together.  The first
// warp copies tiles ahead: when the block meets between a tile's scores and outputs, the tile before it is done with.
//
// 5 requests of 20000 tokens, 28 heads on 4, head_dim 128, groups of 64, bf16: 3 new tokens 37-38 us (as 32 rows 45, as two units of 16 in the other
// kernel 53), 4 new ones 44 (eight warps with 16 rows each 50), 6 new ones 59 (as two units of 24 59; units of 16 in the other kernel 78;
// four warps with 48 rows each 78: 168 registers, 8 warps on an SM, 36 % of the issue slots).  6 at 80000 tokens: 506 instructions for 24
// rows and 16 tokens, half of the issue slots, tensor pipe 41 % (one m16n8k16 every 8 cycles: 576 TFLOP/s is what mma.sync has).  For 16
// rows the other kernel is as good (32 us, 33 here).  Pieces of a prompt, 48 rows a unit: 64 new tokens of one request of 32768 189 us, 256 of
// them 661 (181 TFLOP/s of the pairs that are seen), 2048 of 2048 458: each unit decodes the cache again, and goes through all of the
// request's tiles whatever its rows see.
#include "kv4_attn.cuh"

namespace psa {
namespace {

template <typename T, int D, int G, int NT, int HALVES>
struct Shape {
  using L = Kv4<D, G>;
  static constexpr int kHalves = HALVES, kThreads = 32 * kWarps * HALVES;
  static constexpr int kTiles = NT * kHalves, kRows = 8 * kTiles, kTerms = kWeightTerms<T>;   // 8-row tiles
  static constexpr int kTileBytes = kWarps * L::kSlice;
  static constexpr int kParts = kWarps / L::kBlocks;                               // warps that share a block of channels and its rows
  // Weights times the steps of a group: [terms][groups][slices][kTiles] matrices of 16 tokens x 8 rows.  Two buffers spare a barrier a tile.
  static constexpr int kWeights = kTerms * L::kGroups * kWarps * kTiles * 256, kBuffers = kWeights <= 8192 * HALVES ? 2 : 1;
  static constexpr int kStages = HALVES == 2 ? (D == 128 ? 4 : 6) : D == 64 ? 5 : kWeights > 16384 ? 2 : 3;   // tiles of the ring
  static constexpr int kOutRow = D + 4;                                            // floats; 4 more spread the banks
  static constexpr int kOuts = kParts * kRows * kOutRow * 4;                       // after the last tile: [parts][rows][kOutRow],
  static constexpr int kTotals = kWarps * (L::kGroups + 1) * kRows * 4;            // [slices][middle values of the groups, sums][rows]
  static constexpr int kArea = kBuffers * kWeights > kOuts + kTotals ? kBuffers * kWeights : kOuts + kTotals;
  static constexpr int kQ = kStages * kTileBytes + kArea;                          // [kTiles][blocks][lanes] operands of q, 16 bytes
  static constexpr int kQSum = kQ + kTiles * L::kBlocks * 512;                     // [kTiles][lanes] operands of its sums, 8 bytes
  static constexpr int kColumns = kQSum + kTiles * 256;                            // [row pairs] {factors to log2, keys that the rows see}
  static constexpr int kRise = kColumns + kRows * 8;                               // [slices][rows] scores that ask for a higher reference
  static constexpr int kBars = kRise + kWarps * kRows * 4;                         // full
  static constexpr int kMore = kBars + kStages * 8;                                // scan[10], abort, valid[stages]
  static constexpr int kBytes = kMore + (11 + kStages) * 4;
  static constexpr int64_t kPart = (int64_t)kRows * (D + 2);                       // scratch: output rows, and {reference, sum} of each
};

// 8 x 8 matrices of 16-bit numbers between a warp's registers (lane 4 r + c: row r, columns 2 c and 2 c + 1) and shared memory, a row's 16
// bytes at each lane's address; loads give the transposed matrices.
__device__ __forceinline__ void put4(uint32_t at, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("stmatrix.sync.aligned.m8n8.x4.shared.b16 [%0], {%1,%2,%3,%4};" ::"r"(at), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ void put2(uint32_t at, uint32_t a, uint32_t b) {
  asm volatile("stmatrix.sync.aligned.m8n8.x2.shared.b16 [%0], {%1,%2};" ::"r"(at), "r"(a), "r"(b) : "memory");
}
__device__ __forceinline__ void get4(uint32_t at, uint32_t& a, uint32_t& b, uint32_t& c, uint32_t& d) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(a), "=r"(b), "=r"(c), "=r"(d) : "r"(at) : "memory");
}
__device__ __forceinline__ void get2(uint32_t at, uint32_t& a, uint32_t& b) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x2.trans.shared.b16 {%0,%1}, [%2];" : "=r"(a), "=r"(b) : "r"(at) : "memory");
}

// What a warp carries of its rows.  Lane 4 r + c has rows 8 nt + 2 c + {0, 1} of the warp's: of the scores of its tokens, and of the outputs of
// its channels.
template <typename T, int D, int G, int NT>
struct Rows {
  float2 ref[NT];               // log2, negated
  float2 sum[NT];
  float2 mid[NT][D / G];        // the share of the output that the groups' middle values give
  float out[NT][2][4];          // of channels 4 i, 4 i + 2 (first) and 4 i + 1, 4 i + 3: times 2^-24 and 2^-20
};

// Scores of a slice's 16 tokens and the warp's rows, from 8-row tile `tile0` on: rows of x are the tokens r/2 + 4 (r % 2) and that + 8.
template <typename T, int D, int G, int NT, int HALVES>
__device__ __forceinline__ void score(float (&x)[NT][4], int tile0, const uint8_t* smem, const uint8_t* slice) {
  using L = Kv4<D, G>;
  using S = Shape<T, D, G, NT, HALVES>;
  constexpr int NG = L::kGroups, NB = L::kBlocks, BG = G / 32;   // 32-channel blocks of a group
  const int lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;
  {
    const uint8_t* p = slice + L::kParams + (c < NG ? c : 0) * 4;
    const uint32_t w0 = lds<1>(p + r * NG * 4).w[0], w1 = lds<1>(p + (r + 8) * NG * 4).w[0];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) lowest_part<T>(x[nt], w0, w1, lds<2>(smem + S::kQSum + ((tile0 + nt) * 32 + lane) * 8).w);
  }
  const Words<NB> k0 = lds<NB>(slice + r * L::kRow + c * NB * 4), k1 = lds<NB>(slice + (r + 8) * L::kRow + c * NB * 4);
  const Words<NG> p0 = lds<NG>(slice + L::kParams + r * NG * 4), p1 = lds<NG>(slice + L::kParams + (r + 8) * NG * 4);
#pragma unroll
  for (int g = 0; g < NG; ++g) {
    float acc[NT][4];
#pragma unroll
    for (int i = 0; i < BG; ++i) {
      const int b = g * BG + i;
      const uint32_t w0 = k0.w[b], w1 = k1.w[b];
      const uint32_t a0[4] = {codes(w0, 0), codes(w1, 0), codes(w0, 1), codes(w1, 1)}, a1[4] = {codes(w0, 2), codes(w1, 2), codes(w0, 3), codes(w1, 3)};
#pragma unroll
      for (int k = 0; k < 2; ++k)   // one product of every row tile after the other: none waits for the one before it
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const Words<2> q = lds<2>(smem + S::kQ + (((tile0 + nt) * NB + b) * 32 + lane) * 16 + k * 8);
          if (i == 0 && k == 0) mma_new(acc[nt], a0, q.w);
          else MmaOp<__half>::run(acc[nt], k ? a1 : a0, q.w);
        }
    }
    const float s0 = param<T>(p0.w[g]).x, s1 = param<T>(p1.w[g]).x;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int j = 0; j < 4; j += 2) {
        const float2 y = fma2(both(j ? s1 : s0), make_float2(acc[nt][j], acc[nt][j + 1]), make_float2(x[nt][j], x[nt][j + 1]));
        x[nt][j] = y.x, x[nt][j + 1] = y.y;
      }
  }
}

// Weights e of a slice's tokens: into the sums and the shares of the middle values (count), and times the steps of each group to `to`, the
// place of the slice's first matrix of the warp's rows.  MASKED: nothing that a row does not see counts, NaN or not.
template <typename T, int D, int G, int NT, int HALVES, bool MASKED>
__device__ __forceinline__ void weigh(Rows<T, D, G, NT>& s, const float (&e)[NT][4], bool count, const float4* columns, const uint8_t* slice, int token,
                                      uint32_t to) {
  using L = Kv4<D, G>;
  using S = Shape<T, D, G, NT, HALVES>;
  constexpr int NG = L::kGroups, kTerms = S::kTerms, kGroup = kWarps * S::kTiles * 256, kTerm = NG * kGroup;
  const int lane = threadIdx.x & 31, r = lane >> 2;
  const Words<NG> p0 = lds<NG>(slice + L::kHalf + L::kParams + r * NG * 4), p1 = lds<NG>(slice + L::kHalf + L::kParams + (r + 8) * NG * 4);
  uint32_t hidden[NT] = {};
  if constexpr (MASKED) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const float4 w = columns[4 * nt];
#pragma unroll
      for (int j = 0; j < 4; ++j) hidden[nt] |= token + 8 * (j >> 1) >= __float_as_int(j & 1 ? w.w : w.z) ? 1u << j : 0u;
    }
  }
  if (count) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) s.sum[nt] = add2(add2(s.sum[nt], make_float2(e[nt][0], e[nt][1])), make_float2(e[nt][2], e[nt][3]));
  }
#pragma unroll
  for (int g = 0; g < NG; ++g) {
    const float2 u0 = param<T>(p0.w[g]), u1 = param<T>(p1.w[g]);
    // a slice's first eight tokens: lo + s n; the others: hi - s (15 - n)
    const float ends[2] = {u0.y, fmaf(15.f, u1.x, u1.y)};
    uint32_t w[kTerms][NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const float2 e0 = make_float2(e[nt][0], e[nt][1]), e1 = make_float2(e[nt][2], e[nt][3]);
      const float2 y0 = mul2(e0, both(u0.x)), y1 = mul2(e1, both(-u1.x));
      float y[4] = {y0.x, y0.y, y1.x, y1.y};
      if constexpr (MASKED) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          float& mid = j & 1 ? s.mid[nt][g].y : s.mid[nt][g].x;
          if (hidden[nt] >> j & 1) y[j] = 0.f;
          else if (count) mid = fmaf(e[nt][j], ends[j >> 1], mid);
        }
      } else {
        s.mid[nt][g] = fma2(e1, both(ends[1]), fma2(e0, both(ends[0]), s.mid[nt][g]));
      }
#pragma unroll
      for (int k = 0; k < kTerms; ++k) {
        float first[4];   // 11 bits, cut off where another term follows
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          first[j] = k + 1 < kTerms ? __uint_as_float(__float_as_uint(y[j]) & 0xffffe000u) : y[j];
          y[j] -= first[j];
        }
        w[k][nt][0] = MmaOp<__half>::pack(first[0], first[1]);
        w[k][nt][1] = MmaOp<__half>::pack(first[2], first[3]);
      }
    }
#pragma unroll
    for (int k = 0; k < kTerms; ++k) {
#pragma unroll
      for (int nt = 0; nt + 1 < NT; nt += 2)
        put4(to + k * kTerm + g * kGroup + nt * 256 + lane * 16, w[k][nt][0], w[k][nt][1], w[k][nt + 1][0], w[k][nt + 1][1]);
      if constexpr (NT % 2) put2(to + k * kTerm + g * kGroup + (NT - 1) * 256 + (lane & 15) * 16, w[k][NT - 1][0], w[k][NT - 1][1]);
    }
  }
}

// Scores (times factors, less references) to weights, and nothing for what a row does not see.
template <bool MASKED, int NT>
__device__ __forceinline__ void weights(float (&e)[NT][4], const float (&x)[NT][4], const float2 (&ref)[NT], const float4* columns, int token) {
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const float4 w = columns[4 * nt];
#pragma unroll
    for (int j = 0; j < 4; j += 2) {
      const float2 y = fma2(make_float2(x[nt][j], x[nt][j + 1]), make_float2(w.x, w.y), ref[nt]);
      e[nt][j] = ex2(MASKED && token + 4 * j >= __float_as_int(w.z) ? -INFINITY : y.x);
      e[nt][j + 1] = ex2(MASKED && token + 4 * j >= __float_as_int(w.w) ? -INFINITY : y.y);
    }
  }
}

// Scores and weights of the warp's 16 tokens of a tile; true, and scores in e, where a weight times a step could leave f16 and the references
// have to move first - which is seldom.
template <typename T, int D, int G, int NT, int HALVES, bool MASKED>
__device__ __forceinline__ bool first_try(Rows<T, D, G, NT>& s, float (&e)[NT][4], int tile0, uint8_t* smem, const uint8_t* slice, int token, uint32_t to) {
  using L = Kv4<D, G>;
  using S = Shape<T, D, G, NT, HALVES>;
  constexpr int NG = L::kGroups;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, r = lane >> 2, c = lane & 3;
  const float4* columns = reinterpret_cast<const float4*>(smem + S::kColumns) + 4 * tile0 + c;   // of rows 2 c and 2 c + 1
  score<T, D, G, NT, HALVES>(e, tile0, smem, slice);
  // token by token, in the other kernel's words (the largest need kept: 3 new tokens of 5 x 20000 39 us instead of 38, groups of 32 43.6 instead of 41.2)
  const uint8_t* p = slice + L::kHalf + L::kParams + r * NG * 4;
  const float need[2] = {need_of<T, NG>(lds<NG>(p)), need_of<T, NG>(lds<NG>(p + 8 * NG * 4))};
  float w[NT][4], top[2] = {0.f, 0.f};
  weights<MASKED, NT>(w, e, s.ref, columns, token);
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int j = 0; j < 4; ++j) top[j >> 1] = fmaxf(top[j >> 1], w[nt][j]);
  const bool rises = __any_sync(~0u, fmaxf(top[0] * need[0], top[1] * need[1]) > kMost);
  if (rises) {
    float* rise = reinterpret_cast<float*>(smem + S::kRise) + warp % kWarps * S::kRows + 8 * tile0;
    const float up[2] = {log2_above(need[0]), log2_above(need[1])};
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const float4 of = columns[4 * nt];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float m = -INFINITY, over = 0.f;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          over = fmaxf(over, w[nt][2 * i + j] * need[i]);
          if (!MASKED || token + 8 * i < __float_as_int(j ? of.w : of.z)) m = fmaxf(m, e[nt][2 * i + j] * (j ? of.y : of.x) + up[i]);
        }
#pragma unroll
        for (int d = 4; d < 32; d *= 2) {
          m = fmaxf(m, __shfl_xor_sync(~0u, m, d));
          over = fmaxf(over, __shfl_xor_sync(~0u, over, d));
        }
        if (r == 0) rise[8 * nt + 2 * c + j] = over > kMost ? m : -INFINITY;
      }
    }
  } else {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int j = 0; j < 4; ++j) e[nt][j] = w[nt][j];
    weigh<T, D, G, NT, HALVES, MASKED>(s, e, true, columns, slice, token, to);
  }
  return rises;
}

// All warps' references to where the ones that rise want them, and this warp's weights again.
template <typename T, int D, int G, int NT, int HALVES>
__device__ __forceinline__ void raise(Rows<T, D, G, NT>& s, float (&e)[NT][4], bool rises, int tile0, uint8_t* smem, const uint8_t* slice, int token,
                                      uint32_t to) {
  using S = Shape<T, D, G, NT, HALVES>;
  constexpr int NG = D / G;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = lane & 3;
  const float4* columns = reinterpret_cast<const float4*>(smem + S::kColumns) + 4 * tile0 + c;
  float* rise = reinterpret_cast<float*>(smem + S::kRise) + 8 * tile0;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      float m = -INFINITY;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) m = fmaxf(m, rise[w * S::kRows + 8 * nt + 2 * c + j]);
      float& was = j ? s.ref[nt].y : s.ref[nt].x;
      const float ref = fmaxf(m - kHead, -was), fade = half_of(-was - ref);
      was = -ref;
      float& sum = j ? s.sum[nt].y : s.sum[nt].x;
      sum = faded(sum, fade);
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        float& mid = j ? s.mid[nt][g].y : s.mid[nt][g].x;
        mid = faded(mid, fade);
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        s.out[nt][h][j] = faded(s.out[nt][h][j], fade);
        s.out[nt][h][2 + j] = faded(s.out[nt][h][2 + j], fade);
      }
      if (!rises) {
        e[nt][j] = faded(e[nt][j], fade);
        e[nt][2 + j] = faded(e[nt][2 + j], fade);
      }
    }
  if (rises) weights<true, NT>(e, e, s.ref, columns, token);
  weigh<T, D, G, NT, HALVES, true>(s, e, rises, columns, slice, token, to);
  __syncthreads();
  if (rises)   // nothing asked for any more
    for (int i = lane; i < 8 * NT; i += 32) rise[warp % kWarps * S::kRows + i] = -INFINITY;
}

// Outputs of the warp's 32 channels and rows from its slices of a tile: tokens c + 4 i, i = 0..3, in pairs (c, c + 4) and (c + 8, c + 12).
// weights: the first matrix of the warp's rows.
template <typename T, int D, int G, int NT, int HALVES>
__device__ __forceinline__ void collect(Rows<T, D, G, NT>& s, const uint8_t* tile, uint32_t weights) {
  using L = Kv4<D, G>;
  using S = Shape<T, D, G, NT, HALVES>;
  constexpr int NG = L::kGroups, NB = L::kBlocks, kTerms = S::kTerms, kSlices = kWarps / S::kParts;
  const int lane = threadIdx.x & 31, warp = threadIdx.x / 32 % kWarps, r = lane >> 2, c = lane & 3, b = warp % NB, first = warp / NB * kSlices;
  const uint8_t* v = tile + first * L::kSlice + L::kHalf + (((D == 128 ? r ^ ((c >> 1) << 2) : r) * NB + b) * 2) + c * L::kRow;
  weights += (b / (G / 32) * kWarps + first) * (S::kTiles * 256) + lane * 16;
#pragma unroll
  for (int i = 0; i < kSlices; ++i) {
    uint32_t w[kTerms][NT][2], u[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) u[j] = *reinterpret_cast<const uint16_t*>(v + i * L::kSlice + 4 * j * L::kRow);
#pragma unroll
    for (int k = 0; k < kTerms; ++k) {
      const uint32_t at = weights + (k * NG * kWarps + i) * (S::kTiles * 256);
#pragma unroll
      for (int nt = 0; nt + 1 < NT; nt += 2) get4(at + nt * 256, w[k][nt][0], w[k][nt][1], w[k][nt + 1][0], w[k][nt + 1][1]);
      if constexpr (NT % 2) get2(at + (NT - 1) * 256 - (lane & 16) * 16, w[k][NT - 1][0], w[k][NT - 1][1]);
    }
    const uint32_t v0 = __byte_perm(u[0], u[1], 0x5410), v1 = __byte_perm(u[2], u[3], 0x5410);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint32_t a[4] = {codes(v0, 2 * h), codes(v0, 2 * h + 1), rest(v1, 2 * h), rest(v1, 2 * h + 1)};
#pragma unroll
      for (int k = 0; k < kTerms; ++k)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) MmaOp<__half>::run(s.out[nt][h], a, w[k][nt]);
    }
  }
}

// Tiles copied ahead of the ones that are worked on, over the ends of pieces: the first warp's.
struct Ahead {
  Walk walk;
  Piece piece;
  int next, last_slice;
  int before;   // tiles copied of the pieces before this one
};

template <typename T, int D, int G, int NT, int HALVES>
__global__ void __launch_bounds__(32 * kWarps * HALVES, blocks_of(8 * NT * HALVES)) kv4_attn_rows_kernel(const __grid_constant__ AttnArgs a) {
  using L = Kv4<D, G>;
  using S = Shape<T, D, G, NT, HALVES>;
  constexpr int NG = L::kGroups, NB = L::kBlocks, kRows = S::kRows, kStages = S::kStages, kHalves = HALVES, kThreads = S::kThreads;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ Ahead ahead;
  __shared__ Piece piece;
  uint8_t* area = smem + kStages * S::kTileBytes;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + S::kBars);
  int* scan = reinterpret_cast<int*>(smem + S::kMore);
  volatile int* abort_flag = scan + 10;
  volatile uint32_t* valid = reinterpret_cast<volatile uint32_t*>(scan + 11);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) tc::mbar_init(full + i, 1);
    tc::fence_mbar_init();
    *abort_flag = 0;
  }
  for (int i = threadIdx.x; i < kWarps * kRows; i += kThreads) reinterpret_cast<float*>(smem + S::kRise)[i] = -INFINITY;
  asm volatile("griddepcontrol.launch_dependents;");
  int request, base;
  Shares shares(0, 0, 1);
  line_of<kThreads>(a, kRows, scan, request, base, shares);
  __syncthreads();
  if ((int)blockIdx.x >= shares.blocks) return;
  const int group = a.group;
  const bool whole_tiles = a.page % kTile == 0;
  Walk walk = {request, base, shares.first(blockIdx.x), shares.first(blockIdx.x + 1)};
  Lookup found;
  auto copy_next = [&](int stage) {   // the next tile that has not been copied, if there is one
    if (ahead.next == ahead.piece.tiles) {
      __syncwarp();
      Walk w = ahead.walk;
      Piece p = {};
      const bool more = w.next(a, kRows, p);
      __syncwarp();
      if (lane == 0) {
        ahead.walk = w;
        ahead.before += ahead.next;
        ahead.piece = p;
        ahead.next = 0;
        ahead.last_slice = min((p.length + 15) / 16, (p.tile0 + p.tiles) * kWarps);
      }
      __syncwarp();
      if (!more) return;
    }
    const int i = ahead.next;
    if ((i & (whole_tiles ? 31 : 7)) == 0) found.look(a, ahead.piece, i, whole_tiles, ahead.last_slice);
    found.copy<L::kSlice>(a, i, whole_tiles, ahead.last_slice - (ahead.piece.tile0 + i) * kWarps, smem + stage * S::kTileBytes, full + stage, valid + stage);
    __syncwarp();
    if (lane == 0) ahead.next = i + 1;
    __syncwarp();
  };
  if (warp == 0) {
    if (lane == 0) {
      ahead.walk = walk;
      ahead.piece.tiles = ahead.next = ahead.before = 0;
    }
    __syncwarp();
    for (int i = 0; i < kStages; ++i) copy_next(i);
  }
  int stage = 0;
  uint32_t phase = 0;
  bool dead = false, behind = false;   // a wait ran out: nothing is waited for or copied any more, and what is computed does not count; a tile is done with
  const int r = lane >> 2, c = lane & 3, tile0 = warp / kWarps * NT, own = warp % kWarps;
  while (true) {
    if (warp == 0) {
      Piece next;
      if (!walk.next(a, kRows, next)) next.tiles = 0;
      if (lane == 0) piece = next;
    }
    __syncthreads();
    const Piece& p = piece;   // read where it is needed: registers are what is short
    if (p.tiles == 0) break;
    const T* q = static_cast<const T*>(a.q) + p.b * a.q_stride[0] + 8 * c;
    for (int nt = warp; nt < S::kTiles; nt += kWarps * kHalves) {
      const int row = p.row0 + 8 * nt + r;
      const bool in = row < p.rows;
      uint32_t w[NB][2][2], sum[2];
      const float grow = row_operands<T, D, G>(q + (int64_t)(p.head * group + row % group) * a.q_stride[1] + (int64_t)(row / group) * a.q_stride[2], in, w, sum);
#pragma unroll
      for (int i = 0; i < NB; ++i)
        *reinterpret_cast<uint4*>(smem + S::kQ + ((nt * NB + i) * 32 + lane) * 16) = make_uint4(w[i][0][0], w[i][0][1], w[i][1][0], w[i][1][1]);
      *reinterpret_cast<uint2*>(smem + S::kQSum + (nt * 32 + lane) * 8) = make_uint2(sum[0], sum[1]);
      if (c == 0) {
        float* column = reinterpret_cast<float*>(smem + S::kColumns) + (8 * nt + (r & ~1)) * 2 + (r & 1);
        column[0] = a.scale * 1.4426950408889634f * 16777216.f / grow;
        column[2] = __int_as_float(in ? max(p.length - p.count + row / group + 1, 0) : 0);
      }
    }
    Rows<T, D, G, NT> s;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      s.ref[nt] = both(-kLowest);
      s.sum[nt] = both(0.f);
#pragma unroll
      for (int g = 0; g < NG; ++g) s.mid[nt][g] = both(0.f);
#pragma unroll
      for (int j = 0; j < 8; ++j) s.out[nt][j / 4][j % 4] = 0.f;
    }
    __syncthreads();
    const int all_see = p.length - p.count + p.row0 / group + 1;   // keys that every row of the unit sees
    const uint32_t area_at = tc::smem_u32(area);
    int t0 = p.tile0 * kTile + 16 * own;
    for (int i = 0; i < p.tiles; ++i, t0 = (int)((uint32_t)t0 + kTile)) {
      if (!dead && !__all_sync(~0u, tc::mbar_try_wait(full + stage, phase))) dead = !__all_sync(~0u, tc::mbar_wait(full + stage, phase, abort_flag));
      const uint8_t* tile = smem + stage * S::kTileBytes;
      const uint8_t* slice = tile + own * L::kSlice;
      const bool there = valid[stage] >> own & 1;
      const int token = (there ? t0 : 0x7ffffff0) + (r >> 1) + 4 * (r & 1);   // a slice that is not there lies behind every key
      const uint32_t weights = area_at + (S::kBuffers == 2 && (i & 1) ? S::kWeights : 0) + tile0 * 256, to = weights + own * (S::kTiles * 256);
      float e[NT][4];
      if (S::kBuffers == 1 && i) __syncthreads();                          // the weights before have been used
      const bool rises = there && t0 + 16 <= all_see ? first_try<T, D, G, NT, HALVES, false>(s, e, tile0, smem, slice, token, to)
                                                     : first_try<T, D, G, NT, HALVES, true>(s, e, tile0, smem, slice, token, to);
      const bool move = __syncthreads_or(rises);
      if (warp == 0 && behind && !dead) copy_next(stage ? stage - 1 : kStages - 1);
      behind = true;
      if (__builtin_expect(move, 0)) raise<T, D, G, NT, HALVES>(s, e, rises, tile0, smem, slice, token, to);
      collect<T, D, G, NT, HALVES>(s, tile, weights);
      if (++stage == kStages) stage = 0, phase ^= 1;
    }
    // ------------------------------------------------------------ the warps' shares of the rows
    __syncthreads();
    float* outs = reinterpret_cast<float*>(area);
    float* totals = reinterpret_cast<float*>(area + S::kOuts);
    float* refs = reinterpret_cast<float*>(smem + S::kQSum);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int row = 8 * (tile0 + nt) + 2 * c + j;
#pragma unroll
        for (int g = 0; g <= NG; ++g) {
          const float2 pair = g < NG ? s.mid[nt][g < NG ? g : 0] : s.sum[nt];
          float x = j ? pair.y : pair.x;
#pragma unroll
          for (int d = 4; d < 32; d *= 2) x += __shfl_xor_sync(~0u, x, d);
          if (r == 0) totals[(own * (NG + 1) + g) * kRows + row] = x;
        }
        if (r == 0 && own == 0) refs[row] = j ? -s.ref[nt].y : -s.ref[nt].x;
        *reinterpret_cast<float4*>(outs + (own / NB * kRows + row) * S::kOutRow + 32 * (own % NB) + 4 * r) =
            make_float4(s.out[nt][0][j] * 16777216.f, s.out[nt][0][2 + j] * 1048576.f, s.out[nt][1][j] * 16777216.f, s.out[nt][1][2 + j] * 1048576.f);
      }
    __syncthreads();
    const bool starts = p.tile0 == 0, whole = starts && p.tiles == p.all_tiles;
    float* part = a.parts + ((int64_t)blockIdx.x * 2 + starts) * S::kPart;
    for (int i = threadIdx.x; i < kRows * D / 4; i += kThreads) {
      const int row = i / (D / 4), d = i % (D / 4) * 4;
      if (p.row0 + row >= p.rows) break;
      float sum = 0.f, mid = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        sum += totals[(w * (NG + 1) + NG) * kRows + row];
        mid += totals[(w * (NG + 1) + d / G) * kRows + row];
      }
      float4 o = make_float4(mid, mid, mid, mid);
#pragma unroll
      for (int k = 0; k < S::kParts; ++k) {
        const float4 y = *reinterpret_cast<const float4*>(outs + (k * kRows + row) * S::kOutRow + d);
        o = make_float4(o.x + y.x, o.y + y.y, o.z + y.z, o.w + y.w);
      }
      if (whole) {
        write_row<T>(a, p.b, p.head * group + (p.row0 + row) % group, (p.row0 + row) / group, d, o, refs[row], sum);
      } else {
        const float size = size_of(sum), shrink = ex2(-size);
        *reinterpret_cast<float4*>(part + row * D + d) = make_float4(o.x * shrink, o.y * shrink, o.z * shrink, o.w * shrink);
        if (d == 0) *reinterpret_cast<float2*>(part + kRows * D + 2 * row) = make_float2(refs[row] + size, sum * shrink);
      }
    }
    if (starts && threadIdx.x == 0)   // whose parts the unit is made of: from this block to the one that holds its last tile
      a.owners[((int64_t)p.b * a.kv_heads + p.head) * a.row_tiles + p.row0 / kRows] = make_int2((int)blockIdx.x, shares.owner(p.end - 1));
    __syncthreads();
  }
  if (__syncthreads_or(dead) && threadIdx.x == 0) report(a.status, PSA_ERR_TIMEOUT);
  if (threadIdx.x == 0) {   // what was copied must have landed before the block's memory is another's
    const auto ring = Ring<kStages>::after(ahead.before + ahead.next);
    int unused = 0;
    for (int i = 0; i < kStages; ++i) tc::mbar_wait(full + i, ring.last(i), &unused);
  }
}

template <typename T, int D, int G, int NT, int HALVES>
int launch_tiles(const AttnArgs& a, cudaStream_t st) {
  using S = Shape<T, D, G, NT, HALVES>;
  auto kernel = kv4_attn_rows_kernel<T, D, G, NT, HALVES>;
  static thread_local uint64_t ready = 0;   // devices that know the kernel's shared memory, per thread
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 64 || !(ready >> dev & 1)) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kBytes) != cudaSuccess) {
      set_error("psa_kv4_attention: %d bytes of shared memory: %s", S::kBytes, cudaGetErrorString(cudaGetLastError()));
      return PSA_ERR_CUDA;
    }
    if (dev < 64) ready |= (uint64_t)1 << dev;
  }
  kernel<<<a.blocks, S::kThreads, S::kBytes, st>>>(a);
  PSA_CHECK_LAUNCH("psa_kv4_attention");
  return PSA_OK;
}

}  // namespace

template <typename T, int D, int G>
int launch_rows(const AttnArgs& a, int rows_per_tile, cudaStream_t st) {
  return rows_per_tile == 24 ? launch_tiles<T, D, G, 3, 1>(a, st) : rows_per_tile == 32 ? launch_tiles<T, D, G, 4, 1>(a, st) : launch_tiles<T, D, G, 3, 2>(a, st);
}
#define PSA_ROWS(T, D, G) template int launch_rows<T, D, G>(const AttnArgs&, int, cudaStream_t)
#define PSA_ROWS_OF(T) PSA_ROWS(T, 64, 32); PSA_ROWS(T, 64, 64); PSA_ROWS(T, 128, 32); PSA_ROWS(T, 128, 64); PSA_ROWS(T, 128, 128)
PSA_ROWS_OF(__half);
PSA_ROWS_OF(__nv_bfloat16);

}  // namespace psa
