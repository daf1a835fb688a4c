// Attention of the newest tokens of every request over the cache held in 4 bits (kv4.cuh).
//
// Scores and outputs without a decoded copy of the cache.  With s, lo the step and lowest value of group g and n the codes,
//
//   q . k  = sum_g  s (sum_d q_d n_d) + lo sum_d q_d                      sum over d in g: one product of q with the codes, on
//                                                                         the tensor cores, scaled in 32 bits
//   o_d    = sum_t (p_t s_t) n_td + sum_t p_t lo_t                        the first sum is a product of codes with the weights
//                                                                         times the step, the second a number per row and group
//
// Codes are exact in f16, and so is q times a power of two per row.  The weights times the step are rounded to f16 (11 bits; for f16 tensors
// in two terms); the references of the rows keep them in its range.  Half of a slice's tokens enter as hi - s (15 - n): that keeps the
// accumulators near zero.  Sums of codes alone would grow with the context, the tensor cores cut their sums off, and what is cut off
// adds up (0.1 % of an output of 131072 evenly weighted keys).
//
// Work: one tile is 64 tokens of one key head, for up to R query rows (new tokens x query heads of that key head; 8 or 16 here, 24, 32 or 48 in
// kv4_attn_rows.cu).  All tiles of all requests stand in one line, and every block takes an equal stretch of it, computed from the lengths
// on the device: requests of any mix of lengths load the GPU evenly.  A row's tiles may lie in several blocks; their parts (running
// maximum, sum, output) are joined in order by a second kernel.  A block: one warp copies tiles into a ring (one copy where pages hold
// whole tiles, else one a slice), four warps take a slice of each (16 tokens, contiguous).  A slice's bytes go from shared memory to
// matrix operands with masks and shifts: tokens are the 16 rows of m16n8k16, query rows its 8 columns, and the channel order within a
// product is whatever the stored words give, the same for q.
//
// The floor is the cache's bytes (160 a token and key head at head_dim 128, groups of 32).  mma.sync and not tcgen05: 8 query rows
// against 128 rows of a tcgen05 tile, and operands that are made in registers; the products take a fifth of a warp's issue slots.  8 requests
// of 131071 tokens, 28 heads on 4, bf16: 133-140 us (4.8-5.0 TB/s; 103 us at copy speed).  The copies alone take 104: what bounds it is issue
// slots, 335 instructions a slice - 88 take the codes apart, 17 are products - at two thirds of a slot a cycle.  Waiting for tiles one by
// one cost 30 instructions more (149 us), a ring of its own for every warp 170 us, outputs split by channels as in kv4_attn_rows.cu 164.
#include "kv4_attn.cuh"

namespace psa {
namespace {

constexpr int kThreads = 32 * (kWarps + 1);

template <int D, int G, int NT>
struct Shape {
  static constexpr int kRows = 8 * NT;
  static constexpr int kSlice = Kv4<D, G>::kSlice;
  static constexpr int kStages = D == 128 ? 4 : 6, kPairs = kStages / 2;           // tiles of the ring; they are waited for in pairs
  static constexpr int kOutRow = D + 4;                                            // floats; 4 more spread the banks
  static constexpr int kOut = kStages * kWarps * kSlice;                           // [warps][rows][kOutRow]
  static constexpr int kStats = kOut + kWarps * kRows * kOutRow * 4;               // [warps][rows][2]
  static constexpr int kBars = kStats + kWarps * kRows * 2 * 4;                    // full, empty
  static constexpr int kMore = kBars + 2 * kStages * 8;                            // scan[8], abort, valid[stages]
  static constexpr int kBytes = kMore + (kStages + 16) * 8;
  // scratch: [ctas][2 parts] of output rows and {maximum, sum}
  static constexpr int64_t kPart = (int64_t)kRows * (D + 2);
};

__device__ __forceinline__ uint32_t movmatrix(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
// What a warp carries of a unit's rows: operands of q, and per row its reference (log2), sum, output and the share of the output
// that the groups' middle values give.  Lane 4 r + c: rows of q 8 nt + r as operands, 8 nt + 2 c + {0, 1} as columns.
template <typename T, int D, int G, int NT>
struct Rows {
  static constexpr int NG = D / G, NB = D / 32;
  uint32_t q[NT][NB][2][2];
  uint32_t q_sum[NT][2];    // sum of q over group c in two terms
  float factor[NT][2];      // of a column's scores, to log2
  float ref[NT][2], sum[NT][2];
  float out[NT][2 * NB][4]; // of channels 4 i, 4 i + 2: times 2^-24, of the others: times 2^-20
  float mid[NT][NG][2];
  float cap, limit;         // groups of 32: the largest need so far (a power of two), and the exponent from which a weight times it is too large
  int seen[NT][2];          // keys that a column's row sees
  int last;                 // keys of the request
};

// A slice's scores: rows are the tokens r/2 + 4 (r % 2) and that + 8, which lie in rows r and r + 8 of the keys.
template <typename T, int D, int G, int NT>
__device__ __forceinline__ void score(float (&x)[NT][4], const Rows<T, D, G, NT>& s, const uint8_t* slice) {
  using L = Kv4<D, G>;
  constexpr int NG = L::kGroups, NB = L::kBlocks, BG = G / 32;   // 32-channel blocks of a group
  const int lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;
  {
    const uint8_t* p = slice + L::kParams + (c < NG ? c : 0) * 4;
    const uint32_t w0 = lds<1>(p + r * NG * 4).w[0], w1 = lds<1>(p + (r + 8) * NG * 4).w[0];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) lowest_part<T>(x[nt], w0, w1, s.q_sum[nt]);
  }
  const Words<NB> k0 = lds<NB>(slice + r * L::kRow + c * NB * 4), k1 = lds<NB>(slice + (r + 8) * L::kRow + c * NB * 4);
  const Words<NG> p0 = lds<NG>(slice + L::kParams + r * NG * 4), p1 = lds<NG>(slice + L::kParams + (r + 8) * NG * 4);
#pragma unroll
  for (int g = 0; g < NG; ++g) {
    float acc[NT][4];
#pragma unroll
    for (int i = 0; i < BG; ++i)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const uint32_t w0 = k0.w[g * BG + i], w1 = k1.w[g * BG + i];
        const uint32_t a[4] = {codes(w0, 2 * k), codes(w1, 2 * k), codes(w0, 2 * k + 1), codes(w1, 2 * k + 1)};
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          if (i == 0 && k == 0) mma_new(acc[nt], a, s.q[nt][g * BG][0]);
          else MmaOp<__half>::run(acc[nt], a, s.q[nt][g * BG + i][k]);
        }
      }
    const float s0 = param<T>(p0.w[g]).x, s1 = param<T>(p1.w[g]).x;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int j = 0; j < 4; ++j) x[nt][j] = fmaf(j < 2 ? s0 : s1, acc[nt][j], x[nt][j]);
  }
}

// N slices at once (two hide each other's latencies), the n-th from token t0[n] on.
template <typename T, int D, int G, int NT, int N, bool MASKED>
__device__ __forceinline__ void take(Rows<T, D, G, NT>& s, const uint8_t* const (&slice)[N], const int (&t0)[N]) {
  using L = Kv4<D, G>;
  constexpr int NG = L::kGroups, NB = L::kBlocks, BG = G / 32;
  constexpr int kTerms = kWeightTerms<T>;
  const int lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;
  float x[N][NT][4], e[N][NT][4];
#pragma unroll
  for (int n = 0; n < N; ++n) score<T, D, G, NT>(x[n], s, slice[n]);
  // ---- weights, and whether one times its token's need is too large.  To look token by token takes few instructions where a token has few
  // groups.  With groups of 32 a warp keeps the largest need that it has met and looks only where a weight times that is too large: 8 x 131071
  // tokens of 128 channels 134.5 us instead of 140-142, 16 x 65536 of 64 channels 44.5 instead of 45.9; groups of 64 the other way round: 33
  // ragged requests of 64 channels 34.9 and 33.8, 2 new tokens of 5 x 20000 31.8 and 29.8.
  constexpr bool kKept = G == 32;
  int token[N];
  float need[N][2], widest = 0.f, most = kKept ? -INFINITY : 0.f;
  auto look_up = [&](int n) {
    const uint8_t* p = slice[n] + L::kHalf + L::kParams + r * NG * 4;
    need[n][0] = need_of<T, NG>(lds<NG>(p));
    need[n][1] = need_of<T, NG>(lds<NG>(p + 8 * NG * 4));
  };
  auto distance = [&](int n, int nt, int j) {   // to the reference; then, or at once, weights
    const float t = fmaf(x[n][nt][j], s.factor[nt][j & 1], -s.ref[nt][j & 1]);
    const float u = MASKED && token[n] + 8 * (j >> 1) >= s.seen[nt][j & 1] ? -INFINITY : t;
    return kKept ? u : ex2(u);
  };
#pragma unroll
  for (int n = 0; n < N; ++n) {
    token[n] = t0[n] + (r >> 1) + 4 * (r & 1);
    if constexpr (kKept) {
      const uint8_t* p = slice[n] + L::kHalf + L::kParams + (c < NG ? c : 0) * 4;   // a lane looks at one group of its two rows
      Words<2> w = {lds<1>(p + r * NG * 4).w[0], lds<1>(p + (r + 8) * NG * 4).w[0]};
      if (MASKED) {   // what lies behind the last key may be anything
        w.w[0] = token[n] < s.last ? w.w[0] : 0u;
        w.w[1] = token[n] + 8 < s.last ? w.w[1] : 0u;
      }
      widest = fmaxf(widest, need_of<T, 2>(w));
    } else {
      look_up(n);
    }
    float top[2] = {most, most};
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        e[n][nt][j] = distance(n, nt, j);
        top[j >> 1] = fmaxf(top[j >> 1], e[n][nt][j]);
      }
    most = kKept ? fmaxf(top[0], top[1]) : 0.f;
    if constexpr (!kKept) widest = fmaxf(widest, fmaxf(top[0] * need[n][0], top[1] * need[n][1]));
  }
  // ---- the references move seldom
  if (__any_sync(~0u, kKept ? widest > s.cap || most > s.limit : widest > kMost)) {
    if constexpr (kKept) {
#pragma unroll
      for (int d = 1; d < 32; d *= 2) widest = fmaxf(widest, __shfl_xor_sync(~0u, widest, d));
      s.cap = power_above(s.cap, widest);
      s.limit = kMostLog2 - log2_above(s.cap);
#pragma unroll
      for (int n = 0; n < N; ++n) look_up(n);
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float m = -INFINITY, over = 0.f;
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const float w = e[n][nt][2 * i + j];
            over = fmaxf(over, (kKept ? ex2(w) : w) * need[n][i]);
            if (!MASKED || token[n] + 8 * i < s.seen[nt][j]) m = fmaxf(m, x[n][nt][2 * i + j] * s.factor[nt][j] + log2_above(need[n][i]));
          }
#pragma unroll
        for (int d = 4; d < 32; d *= 2) {
          m = fmaxf(m, __shfl_xor_sync(~0u, m, d));
          over = fmaxf(over, __shfl_xor_sync(~0u, over, d));
        }
        const float ref = over > kMost ? fmaxf(m - kHead, s.ref[nt][j]) : s.ref[nt][j], fade = half_of(s.ref[nt][j] - ref);
        s.ref[nt][j] = ref;
        s.sum[nt][j] = faded(s.sum[nt][j], fade);
#pragma unroll
        for (int g = 0; g < NG; ++g) s.mid[nt][g][j] = faded(s.mid[nt][g][j], fade);
#pragma unroll
        for (int i = 0; i < 2 * NB; ++i) {
          s.out[nt][i][j] = faded(s.out[nt][i][j], fade);
          s.out[nt][i][2 + j] = faded(s.out[nt][i][2 + j], fade);
        }
#pragma unroll
        for (int n = 0; n < N; ++n) {
          e[n][nt][j] = distance(n, nt, j);
          e[n][nt][2 + j] = distance(n, nt, 2 + j);
        }
      }
  }
#pragma unroll
  for (int n = 0; n < N; ++n)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if constexpr (kKept) e[n][nt][j] = ex2(e[n][nt][j]);
        s.sum[nt][j & 1] += e[n][nt][j];
      }
  // ---- outputs: tokens c + 4 i, i = 0..3, in pairs (c, c + 4) and (c + 8, c + 12); channels 32 b + 4 r + 0..3
  constexpr int kV = NB / 2;
#pragma unroll
  for (int n = 0; n < N; ++n) {
    Words<kV> v[4];
    {
      const int u = D == 128 ? r ^ ((c >> 1) << 2) : r;
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = lds<kV>(slice[n] + L::kHalf + (c + 4 * i) * L::kRow + u * NB * 2);
    }
    const Words<NG> p0 = lds<NG>(slice[n] + L::kHalf + L::kParams + r * NG * 4), p1 = lds<NG>(slice[n] + L::kHalf + L::kParams + (r + 8) * NG * 4);
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      const float2 u0 = param<T>(p0.w[g]), u1 = param<T>(p1.w[g]);
      // a slice's first eight tokens: lo + s n; the others: hi - s (15 - n)
      const float ends[2] = {u0.y, fmaf(15.f, u1.x, u1.y)};
      uint32_t w[kTerms][NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float y[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          y[j] = e[n][nt][j] * (j < 2 ? u0.x : -u1.x);
          if (MASKED && token[n] + 8 * (j >> 1) >= s.seen[nt][j & 1]) y[j] = 0.f;   // nor does what a row does not see count, NaN or not
          else s.mid[nt][g][j & 1] = fmaf(e[n][nt][j], ends[j >> 1], s.mid[nt][g][j & 1]);
        }
#pragma unroll
        for (int k = 0; k < kTerms; ++k) {
          float first[4];   // 11 bits, cut off where another term follows
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            first[j] = k + 1 < kTerms ? __uint_as_float(__float_as_uint(y[j]) & 0xffffe000u) : y[j];
            y[j] -= first[j];
          }
          w[k][nt][0] = movmatrix(MmaOp<__half>::pack(first[0], first[1]));
          w[k][nt][1] = movmatrix(MmaOp<__half>::pack(first[2], first[3]));
        }
      }
#pragma unroll
      for (int i = 0; i < BG; ++i) {
        const int b = g * BG + i;
        const uint32_t pick = b & 1 ? 0x7632u : 0x5410u;
        const uint32_t v0 = __byte_perm(v[0].w[b >> 1], v[1].w[b >> 1], pick), v1 = __byte_perm(v[2].w[b >> 1], v[3].w[b >> 1], pick);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t a[4] = {codes(v0, 2 * h), codes(v0, 2 * h + 1), rest(v1, 2 * h), rest(v1, 2 * h + 1)};
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int k = 0; k < kTerms; ++k) MmaOp<__half>::run(s.out[nt][2 * b + h], a, w[k][nt]);
        }
      }
    }
  }
}

template <typename T, int D, int G, int NT>
__global__ void __launch_bounds__(kThreads, blocks_of(8 * NT)) kv4_attn_kernel(const __grid_constant__ AttnArgs a) {
  using L = Kv4<D, G>;
  using S = Shape<D, G, NT>;
  using R = Rows<T, D, G, NT>;
  constexpr int NG = L::kGroups, NB = L::kBlocks, kRows = S::kRows, kStages = S::kStages;
  constexpr bool kJoint = NT == 1;   // two slices' instructions mixed; with 16 rows the registers are not there for it
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ Piece piece;   // of the four warps
  float* out_s = reinterpret_cast<float*>(smem + S::kOut);
  float* stats_s = reinterpret_cast<float*>(smem + S::kStats);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + S::kBars);
  uint64_t* empty = full + S::kPairs;
  int* scan = reinterpret_cast<int*>(smem + S::kMore);
  volatile int* abort_flag = scan + 8;
  volatile uint16_t* valid = reinterpret_cast<volatile uint16_t*>(scan + 9);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < S::kPairs; ++i) {
      tc::mbar_init(full + i, 2);
      tc::mbar_init(empty + i, kWarps);
    }
    tc::fence_mbar_init();
    *abort_flag = 0;
  }
  asm volatile("griddepcontrol.launch_dependents;");
  int request, base;
  Shares shares(0, 0, 1);
  line_of<kThreads>(a, kRows, scan, request, base, shares);
  __syncthreads();
  if ((int)blockIdx.x >= shares.blocks) return;
  const int group = a.group;
  const bool whole_tiles = a.page % kTile == 0;
  Ring<S::kPairs> ring = {0, 0};   // the copying warp's barriers; a computing warp's, which it waits for
  bool dead = false;   // a wait ran out: nothing is copied or handed back any more, and what is computed does not count
  Walk walk = {request, base, shares.first(blockIdx.x), shares.first(blockIdx.x + 1)};
  while (true) {
      if (warp == kWarps) {
        Piece p;
        if (!walk.next(a, kRows, p)) break;
        // ------------------------------------------------------------ copies: one a tile where pages hold whole ones, else one a slice
        const int last_slice = min((p.length + 15) / 16, (p.tile0 + p.tiles) * kWarps);
        Lookup found;
        for (int i = 0; i < p.tiles; i += 2) {
          if (!dead && !__all_sync(~0u, tc::mbar_wait(empty + ring.at, ring.phase ^ 1, abort_flag))) dead = true;
          if (dead) break;
          for (int k = 0; k < 2; ++k) {
            const int t = i + k, at = 2 * ring.at + k;
            if (t < p.tiles && (t & (whole_tiles ? 31 : 7)) == 0) found.look(a, p, t, whole_tiles, last_slice);
            if (t < p.tiles) {
              found.copy<L::kSlice>(a, t, whole_tiles, last_slice - (p.tile0 + t) * kWarps, smem + at * kWarps * L::kSlice, full + ring.at, valid + at);
            } else if (lane == 0) {
              valid[at] = 0;
              tc::mbar_arrive(full + ring.at);
            }
          }
          ring.advance();
        }
      } else {
        // ------------------------------------------------------------ products
        if (warp == 0) {
          Piece next;
          if (!walk.next(a, kRows, next)) next.tiles = 0;
          if (lane == 0) piece = next;
        }
        asm volatile("bar.sync 1, %0;" ::"n"(32 * kWarps) : "memory");
        const Piece& p = piece;   // read where it is needed: registers are what is short
        if (p.tiles == 0) break;
        R s;
        const int r = lane >> 2, c = lane & 3, length = p.length, count = p.count, row0 = p.row0;
        const T* q = static_cast<const T*>(a.q) + p.b * a.q_stride[0] + 8 * c;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const int row = row0 + 8 * nt + r;
          const float grow = row_operands<T, D, G>(q + (int64_t)(p.head * group + row % group) * a.q_stride[1] + (int64_t)(row / group) * a.q_stride[2],
                                                   row < p.rows, s.q[nt], s.q_sum[nt]);
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const int col = row0 + 8 * nt + 2 * c + j;
            s.factor[nt][j] = a.scale * 1.4426950408889634f * 16777216.f / __shfl_sync(~0u, grow, 4 * (2 * c + j));
            s.seen[nt][j] = col < p.rows ? length - count + col / group + 1 : 0;
            s.ref[nt][j] = kLowest;
            s.sum[nt][j] = 0.f;
#pragma unroll
            for (int g = 0; g < NG; ++g) s.mid[nt][g][j] = 0.f;
          }
#pragma unroll
          for (int i = 0; i < 2 * NB; ++i) s.out[nt][i][0] = s.out[nt][i][1] = s.out[nt][i][2] = s.out[nt][i][3] = 0.f;
        }
        s.cap = kLeastNeed<T>;
        s.limit = kMostLog2 - log2_above(s.cap);
        s.last = length;
        const int all_see = length - count + row0 / group + 1;   // keys that every row of the unit sees
        // tiles whose tokens every row sees, then the others
        const int first = p.tile0 * kTile + 16 * warp, plain = all_see - 16 >= first ? min((all_see - 16 - first) / kTile + 1, p.tiles) : 0;
        auto wait = [&]() {
          if (!tc::mbar_try_wait(full + ring.at, ring.phase) && !tc::mbar_wait(full + ring.at, ring.phase, abort_flag)) dead = true;
          __syncwarp();
        };
        auto leave = [&]() {
          __syncwarp();
          if (lane == 0 && !dead) tc::mbar_arrive(empty + ring.at);
          ring.advance();
        };
        int i = 0;
        for (; i + 1 < plain; i += 2) {
          wait();
          const uint8_t* slice = smem + (2 * ring.at * kWarps + warp) * L::kSlice;
          const uint32_t there = *reinterpret_cast<volatile const uint32_t*>(valid + 2 * ring.at) & 0x10001u << warp;   // the slices, a bit each
          if (kJoint && there == 0x10001u << warp) {
            const uint8_t* const two[2] = {slice, slice + kWarps * L::kSlice};
            const int at[2] = {};
            take<T, D, G, NT, 2, false>(s, two, at);
          } else {
#pragma unroll 1
            for (int k = 0; k < 2; ++k)
              if (there >> (16 * k) & 0xffff) {
                const uint8_t* const one[1] = {slice + k * kWarps * L::kSlice};
                const int at[1] = {};
                take<T, D, G, NT, 1, false>(s, one, at);
              }
          }
          leave();
        }
        for (; i < p.tiles; i += 2) {
          wait();
#pragma unroll 1
          for (int k = 0; k < 2; ++k)
            if (valid[2 * ring.at + k] & 1u << warp) {
              const uint8_t* const one[1] = {smem + ((2 * ring.at + k) * kWarps + warp) * L::kSlice};
              const int at[1] = {first + (i + k) * kTile};
              take<T, D, G, NT, 1, true>(s, one, at);
            }
          leave();
        }
        // ------------------------------------------------------------ the four warps' rows into one
        float* mine = out_s + warp * kRows * S::kOutRow;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            float sum = s.sum[nt][j];
#pragma unroll
            for (int d = 4; d < 32; d *= 2) sum += __shfl_xor_sync(~0u, sum, d);
            const int row = 8 * nt + 2 * c + j;
            const float size = size_of(sum), shrink = ex2(-size), even = shrink * 16777216.f, odd = shrink * 1048576.f;
            if (r == 0) {
              stats_s[(warp * kRows + row) * 2] = s.ref[nt][j] + size;
              stats_s[(warp * kRows + row) * 2 + 1] = sum * shrink;
            }
#pragma unroll
            for (int g = 0; g < NG; ++g) {
              float mid = s.mid[nt][g][j];
#pragma unroll
              for (int d = 4; d < 32; d *= 2) mid += __shfl_xor_sync(~0u, mid, d);
              mid *= shrink;
#pragma unroll
              for (int i = g * (G / 32); i < (g + 1) * (G / 32); ++i)
                *reinterpret_cast<float4*>(mine + row * S::kOutRow + 32 * i + 4 * r) =
                    make_float4(fmaf(s.out[nt][2 * i][j], even, mid), fmaf(s.out[nt][2 * i][2 + j], odd, mid),
                                fmaf(s.out[nt][2 * i + 1][j], even, mid), fmaf(s.out[nt][2 * i + 1][2 + j], odd, mid));
            }
          }
        asm volatile("bar.sync 1, %0;" ::"n"(32 * kWarps) : "memory");
        const bool starts = p.tile0 == 0, whole = starts && p.tiles == p.all_tiles;
        float* part = a.parts + ((int64_t)blockIdx.x * 2 + starts) * S::kPart;
        for (int i = threadIdx.x; i < kRows * D / 4; i += 32 * kWarps) {
          const int row = i / (D / 4), d = i % (D / 4) * 4;
          if (row0 + row >= p.rows) break;
          float top = kLowest, sum = 0.f;
          float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
          for (int w = 0; w < kWarps; ++w) top = fmaxf(top, stats_s[(w * kRows + row) * 2]);
#pragma unroll
          for (int w = 0; w < kWarps; ++w) {
            const float f = exp2f(stats_s[(w * kRows + row) * 2] - top);
            const float4 y = *reinterpret_cast<const float4*>(out_s + (w * kRows + row) * S::kOutRow + d);
            sum = fmaf(f, stats_s[(w * kRows + row) * 2 + 1], sum);
            o.x = fmaf(f, y.x, o.x);
            o.y = fmaf(f, y.y, o.y);
            o.z = fmaf(f, y.z, o.z);
            o.w = fmaf(f, y.w, o.w);
          }
          if (whole) {
            write_row<T>(a, p.b, p.head * group + (row0 + row) % group, (row0 + row) / group, d, o, top, sum);
          } else {
            *reinterpret_cast<float4*>(part + row * D + d) = o;
            if (d == 0) *reinterpret_cast<float2*>(part + kRows * D + 2 * row) = make_float2(top, sum);
          }
        }
        if (starts && threadIdx.x == 0) {
          // whose parts the unit is made of: from this block to the one that holds its last tile
          a.owners[((int64_t)p.b * a.kv_heads + p.head) * a.row_tiles + row0 / kRows] = make_int2((int)blockIdx.x, shares.owner(p.end - 1));
        }
        asm volatile("bar.sync 1, %0;" ::"n"(32 * kWarps) : "memory");
      }
  }
  if (lane == 0 && *abort_flag) report(a.status, PSA_ERR_TIMEOUT);
  if (warp == kWarps && lane == 0) {   // what was copied must have landed before the block's memory is another's
    int unused = 0;
    for (int i = 0; i < S::kPairs; ++i) tc::mbar_wait(full + i, ring.last(i), &unused);
  }
}

// Rows whose tiles lay in several blocks, from their parts; rows of nothing.  A block a row: its lane groups (a group reads a part's row of
// channels) take every kGroupsOf-th part, four loads in flight each, and are joined in order.  Launched before the first kernel's
// blocks are done and held here until they are: what a launch costs is spent while they work.
constexpr int kJoinThreads = 256;
template <typename T, int D>
__global__ void __launch_bounds__(kJoinThreads) kv4_join_kernel(const __grid_constant__ AttnArgs a, int rows_per_tile) {
  constexpr int kLanes = D / 4, kGroupsOf = kJoinThreads / kLanes, kInFlight = 4;
  __shared__ float4 out_s[kGroupsOf][kLanes];
  __shared__ float2 stats_s[kGroupsOf];
  const int group = a.group, i = blockIdx.x, head = blockIdx.y, b = blockIdx.z, own = threadIdx.x / kLanes, lane = threadIdx.x % kLanes;
  int length, count;
  const Span span = span_of(a, b, rows_per_tile, length, count);
  if (span.bad && threadIdx.x == 0) report(a.status, PSA_ERR_ARG);
  const int row = i * group + head % group, r = row % rows_per_tile;
  int2 owners = make_int2(0, -1);
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (i < count && span.tiles) {
    owners = a.owners[((int64_t)b * a.kv_heads + head / group) * a.row_tiles + row / rows_per_tile];
    if (owners.x == owners.y) return;
    owners = make_int2(max(owners.x, 0), min(owners.y, a.blocks - 1));
  }
  const int64_t size = (int64_t)rows_per_tile * (D + 2);
  float top = kLowest, sum = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int k0 = owners.x + own; k0 <= owners.y; k0 += kInFlight * kGroupsOf) {
    float4 y[kInFlight];
    float2 st[kInFlight];
#pragma unroll
    for (int u = 0; u < kInFlight; ++u) {
      const int k = k0 + u * kGroupsOf;
      const float* part = a.parts + ((int64_t)min(k, owners.y) * 2 + (k == owners.x)) * size;
      st[u] = k <= owners.y ? *reinterpret_cast<const float2*>(part + rows_per_tile * D + 2 * r) : make_float2(kLowest, 0.f);
      y[u] = k <= owners.y ? *reinterpret_cast<const float4*>(part + r * D + 4 * lane) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
#pragma unroll
    for (int u = 0; u < kInFlight; ++u) {
      const float m = fmaxf(top, st[u].x), f0 = exp2f(top - m), f1 = exp2f(st[u].x - m);
      top = m;
      sum = sum * f0 + st[u].y * f1;
      o.x = o.x * f0 + y[u].x * f1;
      o.y = o.y * f0 + y[u].y * f1;
      o.z = o.z * f0 + y[u].z * f1;
      o.w = o.w * f0 + y[u].w * f1;
    }
  }
  out_s[own][lane] = o;
  if (lane == 0) stats_s[own] = make_float2(top, sum);
  __syncthreads();
  if (threadIdx.x < kLanes) {
#pragma unroll
    for (int w = 1; w < kGroupsOf; ++w) top = fmaxf(top, stats_s[w].x);
    sum = 0.f;
    o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kGroupsOf; ++w) {
      const float f = exp2f(stats_s[w].x - top);
      const float4 y = out_s[w][lane];
      sum += f * stats_s[w].y;
      o.x += f * y.x;
      o.y += f * y.y;
      o.z += f * y.z;
      o.w += f * y.w;
    }
    write_row<T>(a, b, head, i, 4 * lane, o, top, sum);
  }
}

int sm_count() {   // of the current device; asked once for each
  static int known[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0) return 148;
  if (dev < 64 && known[dev]) return known[dev];
  int n = 148;
  cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
  if (dev < 64) known[dev] = n;
  return n;
}

constexpr int kMostSms = 160;   // parts of the scratch are laid out for them
// Rows of a unit: as few units as 48 rows each make, and no more rows than they need.
int rows_per_tile(int64_t rows) {
  const int64_t most = cdiv64(rows, cdiv64(rows, 48));
  return most <= 8 ? 8 : most <= 16 ? 16 : most <= 24 ? 24 : most <= 32 ? 32 : 48;
}
// What a unit's beginning and end cost, in tiles (33 requests of 17 to 16384 tokens, 16 key heads of 64 channels: 87 us with 1, 62 with 2, 46
// with 4, 41 with 8, 45 with 12; the same requests, 4 key heads of 128 channels: 20.8 us with 4, 20.3 with 6, 20.8 with 8, 21.5 with 10, and 5
// requests of 5000: 18.3, 16.6, 16.7, 16.8; 4 key heads of 128 with 5 tokens, more than 16 rows: 74 us with 2, 64 with 3, 63 with 4).
int unit_cells(int head_dim, int rows) { return rows > 16 ? 4 : head_dim == 64 ? 8 : 6; }
// The least cells of a block: few, which leaves a small call's tiles to many blocks (500 tokens, 4 key heads: 8.2 us with 2, 11.7 with 10).
int least_cells(int rows) { return rows > 16 ? 1 : 2; }
size_t owners_bytes(int64_t batch, int kv_heads, int64_t row_tiles) { return ((size_t)batch * kv_heads * row_tiles * sizeof(int2) + 255) & ~(size_t)255; }

template <typename T, int D, int G, int NT>
int launch_few(const AttnArgs& a, cudaStream_t st) {
  using S = Shape<D, G, NT>;
  auto kernel = kv4_attn_kernel<T, D, G, NT>;
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
  kernel<<<a.blocks, kThreads, S::kBytes, st>>>(a);
  PSA_CHECK_LAUNCH("psa_kv4_attention");
  return PSA_OK;
}
template <typename T, int D, int G>
int launch(const AttnArgs& a, int rows, cudaStream_t st) {
  const int first = rows == 8 ? launch_few<T, D, G, 1>(a, st) : rows == 16 ? launch_few<T, D, G, 2>(a, st) : launch_rows<T, D, G>(a, rows, st);
  if (first != PSA_OK) return first;
  const dim3 grid((unsigned)a.tokens, (unsigned)a.heads, (unsigned)a.batch);
  cudaLaunchConfig_t how = {};
  how.gridDim = grid;
  how.blockDim = dim3(kJoinThreads);
  how.stream = st;
  cudaLaunchAttribute early;
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  how.attrs = &early;
  how.numAttrs = 1;
  const cudaError_t rc = cudaLaunchKernelEx(&how, kv4_join_kernel<T, D>, a, rows);
  PSA_REQUIRE(rc == cudaSuccess, PSA_ERR_CUDA, "psa_kv4_attention: launch failed: %s", cudaGetErrorString(rc));
  return PSA_OK;
}

}  // namespace
}  // namespace psa

extern "C" size_t psa_kv4_attention_scratch_bytes(int64_t batch, int64_t tokens, int heads, int kv_heads, int head_dim) {
  using namespace psa;
  if (batch <= 0 || batch >= 65536 || tokens <= 0 || tokens >= 65536 || heads <= 0 || kv_heads <= 0 || heads % kv_heads || head_dim <= 0) return 0;
  const int64_t rows = tokens * (heads / kv_heads), r = rows_per_tile(rows);
  return owners_bytes(batch, kv_heads, cdiv64(rows, r)) + (size_t)kMostSms * blocks_of((int)r) * 2 * r * (head_dim + 2) * sizeof(float);
}

extern "C" int psa_kv4_attention(const void* q, const int64_t* q_strides, const void* data, const int32_t* table, const int32_t* lengths,
                                 const int32_t* counts, void* out, const int64_t* out_strides, float* lse, void* scratch, size_t scratch_bytes,
                                 int64_t pages, int page_size, int64_t width, int64_t batch, int64_t tokens, int heads, int kv_heads,
                                 int head_dim, int group, float sm_scale, int dtype, int32_t* status, void* stream) {
  using namespace psa;
  PSA_REQUIRE(q && q_strides && data && table && lengths && out && out_strides && scratch && status, PSA_ERR_ARG, "psa_kv4_attention: null pointer");
  PSA_REQUIRE(dtype == PSA_F16 || dtype == PSA_BF16, PSA_ERR_UNSUPPORTED, "psa_kv4_attention: f16/bf16 only");
  PSA_REQUIRE(kv4_sizes_ok(head_dim, group), PSA_ERR_ARG, "psa_kv4_attention: head_dim=%d, group=%d (64 or 128, groups of 32, 64 or 128 within it)",
              head_dim, group);
  PSA_REQUIRE(page_size > 0 && page_size % 16 == 0 && pages > 0 && pages < ((int64_t)1 << 31) / page_size && width > 0 &&
                  width < ((int64_t)1 << 31) / page_size, PSA_ERR_ARG, "psa_kv4_attention: %lld pages of %d tokens, %lld a request", (long long)pages,
              page_size, (long long)width);
  PSA_REQUIRE(kv_heads > 0 && (double)pages * (page_size / 16) * kv_heads < 2147483648.0, PSA_ERR_ARG,
              "psa_kv4_attention: %lld pages of %d tokens, %d key heads", (long long)pages, page_size, kv_heads);
  PSA_REQUIRE(heads > 0 && heads % kv_heads == 0 && heads < 65536, PSA_ERR_ARG, "psa_kv4_attention: %d heads on %d key heads", heads,
              kv_heads);
  PSA_REQUIRE(batch > 0 && batch < 65536 && tokens > 0 && tokens < 65536, PSA_ERR_ARG, "psa_kv4_attention: %lld requests, %lld tokens",
              (long long)batch, (long long)tokens);
  PSA_REQUIRE((((uintptr_t)data | (uintptr_t)q | (uintptr_t)out) & 15) == 0, PSA_ERR_ARG, "psa_kv4_attention: operands must be 16-byte aligned");
  for (int i = 0; i < 3; ++i)
    PSA_REQUIRE(q_strides[i] % 8 == 0 && out_strides[i] % 8 == 0, PSA_ERR_ARG, "psa_kv4_attention: strides must be multiples of 8 elements");
  PSA_REQUIRE(((uintptr_t)scratch & 15) == 0 && scratch_bytes >= psa_kv4_attention_scratch_bytes(batch, tokens, heads, kv_heads, head_dim), PSA_ERR_ARG,
              "psa_kv4_attention: scratch of %zu bytes", scratch_bytes);
  AttnArgs a = {};
  a.q = q;
  a.data = static_cast<const uint8_t*>(data);
  for (int i = 0; i < 3; ++i) {
    a.q_stride[i] = q_strides[i];
    a.out_stride[i] = out_strides[i];
  }
  a.table = table;
  a.lengths = lengths;
  a.counts = counts;
  a.out = out;
  a.lse = lse;
  a.status = status;
  a.pages = pages;
  a.batch = (int)batch;
  a.tokens = (int)tokens;
  a.heads = heads;
  a.kv_heads = kv_heads;
  a.group = heads / kv_heads;
  a.width = (int)width;
  a.page = page_size;
  a.scale = sm_scale;
  const int64_t rows = tokens * (heads / kv_heads);
  a.unit_cells = unit_cells(head_dim, rows_per_tile(rows));
  a.least_cells = least_cells(rows_per_tile(rows));
  a.blocks = (sm_count() < kMostSms ? sm_count() : kMostSms) * blocks_of(rows_per_tile(rows));
  a.row_tiles = (int)cdiv64(rows, rows_per_tile(rows));
  PSA_REQUIRE(rows < ((int64_t)1 << 31), PSA_ERR_ARG, "psa_kv4_attention: %lld rows a key head", (long long)rows);
  PSA_REQUIRE((double)batch * (cdiv64(width * page_size, kTile) + a.unit_cells) * a.row_tiles * kv_heads < 2147483648.0, PSA_ERR_UNSUPPORTED,
              "psa_kv4_attention: %lld requests of up to %lld tokens: more than 2^31 tiles", (long long)batch, (long long)(width * page_size));
  a.owners = static_cast<int2*>(scratch);
  a.parts = reinterpret_cast<float*>(static_cast<char*>(scratch) + owners_bytes(batch, kv_heads, a.row_tiles));
  PSA_DISPATCH_KV4(dtype, head_dim, group, T, D, G, return (launch<T, D, G>(a, rows_per_tile(rows), (cudaStream_t)stream)));
  return PSA_OK;
}
