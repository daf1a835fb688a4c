// The cache held in 4 bits: where things lie in it.
//
// data: uint8 [pages][kv heads][page_size / 16][slice].  A slice holds 16 tokens of one head, in two halves of the same form, keys
// and values: 16 rows of D/2 code bytes, then 16 rows of D/G parameter pairs (step, lowest) of the tensors' type.  Code n of group g
// stands for lowest + n * step.  A slice is one warp's work in the attention kernel and the order within it is the one its
// registers want, so that a row's bytes go from shared memory to matrix operands without a shuffle:
//
//   keys     row k_row(t) = 8 (t / 8) + 2 (t % 4) + (t / 4) % 2 (also the row of the parameters, of the values' too); in it
//            32-bit word (d % 32 / 8) * D/32 + d / 32 holds channels 8 i .. 8 i + 7, lowest nibble first
//   values   row t; in it 16-bit unit e * D/32 + d / 32 with e = d % 32 / 4 holds channels 4 i .. 4 i + 3; at D = 128
//            e is XOR-ed by 4 in rows with (t / 2) % 2, which spreads the four rows of a warp's load over all banks
#pragma once
#include "psa_common.cuh"

namespace psa {

template <int D, int G>
struct Kv4 {
  static constexpr int kGroups = D / G, kRow = D / 2, kBlocks = D / 32;
  static constexpr int kParams = 16 * kRow;                      // byte offset of a half's parameters
  static constexpr int kHalf = kParams + 16 * kGroups * 4;       // bytes of the keys' half, and of the values'
  static constexpr int kSlice = 2 * kHalf;
  static __host__ __device__ constexpr int k_row(int t) { return 8 * (t / 8) + 2 * (t % 4) + t / 4 % 2; }
  static __host__ __device__ constexpr int k_word(int t, int d) { return k_row(t) * kRow + (d % 32 / 8 * kBlocks + d / 32) * 4; }
  static __host__ __device__ constexpr int v_unit(int t, int d) {
    const int e = d % 32 / 4;
    return kHalf + t * kRow + ((D == 128 ? e ^ (t / 2 % 2 * 4) : e) * kBlocks + d / 32) * 2;
  }
  static __host__ __device__ constexpr int k_param(int t, int g) { return kParams + (k_row(t) * kGroups + g) * 4; }
  static __host__ __device__ constexpr int v_param(int t, int g) { return kHalf + k_param(t, g); }
};

static inline int kv4_slice_bytes(int head_dim, int group) { return 16 * (head_dim + 8 * (head_dim / group)); }
static inline bool kv4_sizes_ok(int head_dim, int group) {
  return (head_dim == 64 || head_dim == 128) && (group == 32 || group == 64 || group == 128) && group <= head_dim;
}

#define PSA_DISPATCH_KV4(dtype, head_dim, group, T, D, G, ...)                                                     \
  do {                                                                                                             \
    if (dtype == PSA_BF16) { using T = __nv_bfloat16; PSA_DISPATCH_KV4_DG(head_dim, group, D, G, __VA_ARGS__); }     \
    else { using T = __half; PSA_DISPATCH_KV4_DG(head_dim, group, D, G, __VA_ARGS__); }                              \
  } while (0)
#define PSA_DISPATCH_KV4_DG(head_dim, group, D, G, ...)                                                            \
  if (head_dim == 64) {                                                                                            \
    constexpr int D = 64;                                                                                          \
    if (group == 32) { constexpr int G = 32; __VA_ARGS__; } else { constexpr int G = 64; __VA_ARGS__; }             \
  } else {                                                                                                         \
    constexpr int D = 128;                                                                                         \
    if (group == 32) { constexpr int G = 32; __VA_ARGS__; }                                                         \
    else if (group == 64) { constexpr int G = 64; __VA_ARGS__; } else { constexpr int G = 128; __VA_ARGS__; }       \
  }

}  // namespace psa
