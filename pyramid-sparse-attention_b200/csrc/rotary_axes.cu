// Rotary positions with several axes (text, or time / height / width of a video's tokens), applied to queries and keys in one
// launch; the backward pass is the same kernel with the angles negated.
//
// Channel pair i of token (b, t) is turned by the angle pos[axis(i)][b][t] * freq(i).  The angle is kept in turns as a 64-bit
// fraction: turns(i) = freq(i) / 2 pi * 2^64 comes from the host, the product with the position is taken modulo 2^64 - whole turns
// drop out of an integer product by themselves - and its upper half, a signed number of 2^-32 turns, gives the nearest quarter turn
// and what is left of it, at most an eighth.  The error is |pos| * 2^-65 turns plus a few roundings of sine and cosine, at any position
// a model reaches; pos * freq in 32 bits is off by 2^-25 * pos radians (0.004 at position 131072).
#include "psa_common.cuh"

namespace psa {
namespace {

constexpr int kMaxPairs = 128, kMaxAxes = 8, kInFlight = 4;   // kInFlight: heads whose loads a thread issues at once

struct RotaryArgs {
  const void* src[2];
  void* dst[2];
  int64_t src_stride[2][3], dst_stride[2][3];   // batch, head, token; in elements
  int heads[2];
  const void* pos;
  int64_t pos_stride[3];                        // axis, batch, token; in elements
  int64_t batch, seq;
  uint64_t turns[kMaxPairs];
  uint8_t axis[kMaxPairs];
  int pos64, inverse;
};

union Word {
  uint4 u;
  float f[4];
  __half h[8];
  __nv_bfloat16 b[8];
};
template <typename T> __device__ __forceinline__ T* word_of(Word& w);
template <> __device__ __forceinline__ float* word_of<float>(Word& w) { return w.f; }
template <> __device__ __forceinline__ __half* word_of<__half>(Word& w) { return w.h; }
template <> __device__ __forceinline__ __nv_bfloat16* word_of<__nv_bfloat16>(Word& w) { return w.b; }

// Sine and cosine of turn * 2^-32 turns.  Taylor's series at |r| <= pi / 4: what follows the last terms is below r^11 / 11! (2 10^-9) and
// r^10 / 10! (2.5 10^-8, half a rounding of a cosine that is above 0.7).
__device__ __forceinline__ void sine_cosine(int32_t turn, float& sine, float& cosine) {
  const uint32_t quarter = ((uint32_t)turn + (1u << 29)) >> 30;
  const float r = (float)(int32_t)((uint32_t)turn - (quarter << 30)) * 1.4629180792671596e-09f;   // 2 pi / 2^32
  const float x = r * r;
  const float s = fmaf(r * x, fmaf(x, fmaf(x, fmaf(x, 1.f / 362880, -1.f / 5040), 1.f / 120), -1.f / 6), r);
  const float c = fmaf(x, fmaf(x, fmaf(x, fmaf(x, 1.f / 40320, -1.f / 720), 1.f / 24), -0.5f), 1.f);
  const float u = quarter & 1 ? c : s, v = quarter & 1 ? s : c;
  sine = __uint_as_float(__float_as_uint(u) ^ (quarter & 2) << 30);
  cosine = __uint_as_float(__float_as_uint(v) ^ ((quarter + 1) & 2) << 30);
}

// Bound by HBM: 28 + 4 heads of 128, 32768 tokens 88 us (6.1 TB/s, 93 % of a copy), 12 + 12 of 128, 32760 tokens f16 67 us (6.0), 48 + 48 of 64
// token-major 75 us (5.8).  Blocks that stay and take one token after another keep their pairs' turns in registers, 122 of them: 101 us
// for the first.  With few heads the sines count: 1 + 1 heads f32 21.5 us with sincospif and the turns read from the arguments, 14.4 now.
//
// A thread owns V pairs of one token, computes their sines and cosines once and walks the heads with them.  Its two 16-byte words of a
// row lie half a row apart, so that a warp's words are neighbours, whichever channels make a pair: HALF, channels (i, i + D/2), one of
// each word; otherwise neighbours (2i, 2i + 1), V/2 pairs in each.
template <typename T, bool HALF>
__global__ void __launch_bounds__(128) rotary_axes_kernel(const __grid_constant__ RotaryArgs a, int head_dim, int heads_each) {
  constexpr int V = 16 / (int)sizeof(T);
  // turns and axes to shared memory: lanes that read the kernel's arguments at different places wait for one another
  __shared__ uint64_t turns_s[kMaxPairs];
  __shared__ uint8_t axis_s[kMaxPairs];
  for (int i = threadIdx.x; i < head_dim / 2; i += blockDim.x) {
    turns_s[i] = a.turns[i];
    axis_s[i] = a.axis[i];
  }
  __syncthreads();
  const int chunks = head_dim / 2 / V, each = blockDim.x / chunks;   // tokens of a block
  const int own = threadIdx.x / chunks, chunk = threadIdx.x - own * chunks;
  const int64_t tokens = a.batch * a.seq, token = (int64_t)blockIdx.x * each + own;
  if (own >= each || token >= tokens) return;
  const int64_t b = tokens <= 0xffffffffll ? (uint32_t)token / (uint32_t)a.seq : token / a.seq, t = token - b * a.seq;
  const int64_t pos_at = b * a.pos_stride[1] + t * a.pos_stride[2];
  float cs[V], sn[V];
  int64_t p = 0;
  int axis = -1;
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const int pair = HALF ? chunk * V + j : chunk * (V / 2) + j % (V / 2) + (j < V / 2 ? 0 : head_dim / 4);
    if (axis_s[pair] != axis) {
      axis = axis_s[pair];
      const int64_t at = axis * a.pos_stride[0] + pos_at;
      p = a.pos64 ? static_cast<const int64_t*>(a.pos)[at] : static_cast<const int32_t*>(a.pos)[at];
    }
    sine_cosine((int32_t)(((uint64_t)p * turns_s[pair]) >> 32), sn[j], cs[j]);
    if (a.inverse) sn[j] = -sn[j];
  }
  const int first = chunk * V, second = first + head_dim / 2;
  const int heads = min(a.heads[0] + a.heads[1], (int)(blockIdx.y + 1) * heads_each);
  for (int h0 = blockIdx.y * heads_each; h0 < heads; h0 += kInFlight) {
    Word w0[kInFlight], w1[kInFlight];
#pragma unroll
    for (int u = 0; u < kInFlight; ++u) {
      const int h = h0 + u;
      if (h < heads) {
        const int z = h >= a.heads[0], hh = z ? h - a.heads[0] : h;
        const T* src = static_cast<const T*>(a.src[z]) + b * a.src_stride[z][0] + hh * a.src_stride[z][1] + t * a.src_stride[z][2];
        w0[u].u = __ldg(reinterpret_cast<const uint4*>(src + first));
        w1[u].u = __ldg(reinterpret_cast<const uint4*>(src + second));
      }
    }
#pragma unroll
    for (int u = 0; u < kInFlight; ++u) {
      const int h = h0 + u;
      if (h >= heads) break;
      T *e0 = word_of<T>(w0[u]), *e1 = word_of<T>(w1[u]);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        T& r0 = HALF ? e0[j] : (j < V / 2 ? e0[2 * j] : e1[2 * j - V]);
        T& r1 = HALF ? e1[j] : (j < V / 2 ? e0[2 * j + 1] : e1[2 * j + 1 - V]);
        const float x0 = Elem<T>::to_f(r0), x1 = Elem<T>::to_f(r1);
        r0 = Elem<T>::from_f(x0 * cs[j] - x1 * sn[j]);
        r1 = Elem<T>::from_f(x1 * cs[j] + x0 * sn[j]);
      }
      const int z = h >= a.heads[0], hh = z ? h - a.heads[0] : h;
      T* dst = static_cast<T*>(a.dst[z]) + b * a.dst_stride[z][0] + hh * a.dst_stride[z][1] + t * a.dst_stride[z][2];
      *reinterpret_cast<uint4*>(dst + first) = w0[u].u;
      *reinterpret_cast<uint4*>(dst + second) = w1[u].u;
    }
  }
}

template <typename T>
int launch(const RotaryArgs& a, int head_dim, int half, cudaStream_t st) {
  const int64_t blocks = cdiv64(a.batch * a.seq, 128 / (head_dim / 2 / (16 / (int)sizeof(T))));
  PSA_REQUIRE(blocks < ((int64_t)1 << 31), PSA_ERR_ARG, "psa_rotate_axes: too many tokens");
  const int heads = a.heads[0] + a.heads[1];
  // A block's heads are neighbours: in token-major tensors their rows are, too.  Few tokens: the heads are shared out over blocks, down
  // to what a thread loads at once - fewer cost more sines than they hide latency (16 heads of 2536 tokens: 5.2 us by fours, 7.2 one by
  // one) - or to one, where the GPU would be empty otherwise.
  int each = heads;
  while (each > kInFlight && blocks * cdiv64(heads, each) < 148 * 16) each = each > 2 * kInFlight ? (each + 1) / 2 : kInFlight;
  while (each > 1 && blocks * cdiv64(heads, each) < 148) each = (each + 1) / 2;
  const dim3 grid((unsigned)blocks, (unsigned)cdiv64(heads, each));
  if (half) rotary_axes_kernel<T, true><<<grid, 128, 0, st>>>(a, head_dim, each);
  else rotary_axes_kernel<T, false><<<grid, 128, 0, st>>>(a, head_dim, each);
  PSA_CHECK_LAUNCH("psa_rotate_axes");
  return PSA_OK;
}

}  // namespace
}  // namespace psa

extern "C" int psa_rotate_axes(const void* const* src, const int64_t* src_strides, void* const* dst, const int64_t* dst_strides,
                               const int32_t* heads, int n, const void* positions, int position_bits, const int64_t* position_strides,
                               const uint64_t* turns, const uint8_t* axis_of_pair, int axes, int64_t batch, int64_t seq, int head_dim,
                               int half, int inverse, int dtype, void* stream) {
  using namespace psa;
  PSA_REQUIRE(src && src_strides && dst && dst_strides && heads && positions && position_strides && turns && axis_of_pair, PSA_ERR_ARG,
              "psa_rotate_axes: null pointer");
  PSA_REQUIRE(n == 1 || n == 2, PSA_ERR_ARG, "psa_rotate_axes: 1 or 2 operands");
  PSA_REQUIRE(head_dim >= 16 && head_dim <= 2 * kMaxPairs && head_dim % 16 == 0, PSA_ERR_ARG,
              "psa_rotate_axes: head_dim=%d (a multiple of 16 up to %d)", head_dim, 2 * kMaxPairs);
  PSA_REQUIRE(axes >= 1 && axes <= kMaxAxes, PSA_ERR_ARG, "psa_rotate_axes: %d axes (1 to %d)", axes, kMaxAxes);
  PSA_REQUIRE(position_bits == 32 || position_bits == 64, PSA_ERR_ARG, "psa_rotate_axes: positions of %d bits (32 or 64)", position_bits);
  PSA_REQUIRE(batch > 0 && seq > 0 && batch < ((int64_t)1 << 31) && seq < ((int64_t)1 << 31), PSA_ERR_ARG, "psa_rotate_axes: bad shape");
  const int elem = dtype == PSA_F32 ? 4 : 2;
  RotaryArgs a = {};
  for (int i = 0; i < n; ++i) {
    PSA_REQUIRE(src[i] && dst[i] && src[i] != dst[i] && heads[i] > 0, PSA_ERR_ARG, "psa_rotate_axes: operand %d", i);
    PSA_REQUIRE((((uintptr_t)src[i] | (uintptr_t)dst[i]) & 15) == 0, PSA_ERR_ARG, "psa_rotate_axes: operand %d is not 16-byte aligned", i);
    for (int d = 0; d < 3; ++d) {
      PSA_REQUIRE(src_strides[3 * i + d] * elem % 16 == 0 && dst_strides[3 * i + d] * elem % 16 == 0, PSA_ERR_ARG,
                  "psa_rotate_axes: strides of operand %d must be multiples of 16 bytes", i);
      a.src_stride[i][d] = src_strides[3 * i + d];
      a.dst_stride[i][d] = dst_strides[3 * i + d];
    }
    a.src[i] = src[i];
    a.dst[i] = dst[i];
    a.heads[i] = heads[i];
  }
  for (int i = 0; i < head_dim / 2; ++i) {
    PSA_REQUIRE(axis_of_pair[i] < axes, PSA_ERR_ARG, "psa_rotate_axes: pair %d is of axis %d of %d", i, axis_of_pair[i], axes);
    a.turns[i] = turns[i];
    a.axis[i] = axis_of_pair[i];
  }
  a.pos = positions;
  for (int d = 0; d < 3; ++d) a.pos_stride[d] = position_strides[d];
  a.batch = batch;
  a.seq = seq;
  a.pos64 = position_bits == 64;
  a.inverse = inverse != 0;
  PSA_DISPATCH_DTYPE(dtype, T, return launch<T>(a, head_dim, half, (cudaStream_t)stream));
  return PSA_OK;
}
