// Rows of keys and values into the cache held in 4 bits, and back out of it.
//
// Of a group of G channels: lowest = min x, step = (max x - min x) / 15 cut off to the tensors' type, code = (x - lowest) / step
// rounded to the nearest whole number (halfway: the even one) and at most 15.  Cutting the step off keeps lowest + 15 step at or below the
// largest value, so nothing overflows on the way back, and |x - (lowest + code * step)| <= step / 2 (at the upper end the cut step
// misses by 15 units of its last place at most, an eighth of a step in bf16).  A group that holds an infinity or a NaN, or
// whose range does not fit 32 bits, reads as NaN.
#include "kv4.cuh"

namespace psa {
namespace {

struct CacheArgs {
  uint8_t* data;
  const void* src[2];          // keys, values (append)
  void* dst[2];                // (read)
  int64_t stride[2][3];        // batch, head, token; in elements
  const int32_t* slots;        // [batch][tokens]
  int32_t* status;
  int64_t batch, tokens, slots_total;
  int heads, page;
};

// A quotient of which only the rounded value counts: the product with the inverse, corrected by its remainder (Markstein, IBM Journal of
// Research and Development 34, 1990: the quotient rounded to nearest, if the inverse is and nothing leaves the normal range).  With
// a division for each value their special function units bound the kernel.  The sum with 1.5 * 2^23 rounds to whole numbers.
constexpr float kTiny = 8.673617379884035e-19f, kRound = 12582912.f;   // 2^-60

// Largest number of the type that is not above x >= 0 (a NaN stays one).
__device__ __forceinline__ __half cut_off(float x, __half) { return __float2half_rz(x); }
__device__ __forceinline__ __nv_bfloat16 cut_off(float x, __nv_bfloat16) { return __float2bfloat16_rz(x); }

// Two numbers of the type in a word, and the number from which whole numbers up to 15 on are neighbours in it.
template <typename T> struct Pair;
template <> struct Pair<__half> {
  using type = __half2;
  static constexpr uint32_t kBase = 0x64006400u;
  static __device__ __forceinline__ __half2 make(__half a, __half b) { return __halves2half2(a, b); }
  static __device__ __forceinline__ __half2 base() { return __float2half2_rn(1024.f); }
};
template <> struct Pair<__nv_bfloat16> {
  using type = __nv_bfloat162;
  static constexpr uint32_t kBase = 0x43004300u;
  static __device__ __forceinline__ __nv_bfloat162 make(__nv_bfloat16 a, __nv_bfloat16 b) { return __halves2bfloat162(a, b); }
  static __device__ __forceinline__ __nv_bfloat162 base() { return __float2bfloat162_rn(128.f); }
};

constexpr int kHeads = 4;   // heads of a token that a thread takes, their loads in flight together

// D/8 threads hold a row, 8 neighbouring channels each, and take kHeads heads of its token; blockIdx.z: keys or values.
template <int D, int G>
struct Place {
  int u, head0, heads, slot;
  uint32_t row, b, t;
  uint8_t* slice;        // of head0; further heads lie `apart` bytes on
  int64_t apart;
  bool in, good;
  __device__ __forceinline__ Place(const CacheArgs& a) {
    const uint32_t i = blockIdx.x * blockDim.x + threadIdx.x;
    u = i % (D / 8);
    row = blockIdx.x * (256 / (D / 8)) + threadIdx.x / (D / 8);
    in = row < (uint32_t)a.batch * (uint32_t)a.tokens;
    head0 = blockIdx.y * kHeads;
    heads = min(kHeads, a.heads - head0);
    if (!in) row = 0;
    b = row / (uint32_t)a.tokens;
    t = row - b * (uint32_t)a.tokens;
    slot = a.slots[row];
    good = in && slot >= 0 && slot < a.slots_total;
    if (in && !good && slot != -1) *a.status = PSA_ERR_ARG;
    const int page = good ? slot / a.page : 0, at = good ? slot - page * a.page : 0, slices = a.page / 16;
    apart = (int64_t)slices * Kv4<D, G>::kSlice;
    slice = a.data + ((int64_t)page * a.heads + head0) * apart + at / 16 * Kv4<D, G>::kSlice;
  }
};

// Values lie in 16-bit units, and the unit that follows one in memory is of the channels 32 further on: the thread four lanes up holds
// it.  The two swap a unit each, so that both write (or read) 32 bits.  Even 32-channel blocks keep the lower unit's place.
__device__ __forceinline__ uint32_t swap_units(uint32_t codes, bool odd) {
  const uint32_t other = __shfl_xor_sync(~0u, odd ? codes & 0xffffu : codes >> 16, 4);
  return odd ? other | (codes & 0xffff0000u) : (codes & 0xffffu) | other << 16;
}

template <typename T, int D, int G>
__global__ void __launch_bounds__(256) kv4_append_kernel(const CacheArgs a) {
  using L = Kv4<D, G>;
  const int z = blockIdx.z;
  const Place<D, G> at(a);
  uint4 w[kHeads];
  const T* src = static_cast<const T*>(a.src[z]) + at.b * a.stride[z][0] + at.head0 * a.stride[z][1] + at.t * a.stride[z][2] + at.u * 8;
#pragma unroll
  for (int h = 0; h < kHeads; ++h)
    w[h] = at.good && h < at.heads ? __ldg(reinterpret_cast<const uint4*>(src + h * a.stride[z][1])) : make_uint4(0, 0, 0, 0);
  const int r = at.slot & 15, g = at.u * 8 / G;
  const bool odd = at.u >> 2 & 1;
#pragma unroll
  for (int h = 0; h < kHeads; ++h) {
    using T2 = typename Pair<T>::type;
    const T2* e = reinterpret_cast<const T2*>(&w[h]);
    // lowest and negated highest value, two numbers in a word; a NaN stays one
    T2 low = __hmin2_nan(__hmin2_nan(e[0], e[1]), __hmin2_nan(e[2], e[3])), high = __hmax2_nan(__hmax2_nan(e[0], e[1]), __hmax2_nan(e[2], e[3]));
    low = Pair<T>::make(__hmin_nan(low.x, low.y), __hneg(__hmax_nan(high.x, high.y)));
#pragma unroll
    for (int d = 1; d < G / 8; d *= 2) low = __hmin2_nan(low, __shfl_xor_sync(~0u, low, d));
    const float lo = Elem<T>::to_f(low.x), wide = (-Elem<T>::to_f(low.y) - lo) / 15.f;
    T step = cut_off(wide, T());
    T lowest = low.x;
    const float s = Elem<T>::to_f(step);
    uint32_t codes = 0;
    if (!isfinite(wide)) {   // an infinity or a NaN among them, or a range beyond 32 bits
      step = lowest = Elem<T>::from_f(__int_as_float(0x7fffffff));
    } else if (s > kTiny && s < 1.f / kTiny) {
      const float inverse = 1.f / s;
      // a rounded quotient's bits are those of 1.5 * 2^23 plus the code: their sum with weights 16^j, less what the constant makes
#pragma unroll
      for (int j = 7; j >= 0; --j) {
        const float d = Elem<T>::to_f(j & 1 ? e[j / 2].y : e[j / 2].x) - lo, q0 = d * inverse, q = fmaf(fmaf(-q0, s, d), inverse, q0);
        codes = codes * 16u + __float_as_uint(fminf(q, 15.f) + kRound);
      }
      codes -= 0x4b400000u * 0x11111111u;
    } else if (s > 0.f) {
#pragma unroll 1
      for (int j = 0; j < 8; ++j)
        codes |= (__float_as_uint(fminf((Elem<T>::to_f(reinterpret_cast<const T*>(e)[j]) - lo) / s, 15.f) + kRound) & 15u) << (4 * j);
    }
    if (z) codes = swap_units(codes, odd);
    if (!at.good || h >= at.heads) continue;
    uint8_t* slice = at.slice + h * at.apart;
    // after the swap an even block's thread has the units of channels 8 u and 8 u + 32, an odd one's those of 8 u - 28 and 8 u + 4
    const int place = z ? L::v_unit(r, odd ? at.u * 8 - 28 : at.u * 8) : L::k_word(r, at.u * 8);
    *reinterpret_cast<uint32_t*>(slice + place) = codes;
    if (at.u * 8 % G == 0) {
      T pair[2] = {step, lowest};
      *reinterpret_cast<uint32_t*>(slice + (z ? L::v_param(r, g) : L::k_param(r, g))) = *reinterpret_cast<const uint32_t*>(pair);
    }
  }
}

template <typename T, int D, int G>
__global__ void __launch_bounds__(256) kv4_read_kernel(const CacheArgs a) {
  using L = Kv4<D, G>;
  const int z = blockIdx.z;
  const Place<D, G> at(a);
  const int r = at.slot & 15, g = at.u * 8 / G;
  const bool odd = at.u >> 2 & 1;
  uint32_t codes[kHeads], pair[kHeads];
  const int place = z ? L::v_unit(r, odd ? at.u * 8 - 28 : at.u * 8) : L::k_word(r, at.u * 8), params = z ? L::v_param(r, g) : L::k_param(r, g);
#pragma unroll
  for (int h = 0; h < kHeads; ++h) {
    const bool load = at.good && h < at.heads;
    codes[h] = load ? *reinterpret_cast<const uint32_t*>(at.slice + h * at.apart + place) : 0u;
    pair[h] = load ? *reinterpret_cast<const uint32_t*>(at.slice + h * at.apart + params) : 0u;
  }
  T* dst = static_cast<T*>(a.dst[z]) + at.b * a.stride[z][0] + at.head0 * a.stride[z][1] + at.t * a.stride[z][2] + at.u * 8;
#pragma unroll
  for (int h = 0; h < kHeads; ++h) {
    const uint32_t n = z ? swap_units(codes[h], odd) : codes[h];
    using T2 = typename Pair<T>::type;
    const T2 p = *reinterpret_cast<const T2*>(&pair[h]), step = Pair<T>::make(p.x, p.x), lowest = Pair<T>::make(p.y, p.y);
    uint32_t y[4];   // channels i and i + 4: lowest + code * step, rounded once
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t c = (n >> (4 * i) & 0x000f000fu) | Pair<T>::kBase;
      const T2 v = __hfma2(__hsub2(*reinterpret_cast<const T2*>(&c), Pair<T>::base()), step, lowest);
      y[i] = *reinterpret_cast<const uint32_t*>(&v);
    }
    const uint4 w = make_uint4(__byte_perm(y[0], y[1], 0x5410), __byte_perm(y[2], y[3], 0x5410), __byte_perm(y[0], y[1], 0x7632),
                               __byte_perm(y[2], y[3], 0x7632));
    if (at.in && h < at.heads) *reinterpret_cast<uint4*>(dst + h * a.stride[z][1]) = w;
  }
}

int check(const char* what, const void* data, const void* k, const void* v, const int64_t* strides, const int32_t* slots, int64_t pages,
          int heads, int page, int64_t batch, int64_t tokens, int head_dim, int group, int dtype, int32_t* status) {
  PSA_REQUIRE(data && k && v && strides && slots && status, PSA_ERR_ARG, "%s: null pointer", what);
  PSA_REQUIRE(dtype == PSA_F16 || dtype == PSA_BF16, PSA_ERR_UNSUPPORTED, "%s: f16/bf16 only", what);
  PSA_REQUIRE(kv4_sizes_ok(head_dim, group), PSA_ERR_ARG, "%s: head_dim=%d, group=%d (64 or 128, groups of 32, 64 or 128 within it)", what, head_dim, group);
  PSA_REQUIRE(page > 0 && page % 16 == 0 && pages > 0 && pages < ((int64_t)1 << 31) / page && heads > 0 && heads < 65536, PSA_ERR_ARG,
              "%s: %lld pages of %d tokens, %d heads", what, (long long)pages, page, heads);
  PSA_REQUIRE(batch > 0 && tokens > 0 && batch < ((int64_t)1 << 31) && tokens < ((int64_t)1 << 31) && batch * tokens < ((int64_t)1 << 31), PSA_ERR_ARG,
              "%s: bad shape", what);
  PSA_REQUIRE((((uintptr_t)data | (uintptr_t)k | (uintptr_t)v) & 15) == 0, PSA_ERR_ARG, "%s: operands must be 16-byte aligned", what);
  for (int i = 0; i < 6; ++i) PSA_REQUIRE(strides[i] % 8 == 0, PSA_ERR_ARG, "%s: strides must be multiples of 8 elements", what);
  return PSA_OK;
}

CacheArgs arguments(const void* data, const int64_t* strides, const int32_t* slots, int64_t pages, int heads, int page, int64_t batch,
                    int64_t tokens, int32_t* status) {
  CacheArgs a = {};
  a.data = static_cast<uint8_t*>(const_cast<void*>(data));
  for (int i = 0; i < 6; ++i) a.stride[i / 3][i % 3] = strides[i];
  a.slots = slots;
  a.status = status;
  a.batch = batch;
  a.tokens = tokens;
  a.slots_total = pages * page;
  a.heads = heads;
  a.page = page;
  return a;
}

}  // namespace
}  // namespace psa

extern "C" size_t psa_kv4_slice_bytes(int head_dim, int group) {
  return psa::kv4_sizes_ok(head_dim, group) ? (size_t)psa::kv4_slice_bytes(head_dim, group) : 0;
}

extern "C" int psa_kv4_append(void* data, const void* k, const void* v, const int64_t* strides, const int32_t* slots, int64_t pages, int kv_heads,
                              int page_size, int64_t batch, int64_t tokens, int head_dim, int group, int dtype, int32_t* status, void* stream) {
  using namespace psa;
  if (int rc = check("psa_kv4_append", data, k, v, strides, slots, pages, kv_heads, page_size, batch, tokens, head_dim, group, dtype, status)) return rc;
  CacheArgs a = arguments(data, strides, slots, pages, kv_heads, page_size, batch, tokens, status);
  a.src[0] = k;
  a.src[1] = v;
  const dim3 grid((unsigned)cdiv64(batch * tokens, 256 / (head_dim / 8)), (unsigned)cdiv64(kv_heads, kHeads), 2);
  PSA_DISPATCH_KV4(dtype, head_dim, group, T, D, G, kv4_append_kernel<T, D, G><<<grid, 256, 0, (cudaStream_t)stream>>>(a));
  PSA_CHECK_LAUNCH("psa_kv4_append");
  return PSA_OK;
}

extern "C" int psa_kv4_read(const void* data, void* k, void* v, const int64_t* strides, const int32_t* slots, int64_t pages, int kv_heads,
                            int page_size, int64_t batch, int64_t tokens, int head_dim, int group, int dtype, int32_t* status, void* stream) {
  using namespace psa;
  if (int rc = check("psa_kv4_read", data, k, v, strides, slots, pages, kv_heads, page_size, batch, tokens, head_dim, group, dtype, status)) return rc;
  CacheArgs a = arguments(data, strides, slots, pages, kv_heads, page_size, batch, tokens, status);
  a.dst[0] = k;
  a.dst[1] = v;
  const dim3 grid((unsigned)cdiv64(batch * tokens, 256 / (head_dim / 8)), (unsigned)cdiv64(kv_heads, kHeads), 2);
  PSA_DISPATCH_KV4(dtype, head_dim, group, T, D, G, kv4_read_kernel<T, D, G><<<grid, 256, 0, (cudaStream_t)stream>>>(a));
  PSA_CHECK_LAUNCH("psa_kv4_read");
  return PSA_OK;
}
