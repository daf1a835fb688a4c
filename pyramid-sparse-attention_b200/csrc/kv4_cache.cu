// Rows of keys and values into the cache held in 4 bits, and back out of it.
//
// Of a group of G channels: lowest = min x, step = (max x - min x) / 15 cut off to the tensors' type, code = (x - lowest) / step
// rounded to the nearest whole number (halfway: the even one) and at most 15.  Cutting the step off keeps lowest + 15 step at or below the
// largest value, so nothing overflows on the way back, and |x - (lowest + code * step)| <= step / 2 (at the upper end the cut step
// misses by 15 units of its last place at most, an eighth of a step in bf16).  A group that holds an infinity or a NaN, or
// whose range does not fit 32 bits, reads as NaN.
//
// The floor is HBM, 86 MB and 13.1 us each way for 32761 tokens of 4 heads x 128.  Reading takes 15.3 us.  Appending takes 23.1 (f16 24.1), bound by
// instructions (some 590 a thread for 32 values; 74 % of the issue slots): unpacking, two sums and a product a value, the extrema.
// (Divisions by page sizes and numbers of tokens that need none cost 1.5 us each way.)
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
  int64_t head_bytes, page_bytes;   // of the cache
  int heads, page, shift;           // shift: of a page that is a power of two, or -1
};

// A quotient of which only the rounded value counts, as a product with the inverse.  The inverse is off by 2^-24 of itself at most, the
// product at a tie by less than 2^-20; the sum with 16 rounds that to steps of 2^-19, so that a tie is one again, and the sum with 1.5 * 2^23 rounds
// to whole numbers, ties to even.  With a division for each value their special function units bound the kernel: 77 us for what takes 24.
//
// What lies within 2.9 * 2^-20 of a tie (half of 2^-19, the product, the difference) and is none would count as one.  Value, lowest and tie are whole
// numbers of units in the last place of value, lowest and half a step: to be that near and not the same, the value or the lowest must be
// below kTiny steps in size - 2^8 (f16: 2^11) such units are more than it - and not zero; and if it is the value, then -lowest / step is as near to a tie
// as that.  Groups of which this holds (a thousandth of all, f16: a hundredth) look for such values and round them exactly: 32761
// tokens of 4 heads x 128: bf16 23.1 us, f16 24.1; 22.6 without, 25.1-25.9 with a remainder for every value.
constexpr float kTies = 16.f, kRound = 12582912.f;
// Steps for which that holds, and which the type cuts off by less than 1/30 of themselves: 15 is the largest code by itself.
template <typename T> constexpr float kLeastStep = 8.673617379884035e-19f;   // 2^-60
template <> constexpr float kLeastStep<__half> = 6.103515625e-05f;           // 2^-14
constexpr float kMostStep = 1.152921504606847e18f;                           // 2^60
template <typename T> constexpr float kTiny = 7.2e-4f;                       // 2.95 * 2^-12
template <> constexpr float kTiny<__half> = 5.77e-3f;                        // 2.95 * 2^-9

// The code of a value: (x - lowest) / step rounded, ties to even, in 64 bits from the sign of x - lowest - (n + 1/2) step.
__device__ __forceinline__ uint32_t exact_code(float x, float lowest, float step) {
  const double d = (double)x - lowest;
  const float n = fminf(floorf((float)d / step), 14.f);
  const double rest = fma(-(double)(n + 0.5f), (double)step, d);
  const uint32_t code = (uint32_t)n;
  return code + (rest > 0. || (rest == 0. && (code & 1)));
}

// Largest number of the type that is not above x >= 0 (a NaN stays one).
__device__ __forceinline__ __half cut_off(float x, __half) { return __float2half_rz(x); }
__device__ __forceinline__ __nv_bfloat16 cut_off(float x, __nv_bfloat16) { return __float2bfloat16_rz(x); }
// The next smaller number of a positive one.
__device__ __forceinline__ __half below(__half x) { return __ushort_as_half(__half_as_ushort(x) - 1); }
__device__ __forceinline__ __nv_bfloat16 below(__nv_bfloat16 x) { return __ushort_as_bfloat16(__bfloat16_as_ushort(x) - 1); }

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

// Whether a thread's eight channels of a row need more than the product with the inverse: a step that is none, or nearly none, or far beyond any that
// counts; a lowest value or a value near zero.
template <typename T>
__device__ __forceinline__ bool needs_more(const uint4& w, float s, float lo) {
  using T2 = typename Pair<T>::type;
  const T2* e = reinterpret_cast<const T2*>(&w);
  const T2 least = __hmin2(__hmin2(__habs2(e[0]), __habs2(e[1])), __hmin2(__habs2(e[2]), __habs2(e[3])));
  return !(s >= kLeastStep<T> && s < kMostStep) || fminf(fabsf(lo), Elem<T>::to_f(__hmin(least.x, least.y))) < s * kTiny<T>;
}
// Exact codes of a thread's eight channels of a row.
template <typename T>
__device__ __forceinline__ uint32_t exact_codes(uint4 w, float s, float lo) {
  using T2 = typename Pair<T>::type;
  uint32_t codes = 0;
  if (!(s > 0.f)) return codes;
#pragma unroll 1
  for (int i = 0; i < 4; ++i) {   // two channels a round: their registers are the kernel's
    const T2 x = *reinterpret_cast<const T2*>(&w.x);
    codes = codes >> 8 | exact_code(Elem<T>::to_f(x.x), lo, s) << 24 | exact_code(Elem<T>::to_f(x.y), lo, s) << 28;
    w = make_uint4(w.y, w.z, w.w, 0u);
  }
  return codes;
}

constexpr int kRows = 4;   // rows that a thread takes, their loads in flight together

// D/8 threads hold a row, 8 neighbouring channels each; blockIdx.z: keys or values.  A thread's rows are four heads of a token (HS 2), or,
// where there are fewer heads, both heads of two tokens (1) or the one head of four (0).
struct Slot {
  int place;         // in its slice
  int64_t slice;     // byte offset of head 0's slice
  bool in, good;
  __device__ __forceinline__ Slot(const CacheArgs& a, uint32_t row, int slice_bytes) {
    in = row < (uint32_t)a.batch * (uint32_t)a.tokens;
    const int slot = a.slots[in ? row : 0];
    good = in && slot >= 0 && slot < a.slots_total;
    if (in && !good && slot != -1) report(a.status, PSA_ERR_ARG);
    const uint32_t of = good ? (uint32_t)slot : 0u, page = a.shift >= 0 ? of >> a.shift : of / (uint32_t)a.page, at = of - page * (uint32_t)a.page;
    slice = page * a.page_bytes + (int64_t)(at / 16) * slice_bytes;   // a page may be more than 2^31 bytes
    place = (int)(at & 15);
  }
};
template <int D, int G, int HS>
struct Rows {
  static constexpr int kHeads = 1 << HS, kTokens = kRows >> HS;
  int u, head0;
  int64_t apart, stride, slice_[kTokens], at_[kTokens];
  int place_[kTokens], heads;
  bool in_[kTokens], good_[kTokens];
  __device__ __forceinline__ Rows(const CacheArgs& a) {
    const int64_t* strides = a.stride[blockIdx.z];
    u = threadIdx.x % (D / 8);
    head0 = blockIdx.y * kHeads;
    heads = a.heads - head0;
    apart = a.head_bytes;
    stride = strides[1];
    const uint32_t row = (blockIdx.x * (256 / (D / 8)) + threadIdx.x / (D / 8)) * kTokens;
    uint32_t b = a.batch == 1 ? 0u : row / (uint32_t)a.tokens, t = row - b * (uint32_t)a.tokens;
#pragma unroll
    for (int k = 0; k < kTokens; ++k) {
      const Slot s(a, row + k, Kv4<D, G>::kSlice);
      place_[k] = s.place;
      in_[k] = s.in;
      good_[k] = s.good;
      slice_[k] = s.slice + head0 * apart;
      at_[k] = b * strides[0] + t * strides[2] + head0 * stride + u * 8;
      if (++t == (uint32_t)a.tokens) t = 0, ++b;
    }
  }
  __device__ __forceinline__ bool in(int j) const { return in_[j >> HS] && j % kHeads < heads; }
  __device__ __forceinline__ bool good(int j) const { return good_[j >> HS] && j % kHeads < heads; }
  __device__ __forceinline__ int place(int j) const { return place_[j >> HS]; }
  __device__ __forceinline__ int64_t slice(int j) const { return slice_[j >> HS] + j % kHeads * apart; }
  __device__ __forceinline__ int64_t at(int j) const { return at_[j >> HS] + j % kHeads * stride; }
};

// Values lie in 16-bit units, and the unit that follows one in memory is of the channels 32 further on: the thread four lanes up holds
// it.  The two swap a unit each, so that both write (or read) 32 bits.  Even 32-channel blocks keep the lower unit's place.
__device__ __forceinline__ uint32_t swap_units(uint32_t codes, bool odd) {
  const uint32_t other = __shfl_xor_sync(~0u, odd ? codes & 0xffffu : codes >> 16, 4);
  return odd ? other | (codes & 0xffff0000u) : (codes & 0xffffu) | other << 16;
}

template <typename T, int D, int G, int HS>
__global__ void __launch_bounds__(256, 4) kv4_append_kernel(const CacheArgs a) {
  using L = Kv4<D, G>;
  using T2 = typename Pair<T>::type;
  const int z = blockIdx.z;
  const Rows<D, G, HS> to(a);
  uint4 w[kRows];
#pragma unroll
  for (int j = 0; j < kRows; ++j)
    w[j] = to.good(j) ? __ldg(reinterpret_cast<const uint4*>(static_cast<const T*>(a.src[z]) + to.at(j))) : make_uint4(0, 0, 0, 0);
  // lowest and negated highest value of a group, two numbers in a word; a NaN stays one
  uint32_t ends[kRows];
#pragma unroll
  for (int j = 0; j < kRows; ++j) {
    const T2* e = reinterpret_cast<const T2*>(&w[j]);
    T2 low = __hmin2_nan(__hmin2_nan(e[0], e[1]), __hmin2_nan(e[2], e[3])), high = __hmax2_nan(__hmax2_nan(e[0], e[1]), __hmax2_nan(e[2], e[3]));
    low = Pair<T>::make(__hmin_nan(low.x, low.y), __hneg(__hmax_nan(high.x, high.y)));
#pragma unroll
    for (int d = 1; d < G / 8; d *= 2) low = __hmin2_nan(low, __shfl_xor_sync(~0u, low, d));
    ends[j] = *reinterpret_cast<const uint32_t*>(&low);
  }
  // Every lane of a group knows them by now: of four neighbours each does one row's divisions.
  const int lane = threadIdx.x & 31, own = lane & 3;
  uint32_t pair;
  float inverse;   // 0: not for the product with it; negative: values near zero may lie near a tie
  {
    const uint32_t x = own & 2 ? (own & 1 ? ends[3] : ends[2]) : (own & 1 ? ends[1] : ends[0]);
    const bool skip = !(own & 2 ? (own & 1 ? to.good(3) : to.good(2)) : (own & 1 ? to.good(1) : to.good(0)));
    const T2 low = *reinterpret_cast<const T2*>(&x);
    T lowest = low.x;
    const float highest = -Elem<T>::to_f(low.y), wide = (highest - Elem<T>::to_f(lowest)) / 15.f;
    T step = cut_off(wide, T());
    float s = Elem<T>::to_f(step);
    // the difference, or the quotient, was rounded up to a number of the type (the sum with the larger of the two loses nothing near zero)
    if (fmaf(-15.f, s, fmaxf(highest, -Elem<T>::to_f(lowest))) < -fminf(highest, -Elem<T>::to_f(lowest))) {
      step = below(step);
      s = Elem<T>::to_f(step);
    }
    if (!isfinite(wide)) step = lowest = Elem<T>::from_f(__int_as_float(0x7fffffff));   // an infinity or a NaN among them, or a range beyond 32 bits
    inverse = skip ? 1.f : s >= kLeastStep<T> && s < kMostStep && isfinite(wide) ? __frcp_rn(s) : 0.f;
    const float at = fmaf(-Elem<T>::to_f(lowest), inverse, 0.5f), l = fabsf(Elem<T>::to_f(lowest));   // of zero, ties as whole numbers
    if (!skip && (fabsf(at - rintf(at)) < 1.02f * kTiny<T> || l < s * kTiny<T>)) inverse = -inverse;
    const T2 both = Pair<T>::make(step, lowest);
    pair = *reinterpret_cast<const uint32_t*>(&both);
  }
  uint32_t pairs[kRows], codes[kRows];
  uint32_t look = 0;   // rows with values that may need more than the product: a bit each
#pragma unroll
  for (int j = 0; j < kRows; ++j) {
    pairs[j] = __shfl_sync(~0u, pair, (lane & ~3) | j);
    const float inv = __shfl_sync(~0u, inverse, (lane & ~3) | j);
    look |= inv > 0.f ? 0u : 1u << j;
    const T2* e = reinterpret_cast<const T2*>(&w[j]);
    const float lo = Elem<T>::to_f(reinterpret_cast<const T2*>(&pairs[j])->y);
    // a rounded quotient's bits are those of 1.5 * 2^23 plus the code: their sum with weights 16^i, less what the constant makes
    codes[j] = 0u - 0x4b400000u * 0x11111111u;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float x = Elem<T>::to_f(i & 1 ? e[i / 2].y : e[i / 2].x) - lo;
      codes[j] += __float_as_uint(fmaf(x, fabsf(inv), kTies) + (kRound - kTies)) << (4 * i);
    }
  }
  if (look) {
#pragma unroll
    for (int j = 0; j < kRows; ++j) {
      if (!(look >> j & 1)) continue;
      const T2 p = *reinterpret_cast<const T2*>(&pairs[j]);
      const float step = Elem<T>::to_f(p.x), lo = Elem<T>::to_f(p.y);
      if (needs_more<T>(w[j], step, lo)) codes[j] = exact_codes<T>(w[j], step, lo);
    }
  }
  const int g = to.u * 8 / G;
  const bool odd = to.u >> 2 & 1;
#pragma unroll
  for (int j = 0; j < kRows; ++j) {
    if (z) codes[j] = swap_units(codes[j], odd);
    if (!to.good(j)) continue;
    // after the swap an even block's thread has the units of channels 8 u and 8 u + 32, an odd one's those of 8 u - 28 and 8 u + 4
    const int place = z ? L::v_unit(to.place(j), odd ? to.u * 8 - 28 : to.u * 8) : L::k_word(to.place(j), to.u * 8);
    uint8_t* slice = a.data + to.slice(j);
    *reinterpret_cast<uint32_t*>(slice + place) = codes[j];
    if (to.u * 8 % G == 0) *reinterpret_cast<uint32_t*>(slice + (z ? L::v_param(to.place(j), g) : L::k_param(to.place(j), g))) = pairs[j];
  }
}

template <typename T, int D, int G, int HS>
__global__ void __launch_bounds__(256) kv4_read_kernel(const CacheArgs a) {
  using L = Kv4<D, G>;
  const int z = blockIdx.z;
  const Rows<D, G, HS> from(a);
  const int g = from.u * 8 / G;
  const bool odd = from.u >> 2 & 1;
  uint32_t codes[kRows], pair[kRows];
#pragma unroll
  for (int j = 0; j < kRows; ++j) {
    const int r = from.place(j), place = z ? L::v_unit(r, odd ? from.u * 8 - 28 : from.u * 8) : L::k_word(r, from.u * 8);
    const uint8_t* slice = a.data + from.slice(j);
    codes[j] = from.good(j) ? *reinterpret_cast<const uint32_t*>(slice + place) : 0u;
    pair[j] = from.good(j) ? *reinterpret_cast<const uint32_t*>(slice + (z ? L::v_param(r, g) : L::k_param(r, g))) : 0u;
  }
#pragma unroll
  for (int j = 0; j < kRows; ++j) {
    const uint32_t n = z ? swap_units(codes[j], odd) : codes[j];
    using T2 = typename Pair<T>::type;
    const T2 p = *reinterpret_cast<const T2*>(&pair[j]), step = Pair<T>::make(p.x, p.x), lowest = Pair<T>::make(p.y, p.y);
    uint32_t y[4];   // channels i and i + 4: lowest + code * step, rounded once
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t c = (n >> (4 * i) & 0x000f000fu) | Pair<T>::kBase;
      const T2 v = __hfma2(__hsub2(*reinterpret_cast<const T2*>(&c), Pair<T>::base()), step, lowest);
      y[i] = *reinterpret_cast<const uint32_t*>(&v);
    }
    const uint4 w = make_uint4(__byte_perm(y[0], y[1], 0x5410), __byte_perm(y[2], y[3], 0x5410), __byte_perm(y[0], y[1], 0x7632),
                               __byte_perm(y[2], y[3], 0x7632));
    if (from.in(j)) *reinterpret_cast<uint4*>(static_cast<T*>(a.dst[z]) + from.at(j)) = w;
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

int heads_shift(int heads) { return heads >= 3 ? 2 : heads - 1; }

CacheArgs arguments(const void* data, const int64_t* strides, const int32_t* slots, int64_t pages, int heads, int page, int slice_bytes, int64_t batch,
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
  a.head_bytes = (int64_t)(page / 16) * slice_bytes;
  a.page_bytes = heads * a.head_bytes;
  a.shift = -1;
  if ((page & (page - 1)) == 0)
    for (a.shift = 0; 1 << a.shift < page;) ++a.shift;
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
  CacheArgs a = arguments(data, strides, slots, pages, kv_heads, page_size, psa::kv4_slice_bytes(head_dim, group), batch, tokens, status);
  a.src[0] = k;
  a.src[1] = v;
  const int hs = heads_shift(kv_heads);
  const dim3 grid((unsigned)cdiv64(batch * tokens, (256 / (head_dim / 8)) << (2 - hs)), (unsigned)cdiv64(kv_heads, 1 << hs), 2);
  if (hs == 2) PSA_DISPATCH_KV4(dtype, head_dim, group, T, D, G, kv4_append_kernel<T, D, G, 2><<<grid, 256, 0, (cudaStream_t)stream>>>(a));
  else if (hs == 1) PSA_DISPATCH_KV4(dtype, head_dim, group, T, D, G, kv4_append_kernel<T, D, G, 1><<<grid, 256, 0, (cudaStream_t)stream>>>(a));
  else PSA_DISPATCH_KV4(dtype, head_dim, group, T, D, G, kv4_append_kernel<T, D, G, 0><<<grid, 256, 0, (cudaStream_t)stream>>>(a));
  PSA_CHECK_LAUNCH("psa_kv4_append");
  return PSA_OK;
}

extern "C" int psa_kv4_read(const void* data, void* k, void* v, const int64_t* strides, const int32_t* slots, int64_t pages, int kv_heads,
                            int page_size, int64_t batch, int64_t tokens, int head_dim, int group, int dtype, int32_t* status, void* stream) {
  using namespace psa;
  if (int rc = check("psa_kv4_read", data, k, v, strides, slots, pages, kv_heads, page_size, batch, tokens, head_dim, group, dtype, status)) return rc;
  CacheArgs a = arguments(data, strides, slots, pages, kv_heads, page_size, psa::kv4_slice_bytes(head_dim, group), batch, tokens, status);
  a.dst[0] = k;
  a.dst[1] = v;
  const int hs = heads_shift(kv_heads);
  const dim3 grid((unsigned)cdiv64(batch * tokens, (256 / (head_dim / 8)) << (2 - hs)), (unsigned)cdiv64(kv_heads, 1 << hs), 2);
  if (hs == 2) PSA_DISPATCH_KV4(dtype, head_dim, group, T, D, G, kv4_read_kernel<T, D, G, 2><<<grid, 256, 0, (cudaStream_t)stream>>>(a));
  else if (hs == 1) PSA_DISPATCH_KV4(dtype, head_dim, group, T, D, G, kv4_read_kernel<T, D, G, 1><<<grid, 256, 0, (cudaStream_t)stream>>>(a));
  else PSA_DISPATCH_KV4(dtype, head_dim, group, T, D, G, kv4_read_kernel<T, D, G, 0><<<grid, 256, 0, (cudaStream_t)stream>>>(a));
  PSA_CHECK_LAUNCH("psa_kv4_read");
  return PSA_OK;
}
