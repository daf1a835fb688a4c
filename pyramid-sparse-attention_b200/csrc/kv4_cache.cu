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

// Largest number of the type that is not above x >= 0.
__device__ __forceinline__ __half cut_off(float x, __half) { return __float2half_rz(x); }
__device__ __forceinline__ __nv_bfloat16 cut_off(float x, __nv_bfloat16) { return __float2bfloat16_rz(x); }

template <int D, int G>
__device__ __forceinline__ uint8_t* slice_of(const CacheArgs& a, int slot, int head) {
  const int page = slot / a.page, at = slot - page * a.page;
  return a.data + (((int64_t)page * a.heads + head) * (a.page / 16) + at / 16) * Kv4<D, G>::kSlice;
}

// A thread holds 8 neighbouring channels of a row of keys (z = 0) or values (z = 1), D/8 threads a row.  Rows run over tokens, then
// heads, so that a block reads and writes near places whichever way the tensors lie.
template <int D, int G>
__device__ __forceinline__ bool place(const CacheArgs& a, int& u, int& head, int64_t& b, int64_t& t, int& slot) {
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  u = (int)(i % (D / 8));
  int64_t row = i / (D / 8);
  head = (int)(row % a.heads);
  row /= a.heads;
  if (row >= a.batch * a.tokens) return false;
  b = row / a.tokens;
  t = row - b * a.tokens;
  slot = a.slots[row];
  return true;
}

template <typename T, int D, int G>
__global__ void __launch_bounds__(256) kv4_append_kernel(const CacheArgs a) {
  using L = Kv4<D, G>;
  const int z = blockIdx.y;
  int u, head, slot;
  int64_t b, t;
  const bool in = place<D, G>(a, u, head, b, t, slot);
  const bool write = in && slot >= 0 && slot < a.slots_total;
  if (in && !write && slot != -1) *a.status = PSA_ERR_ARG;
  float x[8];
  if (write) {
    const uint4 w = *reinterpret_cast<const uint4*>(static_cast<const T*>(a.src[z]) + b * a.stride[z][0] + head * a.stride[z][1] +
                                                    t * a.stride[z][2] + u * 8);
    const T* e = reinterpret_cast<const T*>(&w);
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = Elem<T>::to_f(e[j]);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = 0.f;
  }
  float lo = x[0], hi = x[0];
  bool finite = true;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    lo = fminf(lo, x[j]);
    hi = fmaxf(hi, x[j]);
    finite = finite && isfinite(x[j]);
  }
#pragma unroll
  for (int d = 1; d < G / 8; d *= 2) {
    lo = fminf(lo, __shfl_xor_sync(~0u, lo, d));
    hi = fmaxf(hi, __shfl_xor_sync(~0u, hi, d));
    finite = __shfl_xor_sync(~0u, (int)finite, d) && finite;
  }
  if (!write) return;
  const float wide = (hi - lo) / 15.f;
  T step = cut_off(wide, T());
  T lowest = Elem<T>::from_f(lo);
  const float s = Elem<T>::to_f(step);
  uint32_t codes = 0;
  if (!finite || !isfinite(wide)) {
    step = lowest = Elem<T>::from_f(__int_as_float(0x7fffffff));
  } else if (s > 0.f) {
#pragma unroll
    for (int j = 0; j < 8; ++j) codes |= (uint32_t)fminf(rintf((x[j] - lo) / s), 15.f) << (4 * j);
  }
  uint8_t* slice = slice_of<D, G>(a, slot, head);
  const int r = slot % 16, g = u * 8 / G;
  if (z == 0) {
    *reinterpret_cast<uint32_t*>(slice + L::k_word(r, u * 8)) = codes;
  } else {
    *reinterpret_cast<uint16_t*>(slice + L::v_unit(r, u * 8)) = (uint16_t)codes;
    *reinterpret_cast<uint16_t*>(slice + L::v_unit(r, u * 8 + 4)) = (uint16_t)(codes >> 16);
  }
  if (u * 8 % G == 0) {
    T* p = reinterpret_cast<T*>(slice + (z == 0 ? L::k_param(r, g) : L::v_param(r, g)));
    p[0] = step;
    p[1] = lowest;
  }
}

template <typename T, int D, int G>
__global__ void __launch_bounds__(256) kv4_read_kernel(const CacheArgs a) {
  using L = Kv4<D, G>;
  const int z = blockIdx.y;
  int u, head, slot;
  int64_t b, t;
  if (!place<D, G>(a, u, head, b, t, slot)) return;
  uint4 w = make_uint4(0, 0, 0, 0);
  if (slot >= 0 && slot < a.slots_total) {
    const uint8_t* slice = slice_of<D, G>(a, slot, head);
    const int r = slot % 16, g = u * 8 / G;
    uint32_t codes;
    if (z == 0) {
      codes = *reinterpret_cast<const uint32_t*>(slice + L::k_word(r, u * 8));
    } else {
      codes = *reinterpret_cast<const uint16_t*>(slice + L::v_unit(r, u * 8)) |
              (uint32_t)*reinterpret_cast<const uint16_t*>(slice + L::v_unit(r, u * 8 + 4)) << 16;
    }
    const T* p = reinterpret_cast<const T*>(slice + (z == 0 ? L::k_param(r, g) : L::v_param(r, g)));
    const float step = Elem<T>::to_f(p[0]), lowest = Elem<T>::to_f(p[1]);
    T* e = reinterpret_cast<T*>(&w);
#pragma unroll
    for (int j = 0; j < 8; ++j) e[j] = Elem<T>::from_f(fmaf((float)(codes >> (4 * j) & 15), step, lowest));
  } else if (slot != -1) {
    *a.status = PSA_ERR_ARG;
  }
  *reinterpret_cast<uint4*>(static_cast<T*>(a.dst[z]) + b * a.stride[z][0] + head * a.stride[z][1] + t * a.stride[z][2] + u * 8) = w;
}

int check(const char* what, const void* data, const void* k, const void* v, const int64_t* strides, const int32_t* slots, int64_t pages,
          int heads, int page, int64_t batch, int64_t tokens, int head_dim, int group, int dtype, int32_t* status) {
  PSA_REQUIRE(data && k && v && strides && slots && status, PSA_ERR_ARG, "%s: null pointer", what);
  PSA_REQUIRE(dtype == PSA_F16 || dtype == PSA_BF16, PSA_ERR_UNSUPPORTED, "%s: f16/bf16 only", what);
  PSA_REQUIRE(kv4_sizes_ok(head_dim, group), PSA_ERR_ARG, "%s: head_dim=%d, group=%d (64 or 128, groups of 32, 64 or 128 within it)", what, head_dim, group);
  PSA_REQUIRE(page > 0 && page % 16 == 0 && pages > 0 && pages < ((int64_t)1 << 31) / page && heads > 0 && heads < 65536, PSA_ERR_ARG,
              "%s: %lld pages of %d tokens, %d heads", what, (long long)pages, page, heads);
  PSA_REQUIRE(batch > 0 && tokens > 0 && batch * tokens < ((int64_t)1 << 31) && cdiv64(batch * tokens * heads * (head_dim / 8), 256) < ((int64_t)1 << 31),
              PSA_ERR_ARG, "%s: bad shape", what);
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
  const dim3 grid((unsigned)cdiv64(batch * tokens * kv_heads * (head_dim / 8), 256), 2);
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
  const dim3 grid((unsigned)cdiv64(batch * tokens * kv_heads * (head_dim / 8), 256), 2);
  PSA_DISPATCH_KV4(dtype, head_dim, group, T, D, G, kv4_read_kernel<T, D, G><<<grid, 256, 0, (cudaStream_t)stream>>>(a));
  PSA_CHECK_LAUNCH("psa_kv4_read");
  return PSA_OK;
}
