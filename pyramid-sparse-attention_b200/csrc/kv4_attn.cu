// Attention of the newest tokens of every request over the cache held in 4 bits (kv4.cuh).
#include "kv4.cuh"

namespace psa {
namespace {

struct AttnArgs {
  const void* q;
  int64_t q_stride[3], out_stride[3];   // batch, head, token; in elements
  const uint8_t* data;
  const int32_t *table, *lengths, *counts;
  void* out;
  float* lse;
  int32_t* status;
  int64_t pages;
  int batch, tokens, heads, kv_heads, width, page;
  float scale;
};

// One query row a block: a thread scores one of 128 tokens, then gathers one channel over them.
template <typename T, int D, int G>
__global__ void __launch_bounds__(128) kv4_attn_rows_kernel(const AttnArgs a) {
  using L = Kv4<D, G>;
  __shared__ float q[D], p[128], red[4];
  __shared__ int64_t at[128];
  const int i = blockIdx.x, head = blockIdx.y, b = blockIdx.z, tid = threadIdx.x, group = a.heads / a.kv_heads;
  int64_t length = a.lengths[b];
  const int count = a.counts ? a.counts[b] : a.tokens;
  if (length < 0 || length > (int64_t)a.width * a.page || count < 0 || count > a.tokens) {
    if (tid == 0) *a.status = PSA_ERR_ARG;
    length = min(max(length, (int64_t)0), (int64_t)a.width * a.page);
  }
  const int64_t seen = i < count ? length - count + i + 1 : 0;
  const T* row = static_cast<const T*>(a.q) + b * a.q_stride[0] + head * a.q_stride[1] + i * a.q_stride[2];
  if (tid < D) q[tid] = Elem<T>::to_f(row[tid]);
  float m = -INFINITY, l = 0.f, acc = 0.f;
  for (int64_t t0 = 0; t0 < seen; t0 += 128) {
    __syncthreads();
    const int64_t t = t0 + tid;
    float s = -INFINITY;
    int64_t from = -1;
    if (t < seen) {
      const int page = a.table[(int64_t)b * a.width + t / a.page];
      if (page >= 0 && page < a.pages) {
        from = (((int64_t)page * a.kv_heads + head / group) * (a.page / 16) + t % a.page / 16) * L::kSlice;
        const uint8_t* slice = a.data + from;
        const int r = (int)(t % 16);
        s = 0.f;
        for (int g = 0; g < L::kGroups; ++g) {
          const T* par = reinterpret_cast<const T*>(slice + L::k_param(r, g));
          float dot = 0.f, sum = 0.f;
          for (int d = g * G; d < (g + 1) * G; d += 8) {
            const uint32_t w = *reinterpret_cast<const uint32_t*>(slice + L::k_word(r, d));
            for (int j = 0; j < 8; ++j) {
              dot += q[d + j] * (float)(w >> (4 * j) & 15);
              sum += q[d + j];
            }
          }
          s += Elem<T>::to_f(par[0]) * dot + Elem<T>::to_f(par[1]) * sum;
        }
        s *= a.scale;
      } else {
        *a.status = PSA_ERR_ARG;
      }
    }
    at[tid] = from;
    float top = s;
    for (int d = 16; d; d /= 2) top = fmaxf(top, __shfl_xor_sync(~0u, top, d));
    if (tid % 32 == 0) red[tid / 32] = top;
    __syncthreads();
    top = fmaxf(m, fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])));
    const float ref = top == -INFINITY ? 0.f : top;
    const float e = from >= 0 ? expf(s - ref) : 0.f;
    p[tid] = e;
    float sum = e;
    for (int d = 16; d; d /= 2) sum += __shfl_xor_sync(~0u, sum, d);
    __syncthreads();
    if (tid % 32 == 0) red[tid / 32] = sum;
    __syncthreads();
    const float fade = m == -INFINITY ? 0.f : expf(m - ref);
    l = l * fade + red[0] + red[1] + red[2] + red[3];
    m = top;
    if (tid < D) {
      acc *= fade;
      for (int j = 0; j < 128 && t0 + j < seen; ++j) {
        if (at[j] < 0) continue;
        const uint8_t* slice = a.data + at[j];
        const int r = (int)((t0 + j) % 16);
        const uint32_t w = *reinterpret_cast<const uint16_t*>(slice + L::v_unit(r, tid));
        const T* par = reinterpret_cast<const T*>(slice + L::v_param(r, tid / G));
        acc += p[j] * (Elem<T>::to_f(par[1]) + Elem<T>::to_f(par[0]) * (float)(w >> (tid % 4 * 4) & 15));
      }
    }
  }
  if (tid < D)
    static_cast<T*>(a.out)[b * a.out_stride[0] + head * a.out_stride[1] + i * a.out_stride[2] + tid] = Elem<T>::from_f(l == 0.f ? 0.f : acc / l);
  if (a.lse && tid == 0) a.lse[((int64_t)b * a.heads + head) * a.tokens + i] = l == 0.f ? -INFINITY : m + logf(l);
}

}  // namespace
}  // namespace psa

extern "C" size_t psa_kv4_attention_scratch_bytes(int64_t batch, int64_t tokens, int heads, int kv_heads, int head_dim) {
  return batch > 0 && tokens > 0 && heads > 0 && kv_heads > 0 && head_dim > 0 ? 16 : 0;
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
  PSA_REQUIRE(kv_heads > 0 && heads > 0 && heads % kv_heads == 0 && heads < 65536, PSA_ERR_ARG, "psa_kv4_attention: %d heads on %d key heads", heads,
              kv_heads);
  PSA_REQUIRE(batch > 0 && batch < 65536 && tokens > 0 && tokens < 65536, PSA_ERR_ARG, "psa_kv4_attention: %lld requests, %lld tokens",
              (long long)batch, (long long)tokens);
  PSA_REQUIRE((((uintptr_t)data | (uintptr_t)q | (uintptr_t)out) & 15) == 0, PSA_ERR_ARG, "psa_kv4_attention: operands must be 16-byte aligned");
  for (int i = 0; i < 3; ++i)
    PSA_REQUIRE(q_strides[i] % 8 == 0 && out_strides[i] % 8 == 0, PSA_ERR_ARG, "psa_kv4_attention: strides must be multiples of 8 elements");
  PSA_REQUIRE(scratch_bytes >= psa_kv4_attention_scratch_bytes(batch, tokens, heads, kv_heads, head_dim), PSA_ERR_ARG,
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
  a.width = (int)width;
  a.page = page_size;
  a.scale = sm_scale;
  const dim3 grid((unsigned)tokens, (unsigned)heads, (unsigned)batch);
  PSA_DISPATCH_KV4(dtype, head_dim, group, T, D, G, kv4_attn_rows_kernel<T, D, G><<<grid, 128, 0, (cudaStream_t)stream>>>(a));
  PSA_CHECK_LAUNCH("psa_kv4_attention");
  return PSA_OK;
}
