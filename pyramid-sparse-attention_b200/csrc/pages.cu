// Block tables, request lengths and slot maps of a cache in pages, made on the GPU: a step of a server whose sizes the host does
// not read back, so that it can be captured in a CUDA graph.
//
// Request b holds ceil(length / page) pages, listed in row b of the table.  It is given room for count more tokens: the pages it
// lacks come from the top of the pool of free pages, in the order of the requests, which makes their places an exclusive prefix sum
// over the requests' needs.  A request that needs pages gets them as long as the running total of all needs up to it fits the pool;
// the others are given no room at all.  Integers only, and a few thousand of them: a step is bound by the launch and by a chain of
// dependent loads, not by a rate.
#include "psa_common.cuh"

namespace psa {
namespace {

constexpr int kPlanThreads = 1024;

// Of each request, for the second kernel: pages held before, pages given, place of the first given page from the top of the
// pool, tokens given, length before.
struct Grant {
  int32_t held, given, first, tokens, length;
};

__device__ __forceinline__ int block_scan(int x, int* warp_sums) {   // inclusive, over kPlanThreads
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int d = 1; d < 32; d *= 2) {
    const int y = __shfl_up_sync(~0u, x, d);
    if (lane >= d) x += y;
  }
  if (lane == 31) warp_sums[warp] = x;
  __syncthreads();
  if (warp == 0) {
    int s = warp_sums[lane];
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
      const int y = __shfl_up_sync(~0u, s, d);
      if (lane >= d) s += y;
    }
    warp_sums[lane] = s;
  }
  __syncthreads();
  return x + (warp ? warp_sums[warp - 1] : 0);
}

__device__ __forceinline__ int pages_of(int64_t tokens, int page) { return (int)((tokens + page - 1) / page); }

// Who gets what, and the new lengths.  One block, requests in rounds of one a thread.
__global__ void __launch_bounds__(kPlanThreads) plan_kernel(const int32_t* lengths, const int32_t* counts, const int32_t* free_in,
                                                            int32_t* lengths_out, int32_t* free_out, Grant* grants, int32_t* free_before,
                                                            int requests, int width, int pool_size, int page, int tokens,
                                                            int32_t* status) {
  __shared__ int warp_sums[32];
  __shared__ int taken;
  const int available = min(max(free_in[0], 0), pool_size);
  if (threadIdx.x == 0) taken = 0;
  int before = 0;   // needs of the rounds so far
  for (int b0 = 0; b0 < requests; b0 += kPlanThreads) {
    const int b = b0 + threadIdx.x;
    int length = 0, count = 0, held = 0, need = 0;
    bool bad = false;
    if (b < requests) {
      length = lengths[b];
      count = counts[b];
      bad = length < 0 || length > (int64_t)width * page || count < 0 || count > tokens || (int64_t)length + count > (int64_t)width * page;
      if (bad) count = 0;
      held = pages_of(min(max(length, 0), width * page), page);
      need = bad ? 0 : pages_of((int64_t)length + count, page) - held;
    }
    const int total = before + block_scan(need, warp_sums);
    if (b < requests) {
      const bool served = need == 0 || total <= available;
      if (!served || bad) *status = PSA_ERR_ARG;
      if (!served) count = 0;
      else if (need) atomicMax(&taken, total);
      grants[b] = {held, served ? need : 0, total - need, count, length};
      lengths_out[b] = length + count;
    }
    before += warp_sums[31];
    __syncthreads();
  }
  if (threadIdx.x == 0) {
    *free_before = available;
    *free_out = available - taken;
  }
}

// The tables' rows and the slots of the new tokens.
__global__ void __launch_bounds__(256) fill_kernel(const int32_t* table, const int32_t* pool, const Grant* grants, const int32_t* free_before,
                                                   int32_t* table_out, int32_t* slots, int width, int page, int tokens) {
  const int b = blockIdx.y;
  const Grant g = grants[b];
  const int top = *free_before - 1 - g.first;
  for (int j = blockIdx.x * blockDim.x + threadIdx.x; j < max(width, tokens); j += gridDim.x * blockDim.x) {
    if (j < width) {
      const bool fresh = j >= g.held && j < g.held + g.given;
      if (fresh || table_out != table) table_out[(int64_t)b * width + j] = fresh ? pool[top - (j - g.held)] : table[(int64_t)b * width + j];
    }
    if (j < tokens) {
      int slot = -1;
      if (j < g.tokens) {
        const int at = g.length + j, k = at / page;
        const int p = k < g.held ? table[(int64_t)b * width + k] : pool[top - (k - g.held)];
        if (p >= 0 && p < 0x7fffffff / page) slot = p * page + at % page;
      }
      slots[(int64_t)b * tokens + j] = slot;
    }
  }
}

// Pages of the requests marked in `which` go back on top of the pool, the last request's last page first: a request that is given
// room and released at once leaves the pool as it was.
__global__ void __launch_bounds__(kPlanThreads) release_kernel(const int32_t* table, int32_t* lengths, const uint8_t* which, int32_t* pool,
                                                               int32_t* free_count, int requests, int width, int pool_size, int page,
                                                               int32_t* status) {
  __shared__ int warp_sums[32], held_of[kPlanThreads], end_of[kPlanThreads];
  const int top = min(max(free_count[0], 0), pool_size);
  int before = 0;
  for (int b0 = 0; b0 < requests; b0 += kPlanThreads) {
    const int b = requests - 1 - (b0 + (int)threadIdx.x);
    int held = 0;
    if (b >= 0 && which[b]) held = pages_of(min(max(lengths[b], 0), width * page), page);
    held_of[threadIdx.x] = held;
    end_of[threadIdx.x] = before + block_scan(held, warp_sums);
    if (held) lengths[b] = 0;
    before += warp_sums[31];
    __syncthreads();
    const int n = min(kPlanThreads, requests - b0);
    for (int i = threadIdx.x >> 5; i < n; i += kPlanThreads / 32) {   // a warp moves a request's pages
      const int32_t* row = table + (int64_t)(requests - 1 - (b0 + i)) * width;
      for (int j = threadIdx.x & 31; j < held_of[i]; j += 32) {
        const int64_t at = (int64_t)top + end_of[i] - 1 - j;
        if (at < pool_size) pool[at] = row[j];
        else *status = PSA_ERR_ARG;
      }
    }
    __syncthreads();
  }
  if (threadIdx.x == 0) free_count[0] = (int)min((int64_t)top + before, (int64_t)pool_size);
}

int check_sizes(const char* what, int64_t requests, int64_t width, int64_t pool_size, int page) {
  PSA_REQUIRE(requests > 0 && requests < 65536 && width > 0 && page > 0 && page % 16 == 0, PSA_ERR_ARG,
              "%s: %lld requests (1 to 65535), %lld pages each, page size %d (a multiple of 16)", what, (long long)requests, (long long)width, page);
  PSA_REQUIRE(width < ((int64_t)1 << 31) / page && requests * width < ((int64_t)1 << 31) && pool_size > 0 && pool_size < ((int64_t)1 << 31) / page,
              PSA_ERR_ARG, "%s: token numbers of a request and of the pool, and pages of all requests, must stay below 2^31", what);
  return PSA_OK;
}

}  // namespace
}  // namespace psa

extern "C" size_t psa_plan_pages_scratch_bytes(int64_t requests) {
  return requests > 0 ? sizeof(psa::Grant) * (size_t)requests + 16 : 0;
}

extern "C" int psa_plan_pages(const int32_t* table, const int32_t* lengths, const int32_t* counts, const int32_t* pool, const int32_t* free_in,
                              int32_t* table_out, int32_t* lengths_out, int32_t* free_out, int32_t* slots, void* scratch, size_t scratch_bytes,
                              int64_t requests, int64_t width, int64_t pool_size, int page_size, int64_t tokens, int32_t* status, void* stream) {
  using namespace psa;
  PSA_REQUIRE(table && lengths && counts && pool && free_in && table_out && lengths_out && free_out && slots && scratch && status, PSA_ERR_ARG,
              "psa_plan_pages: null pointer");
  if (int rc = check_sizes("psa_plan_pages", requests, width, pool_size, page_size)) return rc;
  PSA_REQUIRE(tokens > 0 && tokens < ((int64_t)1 << 31) && scratch_bytes >= psa_plan_pages_scratch_bytes(requests), PSA_ERR_ARG,
              "psa_plan_pages: %lld tokens, scratch of %zu bytes", (long long)tokens, scratch_bytes);
  cudaStream_t st = (cudaStream_t)stream;
  int32_t* free_before = static_cast<int32_t*>(scratch);
  Grant* grants = reinterpret_cast<Grant*>(static_cast<char*>(scratch) + 16);
  plan_kernel<<<1, kPlanThreads, 0, st>>>(lengths, counts, free_in, lengths_out, free_out, grants, free_before, (int)requests, (int)width,
                                          (int)pool_size, page_size, (int)tokens, status);
  PSA_CHECK_LAUNCH("psa_plan_pages");
  const int64_t wide = width > tokens ? width : tokens;
  const dim3 grid((unsigned)(cdiv64(wide, 256) < 64 ? cdiv64(wide, 256) : 64), (unsigned)requests);
  fill_kernel<<<grid, 256, 0, st>>>(table, pool, grants, free_before, table_out, slots, (int)width, page_size, (int)tokens);
  PSA_CHECK_LAUNCH("psa_plan_pages");
  return PSA_OK;
}

extern "C" int psa_release_pages(const int32_t* table, int32_t* lengths, const uint8_t* which, int32_t* pool, int32_t* free_count,
                                 int64_t requests, int64_t width, int64_t pool_size, int page_size, int32_t* status, void* stream) {
  using namespace psa;
  PSA_REQUIRE(table && lengths && which && pool && free_count && status, PSA_ERR_ARG, "psa_release_pages: null pointer");
  if (int rc = check_sizes("psa_release_pages", requests, width, pool_size, page_size)) return rc;
  release_kernel<<<1, kPlanThreads, 0, (cudaStream_t)stream>>>(table, lengths, which, pool, free_count, (int)requests, (int)width, (int)pool_size,
                                                               page_size, status);
  PSA_CHECK_LAUNCH("psa_release_pages");
  return PSA_OK;
}
