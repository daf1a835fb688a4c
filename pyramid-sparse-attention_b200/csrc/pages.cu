// Block tables, request lengths and slot maps of a cache in pages, made on the GPU: a step of a server whose sizes the host does
// not read back, so that it can be captured in a CUDA graph.
//
// Request b holds ceil(length / page) pages, listed in row b of the table.  It is given room for count more tokens: the pages it
// lacks come from the top of the pool of free pages, in the order of the requests, which makes their places an exclusive prefix sum
// over the requests' needs.  A request that needs pages gets them as long as the running total of all needs up to it fits the pool;
// the others are given no room at all.  Integers only, and a few thousand of them: a step is bound by the launch and by a chain of
// dependent loads, not by a rate: 64 requests and one token 3.0 us, 250 requests with 8192 slots each 5.9 us (8.2 MB of slots; 9.4 with a
// number a thread and a division each).
#include "psa_common.cuh"

namespace psa {
namespace {

constexpr int kPlanThreads = 1024;
constexpr int64_t kFewEntries = 1 << 15;   // slots that one block writes about as fast as a second launch starts

// Of each request, for the second kernel: pages held before, pages given, place of the first given page from the top of the
// pool, tokens given, length before.
struct Grant {
  int32_t held, given, first, tokens, length;
};

template <int THREADS = kPlanThreads>
__device__ __forceinline__ int block_scan(int x, int* warp_sums) {   // inclusive; warp_sums: 32 words, the last one gets the whole sum
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int d = 1; d < 32; d *= 2) {
    const int y = __shfl_up_sync(~0u, x, d);
    if (lane >= d) x += y;
  }
  if (lane == 31) warp_sums[warp] = x;
  __syncthreads();
  if (warp == 0) {
    int s = lane < THREADS / 32 ? warp_sums[lane] : 0;
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

// Tokens below 2^31.  Pages of a power of two (shift >= 0) need no division.
__device__ __forceinline__ int page_of(int token, int page, int shift) { return shift >= 0 ? token >> shift : (int)((uint32_t)token / (uint32_t)page); }
__device__ __forceinline__ int pages_of(int tokens, int page, int shift) {
  const uint32_t up = (uint32_t)tokens + (uint32_t)page - 1u;
  return (int)(shift >= 0 ? up >> shift : up / (uint32_t)page);
}

struct PlanArgs {
  const int32_t *table, *lengths, *counts, *pool, *free_in;
  int32_t *table_out, *lengths_out, *free_out, *slots, *status;
  Grant* grants;
  int32_t* free_before;
  int requests, width, pool_size, page, tokens, shift;
  bool fours;   // rows of the table and of the slots are whole 16-byte words
};

// What a request holds, wants and has a right to want.
struct Want {
  int length, count, held, need;
  bool bad;
};
__device__ __forceinline__ Want want_of(const PlanArgs& a, int b) {
  Want w;
  w.length = a.lengths[b];
  w.count = a.counts[b];
  const int64_t most = (int64_t)a.width * a.page;
  w.bad = w.length < 0 || w.length > most || w.count < 0 || w.count > a.tokens || (int64_t)w.length + w.count > most;
  if (w.bad) w.count = 0;
  w.held = pages_of(min(max(w.length, 0), (int)most), a.page, a.shift);
  w.need = w.bad ? 0 : pages_of(w.length + w.count, a.page, a.shift) - w.held;
  return w;
}
__device__ __forceinline__ Grant grant_of(const PlanArgs& a, const Want& w, int total, int available) {
  const bool served = w.need == 0 || total <= available;
  if (!served || w.bad) report(a.status, PSA_ERR_ARG);
  return {w.held, served ? w.need : 0, total - w.need, served ? w.count : 0, w.length};
}

// Entries [from, to) of a row, four neighbours a thread (`own` of `threads`), as `value` gives them.
template <typename F>
__device__ __forceinline__ void fill(int32_t* row, bool fours, int from, int to, int own, int threads, F value) {
  for (int j = (from & ~3) + 4 * own; j < to; j += 4 * threads) {
    int x[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = j + i >= from && j + i < to ? value(j + i) : 0;
    if (fours && j >= from && j + 3 < to) {
      *reinterpret_cast<int4*>(row + j) = make_int4(x[0], x[1], x[2], x[3]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (j + i >= from && j + i < to) row[j + i] = x[i];
    }
  }
}

// Part [from, to) of a request's row of the table - in place, of its new pages only - and of its slots.
__device__ __forceinline__ void fill_row(const PlanArgs& a, int b, const Grant& g, int available, int from, int to, int own, int threads) {
  const int top = available - 1 - g.first, most_pages = 0x7fffffff / a.page;
  const int32_t* table = a.table + (int64_t)b * a.width;
  int32_t* table_out = a.table_out + (int64_t)b * a.width;
  const bool in_place = table_out == table;
  fill(table_out, a.fours, in_place ? max(from, g.held) : from, min(to, in_place ? g.held + g.given : a.width), own, threads,
       [&](int j) { return j >= g.held && j < g.held + g.given ? a.pool[top - (j - g.held)] : table[j]; });
  int last = -1, page = -1;   // the page looked up before
  fill(a.slots + (int64_t)b * a.tokens, a.fours, from, min(to, a.tokens), own, threads, [&](int j) {
    if (j >= g.tokens) return -1;
    const int at = g.length + j, k = page_of(at, a.page, a.shift);
    if (k != last) {
      last = k;
      page = k < g.held ? table[k] : a.pool[top - (k - g.held)];
      if ((uint32_t)page >= (uint32_t)most_pages) {   // no slot has such a number
        page = -1;
        report(a.status, PSA_ERR_ARG);
      }
    }
    return page >= 0 ? page * a.page + (at - k * a.page) : -1;
  });
}

// Outputs beside the inputs, up to kPlanThreads requests: a block fills a stretch of a request's row and sums the needs of the requests
// before it for itself - a few hundred numbers that all blocks find in L2 - which spares a launch that would do nothing else.
constexpr int kRowThreads = 256, kRowEntries = 4096;
__global__ void __launch_bounds__(kRowThreads) plan_rows_kernel(const PlanArgs a) {
  __shared__ int warp_sums[32], taken;
  const int b = blockIdx.y, available = min(max(a.free_in[0], 0), a.pool_size);
  int before = 0;
  for (int i = threadIdx.x; i < b; i += kRowThreads) before += want_of(a, i).need;
  block_scan<kRowThreads>(before, warp_sums);
  const Want w = want_of(a, b);
  const Grant g = grant_of(a, w, warp_sums[31] + w.need, available);
  fill_row(a, b, g, available, blockIdx.x * kRowEntries, (blockIdx.x + 1) * kRowEntries, threadIdx.x, kRowThreads);
  if (blockIdx.x) return;
  if (threadIdx.x == 0) a.lengths_out[b] = g.length + g.tokens;
  if (b) return;
  // pages taken: the largest running total that fits
  if (threadIdx.x == 0) taken = 0;
  int total = 0;
  for (int b0 = 0; b0 < a.requests; b0 += kRowThreads) {
    const int i = b0 + threadIdx.x;
    __syncthreads();
    const int sum = total + block_scan<kRowThreads>(i < a.requests ? want_of(a, i).need : 0, warp_sums);
    if (i < a.requests && sum <= available) atomicMax(&taken, sum);
    total += warp_sums[31];
  }
  __syncthreads();
  if (threadIdx.x == 0) a.free_out[0] = available - taken;
}

// Outputs that may be the inputs' own memory.  Who gets what, and the new lengths: one block, requests in rounds of one a thread.  It
// fills the rows too where that is little (FILL); another kernel does where it is much.
template <bool FILL>
__global__ void __launch_bounds__(kPlanThreads) plan_kernel(const PlanArgs a) {
  __shared__ int warp_sums[32], taken;
  __shared__ Grant given[FILL ? kPlanThreads : 1];
  const int available = min(max(a.free_in[0], 0), a.pool_size);
  if (threadIdx.x == 0) taken = 0;
  int before = 0;   // needs of the rounds so far
  for (int b0 = 0; b0 < a.requests; b0 += kPlanThreads) {
    const int b = b0 + threadIdx.x;
    Want w = {};
    if (b < a.requests) w = want_of(a, b);
    const int total = before + block_scan(w.need, warp_sums);
    if (b < a.requests) {
      const Grant g = grant_of(a, w, total, available);
      if (g.given) atomicMax(&taken, total);
      if (FILL) given[threadIdx.x] = g;
      else a.grants[b] = g;
      a.lengths_out[b] = g.length + g.tokens;
    }
    before += warp_sums[31];
    __syncthreads();
    if (FILL) {
      const int n = min(kPlanThreads, a.requests - b0);
      for (int i = threadIdx.x >> 5; i < n; i += kPlanThreads / 32) {   // a warp a request: its new pages, its slots
        const Grant g = given[i];
        fill_row(a, b0 + i, g, available, 0, max(a.tokens, a.width), threadIdx.x & 31, 32);
      }
      __syncthreads();
    }
  }
  if (threadIdx.x == 0) {
    if (!FILL) *a.free_before = available;
    a.free_out[0] = available - taken;
  }
}

__global__ void __launch_bounds__(kRowThreads) fill_kernel(const PlanArgs a) {
  const int b = blockIdx.y;
  fill_row(a, b, a.grants[b], *a.free_before, blockIdx.x * kRowEntries, (blockIdx.x + 1) * kRowEntries, threadIdx.x, kRowThreads);
}

// Pages of the requests marked in `which` go back on top of the pool, the last request's last page first: a request that is given
// room and released at once leaves the pool as it was.  64 requests of 126 pages 4.1 us, 250 of 128 9.8.  Entries with numbers that no slot
// can have stay away and leave no gap: where a round of requests has some, it is done again by the numbers of good entries.  (To count
// those first took 5.3 and 14.3 us.)
__global__ void __launch_bounds__(kPlanThreads) release_kernel(const int32_t* table, int32_t* lengths, const uint8_t* which, int32_t* pool,
                                                               int32_t* free_count, int requests, int width, int pool_size, int page,
                                                               int32_t* status) {
  __shared__ int warp_sums[32], held_of[kPlanThreads], end_of[kPlanThreads];
  const int top = min(max(free_count[0], 0), pool_size), lane = threadIdx.x & 31, most = width * page;
  const uint32_t most_pages = 0x7fffffffu / page;
  int before = 0;
  for (int b0 = 0; b0 < requests; b0 += kPlanThreads) {
    const int b = requests - 1 - (b0 + (int)threadIdx.x);
    int held = 0;
    if (b >= 0 && which[b]) {
      const int length = lengths[b];
      if (length < 0 || length > most) report(status, PSA_ERR_ARG);
      held = pages_of(min(max(length, 0), most), page, -1);
      lengths[b] = 0;
    }
    held_of[threadIdx.x] = held;
    end_of[threadIdx.x] = before + block_scan(held, warp_sums);
    const int all = warp_sums[31];
    __syncthreads();
    const int n = min(kPlanThreads, requests - b0);
    bool stays = false;
    for (int i = threadIdx.x >> 5; i < n; i += kPlanThreads / 32) {   // a warp moves a request's pages
      const int32_t* row = table + (int64_t)(requests - 1 - (b0 + i)) * width;
      for (int j = lane; j < held_of[i]; j += 32) {
        const int64_t at = (int64_t)top + end_of[i] - 1 - j;
        const int number = row[j];
        if ((uint32_t)number < most_pages && at < pool_size) pool[at] = number;
        else stays = true;
      }
    }
    if (!__syncthreads_or(stays)) {
      before += all;
      continue;
    }
    if (threadIdx.x == 0) report(status, PSA_ERR_ARG);
    for (int i = threadIdx.x >> 5; i < n; i += kPlanThreads / 32) {   // how many go back
      const int32_t* row = table + (int64_t)(requests - 1 - (b0 + i)) * width;
      int good = 0;
      for (int j = lane; j < held_of[i]; j += 32) good += (uint32_t)row[j] < most_pages;
      good = __reduce_add_sync(~0u, good);
      if (lane == 0) end_of[i] = good;
    }
    __syncthreads();
    const int end = before + block_scan((int)threadIdx.x < n ? end_of[threadIdx.x] : 0, warp_sums);
    end_of[threadIdx.x] = end;
    before += warp_sums[31];
    __syncthreads();
    for (int i = threadIdx.x >> 5; i < n; i += kPlanThreads / 32) {
      const int32_t* row = table + (int64_t)(requests - 1 - (b0 + i)) * width;
      int64_t at = (int64_t)top + end_of[i] - 1;   // of the first page of 32
      for (int j0 = 0; j0 < held_of[i]; j0 += 32) {
        const int number = j0 + lane < held_of[i] ? row[j0 + lane] : -1;
        const uint32_t mask = __ballot_sync(~0u, (uint32_t)number < most_pages);
        const int64_t to = at - __popc(mask & ((1u << lane) - 1));
        if ((uint32_t)number < most_pages && to < pool_size) pool[to] = number;
        at -= __popc(mask);
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
  PSA_REQUIRE(table && lengths && counts && pool && free_in && table_out && lengths_out && free_out && slots && status, PSA_ERR_ARG,
              "psa_plan_pages: null pointer");
  if (int rc = check_sizes("psa_plan_pages", requests, width, pool_size, page_size)) return rc;
  // blocks read counts and pool while others write: an output may be its own input's memory, not another's
  for (const int32_t* out : {(const int32_t*)table_out, (const int32_t*)lengths_out, (const int32_t*)free_out, (const int32_t*)slots})
    PSA_REQUIRE(out != counts && out != pool && (out == table_out || out != table) && (out == lengths_out || out != lengths) &&
                    (out == free_out || out != free_in), PSA_ERR_ARG, "psa_plan_pages: an output in another input's memory");
  PSA_REQUIRE(table_out != lengths_out && table_out != free_out && table_out != slots && lengths_out != free_out && lengths_out != slots &&
                  free_out != slots, PSA_ERR_ARG, "psa_plan_pages: two outputs in the same memory");
  PSA_REQUIRE(tokens > 0 && tokens <= ((int64_t)1 << 30), PSA_ERR_ARG, "psa_plan_pages: %lld tokens", (long long)tokens);
  const int64_t wide = width > tokens ? width : tokens;
  const bool apart = lengths_out != lengths && free_out != free_in && table_out != table && requests <= kPlanThreads;
  const bool few = requests * (table_out == table ? tokens : wide) <= kFewEntries;
  PSA_REQUIRE(apart || (scratch && scratch_bytes >= psa_plan_pages_scratch_bytes(requests)), PSA_ERR_ARG, "psa_plan_pages: scratch of %zu bytes",
              scratch_bytes);
  cudaStream_t st = (cudaStream_t)stream;
  PlanArgs a = {table, lengths, counts, pool, free_in, table_out, lengths_out, free_out, slots, status,
                reinterpret_cast<Grant*>(static_cast<char*>(scratch) + 16), static_cast<int32_t*>(scratch), (int)requests, (int)width, (int)pool_size,
                page_size, (int)tokens, -1, false};
  if ((page_size & (page_size - 1)) == 0)
    for (a.shift = 0; 1 << a.shift < page_size;) ++a.shift;
  a.fours = ((((uintptr_t)table_out | (uintptr_t)slots) & 15) | (uintptr_t)(width & 3) | (uintptr_t)(tokens & 3)) == 0;
  const dim3 rows((unsigned)cdiv64(wide, kRowEntries), (unsigned)requests);
  if (apart) {
    plan_rows_kernel<<<rows, kRowThreads, 0, st>>>(a);
  } else if (few) {
    plan_kernel<true><<<1, kPlanThreads, 0, st>>>(a);
  } else {
    plan_kernel<false><<<1, kPlanThreads, 0, st>>>(a);
    PSA_CHECK_LAUNCH("psa_plan_pages");
    fill_kernel<<<rows, kRowThreads, 0, st>>>(a);
  }
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
