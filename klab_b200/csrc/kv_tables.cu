// Page tables of a batch of requests, built on the GPU: which pages the new tokens of a step get, where each token goes,
// and the pages that ended requests give back. Stands beside the single-sequence cache of decode_attn.cu, whose append
// position is one length.
//
// Step: request i holds ceil(l_i / P) pages and needs ceil((l_i + n_i) / P); the k-th new page (requests in order, pages
// in order) is the k-th from the top of the free stack, so the result depends on no order of execution. Token x belongs
// to the request whose range of `starts` holds it; its position is l_i + x - starts_i and its slot
// table[i][position / P] * P + position mod P.
//
// What bounds it: latency. A step of 8 requests moves 236 bytes, one of 1024 requests with 100 thousand new tokens 1.4 MB.
// Each CTA scans all requests by itself (two running sums, kept in shared memory), then takes its share of the tokens and
// new pages, finding the request by bisection in shared memory, so one long prompt spreads over every thread. State that is
// updated in place must not be written before every CTA has read it: then the CTAs form one cluster (at most 8) and its
// barrier stands between. Otherwise up to 128 CTAs share the work (1024 requests, 110 thousand tokens: 5.4 us, and in place
// with 8 CTAs 17; 8 requests of one token 2.5 us and 2.8). Release is one CTA, whose threads take the pages in turn: 166 pages
// 2.2 us, 7414 13.7, 15651 25.
#include <atomic>
#include <climits>
#include <cstdint>

#include "common.cuh"
#include "klab_b200.h"
#include "klab_kernels.h"
#include "kv_pages.cuh"
#include "launch.cuh"

namespace klab {
namespace {

constexpr int kStepThreads = 1024;
constexpr int kStepClusterTokens = 2048;  // tokens that one CTA of the cluster takes before another is added
constexpr int kStepClusterCtas = 8, kStepMaxCtas = 128;

struct Sums {
  long long tokens, pages;
};

__device__ __forceinline__ Sums operator+(Sums a, Sums b) { return {a.tokens + b.tokens, a.pages + b.pages}; }

__device__ __forceinline__ Sums shfl_up(Sums v, int d) {
  return {__shfl_up_sync(0xffffffffu, v.tokens, d), __shfl_up_sync(0xffffffffu, v.pages, d)};
}

// Inclusive scan over the block's threads; `parts` holds 32 entries. Two barriers.
__device__ Sums block_scan(Sums v, Sums* parts) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const Sums up = shfl_up(v, d);
    if (lane >= d) v = v + up;
  }
  if (lane == 31) parts[warp] = v;
  __syncthreads();
  if (warp == 0) {
    Sums w = lane < warps ? parts[lane] : Sums{0, 0};
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const Sums up = shfl_up(w, d);
      if (lane >= d) w = w + up;
    }
    parts[lane] = w;
  }
  __syncthreads();
  return warp ? v + parts[warp - 1] : v;
}

// The last i in [0, n) with first[i] <= x (first[0] = 0 <= x).
__device__ __forceinline__ int last_not_above(const int* first, int n, int x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (first[mid] <= x)
      lo = mid;
    else
      hi = mid;
  }
  return lo;
}

struct StepParams {
  const int* new_tokens;
  const int* lengths;
  int* table;
  const int* free_pages;
  const int* free_count;
  int* slots;
  int* positions;
  int* rows;
  int* starts;
  int* lengths_out;
  int* free_count_out;
  int* result;
  int* status;
  int requests, width, num_pages, page_shift, max_tokens;
};

__global__ void __launch_bounds__(kStepThreads) build_step_kernel(const StepParams p) {
  extern __shared__ int sm[];
  int* first = sm;                      // [requests] first token of each request
  int* fresh = sm + p.requests;         // [requests] first new page of each request
  int* cached = sm + 2 * p.requests;    // [requests] tokens before the step
  __shared__ Sums parts[32];
  __shared__ int bad;
  const int tid = threadIdx.x, threads = blockDim.x, full = (1 << p.page_shift) - 1;
  grid_dependency_wait();
  grid_launch_dependents();
  if (tid == 0) bad = KLAB_STEP_OK;
  __syncthreads();
  Sums total = {0, 0};
  for (int base = 0; base < p.requests; base += threads) {
    const int i = base + tid;
    Sums mine = {0, 0};
    if (i < p.requests) {
      const int n = p.new_tokens[i], l = p.lengths[i];
      cached[i] = l;
      if (n < 0 || l < 0) {
        atomicMax(&bad, KLAB_STEP_LENGTH);
      } else {
        const long long need = (static_cast<long long>(l) + n + full) >> p.page_shift;
        const long long have = (static_cast<long long>(l) + full) >> p.page_shift;
        if (need > p.width) atomicMax(&bad, KLAB_STEP_TABLE);
        mine = {n, need - have};
      }
    }
    const Sums upto = block_scan(mine, parts);
    if (i < p.requests) {  // truncated only where a sum passes its limit, and then nothing is used
      first[i] = static_cast<int>(total.tokens + upto.tokens - mine.tokens);
      fresh[i] = static_cast<int>(total.pages + upto.pages - mine.pages);
    }
    total = total + parts[31];
    __syncthreads();
  }
  const int count = *p.free_count;
  int code = bad;
  if (code == KLAB_STEP_OK) {
    if (total.tokens > p.max_tokens)
      code = KLAB_STEP_TOKENS;
    else if (count < 0 || count > p.num_pages || total.pages > count)
      code = KLAB_STEP_PAGES;
  }
  const bool good = code == KLAB_STEP_OK;
  const int tokens = good ? static_cast<int>(total.tokens) : 0, pages = good ? static_cast<int>(total.pages) : 0;
  const int stride = gridDim.x * threads, at = blockIdx.x * threads + tid;
  bool wrong = false;
  for (long long x = at; x < p.max_tokens; x += stride) {
    int slot = -1, position = 0, row = -1;
    if (x < tokens) {
      row = last_not_above(first, p.requests, static_cast<int>(x));
      const int l = cached[row];
      position = l + static_cast<int>(x) - first[row];
      const int have = static_cast<int>((static_cast<unsigned>(l) + full) >> p.page_shift), page = position >> p.page_shift;
      const int id = page < have ? p.table[static_cast<long long>(row) * p.width + page]
                                 : p.free_pages[count - 1 - (fresh[row] + page - have)];
      if (id < 0 || id >= p.num_pages)
        wrong = true;
      else
        slot = (id << p.page_shift) + (position & full);
    }
    p.slots[x] = slot;
    p.positions[x] = position;
    p.rows[x] = row;
  }
  for (int k = at; k < pages; k += stride) {
    const int row = last_not_above(fresh, p.requests, k);
    const int have = static_cast<int>((static_cast<unsigned>(cached[row]) + full) >> p.page_shift);
    p.table[static_cast<long long>(row) * p.width + have + k - fresh[row]] = p.free_pages[count - 1 - k];
  }
  if (wrong) record_status(p.status, kStatusBadPage);
  // In place: every CTA of the cluster has read the old lengths and count, the state may be written over them.
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  if (blockIdx.x == 0) {
    for (int i = tid; i < p.requests; i += threads) {
      const int l = cached[i];
      const int next = i + 1 < p.requests ? first[i + 1] : tokens;
      p.starts[i] = good ? first[i] : 0;
      p.lengths_out[i] = good ? l + next - first[i] : l;
    }
    if (tid == 0) {
      p.starts[p.requests] = tokens;
      *p.free_count_out = good ? count - pages : count;
      *p.result = code;
      if (!good) record_status(p.status, kStatusStepRefused);
    }
  }
}

// Ended requests give their pages back: one CTA, a first pass that checks every page, a second that pushes them.
__global__ void __launch_bounds__(kStepThreads) release_kernel(const unsigned char* ended, int* lengths, int* table,
                                                               int* free_pages, int* free_count, int* status,
                                                               int requests, int width, int num_pages,
                                                               int page_size) {
  extern __shared__ int sm[];
  int* first = sm;  // [requests] pages given back before this request's
  __shared__ Sums parts[32];
  const int tid = threadIdx.x, threads = blockDim.x;
  grid_dependency_wait();
  grid_launch_dependents();
  int wrong = 0;
  Sums total = {0, 0};
  for (int base = 0; base < requests; base += threads) {
    const int i = base + tid;
    Sums mine = {0, 0};
    if (i < requests && ended[i]) {
      const int l = lengths[i];
      const long long have = (static_cast<long long>(l) + page_size - 1) / page_size;
      if (l < 0 || have > width)
        wrong = 1;
      else
        mine.pages = have;
    }
    const Sums upto = block_scan(mine, parts);
    if (i < requests) first[i] = static_cast<int>(total.pages + upto.pages - mine.pages);
    total = total + parts[31];
    __syncthreads();
  }
  const int count = *free_count;
  if (count < 0 || count + total.pages > num_pages) wrong = 1;
  wrong = __syncthreads_or(wrong);
  const int pages = wrong ? 0 : static_cast<int>(total.pages);
  for (int k = tid; k < pages; k += threads) {
    const int row = last_not_above(first, requests, k);
    const int id = table[static_cast<long long>(row) * width + k - first[row]];
    if (id < 0 || id >= num_pages) wrong = 1;
  }
  if (__syncthreads_or(wrong)) {  // nothing is given back
    if (tid == 0) record_status(status, kStatusBadPage);
    return;
  }
  for (int k = tid; k < pages; k += threads) {
    const int row = last_not_above(first, requests, k);
    int* entry = table + static_cast<long long>(row) * width + k - first[row];
    free_pages[count + k] = *entry;
    *entry = -1;
  }
  for (int i = tid; i < requests; i += threads)
    if (ended[i]) lengths[i] = 0;
  if (tid == 0) *free_count = count + pages;
}

std::atomic<unsigned long long> g_step_ready{0};  // devices whose kernels may use large shared memory

int prepare_step_device() {
  int dev = 0;
  cudaError_t err = cudaGetDevice(&dev);
  if (err != cudaSuccess) return err;
  if (dev < 0 || dev >= 64) return KLAB_E_UNSUPPORTED;
  if (g_step_ready.load() >> dev & 1) return 0;
  err = cudaFuncSetAttribute(build_step_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 12 * kKvMaxRequests);
  if (err != cudaSuccess) return err;
  err = cudaFuncSetAttribute(release_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 4 * kKvMaxRequests);
  if (err != cudaSuccess) return err;
  g_step_ready.fetch_or(1ull << dev);
  return 0;
}

int check_tables(int requests, int width, int num_pages, int page_size) {
  if (requests <= 0 || width <= 0 || num_pages <= 0) return KLAB_E_INVALID;
  if (requests > kKvMaxRequests || !kv_page_size_ok(page_size)) return KLAB_E_SHAPE;
  if (static_cast<long long>(num_pages) * page_size > INT_MAX || static_cast<long long>(width) * page_size > INT_MAX)
    return KLAB_E_SHAPE;
  return 0;
}

}  // namespace
}  // namespace klab

extern "C" {

KLAB_API int klab_kv_build_step(const int* new_tokens, const int* lengths, int* table, const int* free_pages,
                                const int* free_count, int requests, int width, int num_pages, int page_size,
                                int max_tokens, int* slots, int* positions, int* rows, int* starts, int* lengths_out,
                                int* free_count_out, int* result, void* stream) {
  using namespace klab;
  if (!new_tokens || !lengths || !table || !free_pages || !free_count || !slots || !positions || !rows || !starts ||
      !lengths_out || !free_count_out || !result || max_tokens <= 0)
    return KLAB_E_INVALID;
  int rc = check_tables(requests, width, num_pages, page_size);
  if (rc) return rc;
  if ((rc = prepare_step_device())) return rc;
  StepParams p{new_tokens, lengths, table,    free_pages,     free_count, slots,
               positions,  rows,    starts,   lengths_out,    free_count_out, result,
               device_status_address(), requests, width, num_pages, kv_page_shift(page_size), max_tokens};
  const bool inplace = lengths_out == lengths || free_count_out == free_count;
  int threads = 128, ctas = 1;
  const int busy = max_tokens > requests ? max_tokens : requests;
  while (threads < kStepThreads && threads < busy) threads *= 2;
  if (inplace) {
    while (ctas < kStepClusterCtas && static_cast<long long>(ctas) * kStepClusterTokens < max_tokens) ctas *= 2;
  } else {
    ctas = (max_tokens - 1) / threads + 1;
    if (ctas > kStepMaxCtas) ctas = kStepMaxCtas;
  }
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  cfg.gridDim = dim3(static_cast<unsigned>(ctas));
  cfg.blockDim = dim3(static_cast<unsigned>(threads));
  cfg.dynamicSmemBytes = 12 * static_cast<size_t>(requests);
  cfg.stream = static_cast<cudaStream_t>(stream);
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(inplace ? ctas : 1);
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = klab_get_option(KLAB_OPT_PDL) ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, build_step_kernel, p);
}

KLAB_API int klab_kv_release(const unsigned char* ended, int* lengths, int* table, int* free_pages, int* free_count,
                             int requests, int width, int num_pages, int page_size, void* stream) {
  using namespace klab;
  if (!ended || !lengths || !table || !free_pages || !free_count) return KLAB_E_INVALID;
  int rc = check_tables(requests, width, num_pages, page_size);
  if (rc) return rc;
  if ((rc = prepare_step_device())) return rc;
  return launch_dependent(release_kernel, dim3(1), kStepThreads, 4 * static_cast<size_t>(requests), stream, ended, lengths, table,
                          free_pages, free_count, device_status_address(), requests, width, num_pages, page_size);
}

}  // extern "C"
