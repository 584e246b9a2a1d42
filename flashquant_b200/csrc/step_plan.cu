// A step's block tables, slots and positions from the lengths of its requests, and the way back of the pages of
// finished requests.  Free pages are a stack in global memory; requests take from its top in their order.
//
// Bound: latency for a decode step (a few KB), the slots and positions written (16 bytes a token) for a prefill
// step.  One launch: every CTA finds the prefix sums over the requests for itself (8 bytes a request from the L2, no
// exchange), then takes a share of the pages and tokens.  Where the stack's height is updated in place it must not be
// written before all CTAs have read it: then they are one cluster, which has a barrier; else as many as there is work
// for.
//
// Measured: 256 requests of a token each 5.5 us, 64 prompts of 39 000 tokens 5.9, 1024 requests with 128 000 pages
// released 4.6; of these the launch takes 2, the lengths and the scan 2.
#include <algorithm>

#include "fq_common.cuh"

namespace fq {

constexpr int kPlanThreads = 1024;
constexpr int kPlanBatch = 4;  // pages or tokens of a thread whose loads are in flight together
constexpr int kPlanMaxRequests = 4096;

struct PlanArgs {
  const int32_t *context, *query;
  int32_t* table;
  int64_t table_stride;
  int width, requests, block_size;
  const int32_t* free_pages;
  int64_t capacity;
  const int32_t* free_count;
  int64_t room;               // slots and positions
  int32_t *seq_lens, *starts;
  int64_t *slots, *positions;
  uint8_t* served;
  int32_t* count_out;
};

// Sums of two 64-bit values over the requests in order, a run of `each` consecutive ones per thread: what stands
// before this thread's run.
__device__ __forceinline__ void plan_before(int64_t& x, int64_t& y, int64_t (*sums)[2], int tid) {
  const int lane = tid & 31, warp = tid >> 5;
  int64_t a = x, b = y;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t u = __shfl_up_sync(0xffffffffu, a, o), w = __shfl_up_sync(0xffffffffu, b, o);
    if (lane >= o) {
      a += u;
      b += w;
    }
  }
  if (lane == 31) {
    sums[warp][0] = a;
    sums[warp][1] = b;
  }
  __syncthreads();
  x = a - x;
  y = b - y;
  int64_t u = lane < warp ? sums[lane][0] : 0, w = lane < warp ? sums[lane][1] : 0;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    u += __shfl_xor_sync(0xffffffffu, u, o);
    w += __shfl_xor_sync(0xffffffffu, w, o);
  }
  x += u;
  y += w;
}
static_assert(kPlanThreads == 1024, "a lane to a warp's sums");

// A request as it is treated: a negative length or more pages than a row of the block table holds make it
// invalid, which counts as one without tokens.
struct PlanRequest {
  int32_t context, query;  // (query: 0 where invalid)
  int32_t grow;            // pages it takes
  bool valid;
};
__device__ __forceinline__ uint32_t plan_pages(uint32_t tokens, uint32_t block_size) {
  const uint32_t n = tokens / block_size;
  return n + (n * block_size != tokens);
}
__device__ __forceinline__ PlanRequest plan_request(const PlanArgs& p, int i) {
  PlanRequest r;
  r.context = p.context[i];
  r.query = p.query[i];
  r.valid = r.context >= 0 && r.query >= 0;
  r.grow = 0;
  if (r.valid) {  // (the sum of both fits into 32 bits without a sign)
    const uint32_t need = plan_pages(uint32_t(r.context) + uint32_t(r.query), p.block_size);
    r.valid = need <= uint32_t(p.width);
    if (r.valid && r.query > 0) r.grow = need - plan_pages(r.context, p.block_size);
  }
  if (!r.valid) r.query = 0;
  return r;
}

// the last i of [0, n) with first[i] <= x, of those with the same first the last
__device__ __forceinline__ int plan_owner(const int32_t* first, int n, int32_t x) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (first[mid] <= x) lo = mid; else hi = mid - 1;
  }
  return lo;
}

__global__ void __launch_bounds__(kPlanThreads) plan_step_kernel(const PlanArgs p) {
  extern __shared__ int32_t plan_smem[];
  int32_t* const starts = plan_smem;                  // [requests]: first token
  int32_t* const taken = plan_smem + p.requests;      // [requests]: first page off the stack
  __shared__ int64_t sums[kPlanThreads / 32][2];
  __shared__ int cut;                                 // the first request that does not fit
  __shared__ int32_t all_tokens, all_pages;
  const int tid = threadIdx.x;
  const int ctas = gridDim.x, cta = blockIdx.x;
  int64_t height = *p.free_count;
  height = height < 0 ? 0 : (height > p.capacity ? p.capacity : height);

  // ---- prefix sums ------------------------------------------------------------------------------------
  // Both sums only grow, so the requests that do not fit are a tail of those that need something.
  if (tid == 0) cut = p.requests;
  const int each = (p.requests + kPlanThreads - 1) / kPlanThreads;
  const int i0 = min(tid * each, p.requests), i1 = min(i0 + each, p.requests);
  PlanRequest mine{};  // (kept: up to 1024 requests each thread has one)
  if (i0 < i1) mine = plan_request(p, i0);
  auto request = [&](int i) { return i == i0 ? mine : plan_request(p, i); };
  int64_t tokens = 0, pages = 0;
  for (int i = i0; i < i1; ++i) {
    const PlanRequest r = request(i);
    tokens += r.query;
    pages += r.grow;
  }
  plan_before(tokens, pages, sums, tid);
  {
    int64_t t = tokens, g = pages;
    for (int i = i0; i < i1; ++i) {
      const PlanRequest r = request(i);
      t += r.query;
      g += r.grow;
      if (r.query > 0 && (t > p.room || g > height)) {
        atomicMin(&cut, i);
        break;
      }
    }
  }
  __syncthreads();
  for (int i = i0; i < i1; ++i) {
    const PlanRequest r = request(i);
    if (i <= cut) {  // (fits into 32 bits: all before `cut` do)
      starts[i] = int32_t(tokens);
      taken[i] = int32_t(pages);
    }
    if (i == cut || i == p.requests - 1) {
      if (i < cut) {
        all_tokens = int32_t(tokens + r.query);
        all_pages = int32_t(pages + r.grow);
      } else if (i == cut) {
        all_tokens = int32_t(tokens);
        all_pages = int32_t(pages);
      }
    }
    tokens += r.query;
    pages += r.grow;
  }
  if (p.requests == 0 && tid == 0) all_tokens = all_pages = 0;
  __syncthreads();
  const int some = min(cut + 1, p.requests);  // entries of `starts` and `taken`

  // ---- what each request is told -----------------------------------------------------------------------
  const int64_t most = int64_t(p.width) * p.block_size;
  for (int i = cta * kPlanThreads + tid; i < p.requests; i += ctas * kPlanThreads) {
    const PlanRequest r = plan_request(p, i);
    const bool served = r.valid && (r.query == 0 || i < cut);
    int64_t len = r.context < 0 ? 0 : (r.context > most ? most : int64_t(r.context));
    if (served) len += r.query;
    p.seq_lens[i] = int32_t(len);
    p.starts[i] = i < some ? starts[i] : all_tokens;
    p.served[i] = served;
  }
  if (cta == 0 && tid == 0) p.starts[p.requests] = all_tokens;

  // ---- pages off the stack ------------------------------------------------------------------------------
  const int64_t first = int64_t(cta) * kPlanThreads + tid, step = int64_t(ctas) * kPlanThreads;
  for (int64_t x0 = first; x0 < all_pages; x0 += kPlanBatch * step) {
    int32_t id[kPlanBatch], context[kPlanBatch];
    int owner[kPlanBatch];
#pragma unroll
    for (int k = 0; k < kPlanBatch; ++k) {
      const int64_t x = x0 + k * step;
      if (x >= all_pages) continue;
      owner[k] = plan_owner(taken, some, int32_t(x));
      context[k] = p.context[owner[k]];
      id[k] = p.free_pages[height - 1 - x];
    }
#pragma unroll
    for (int k = 0; k < kPlanBatch; ++k) {
      const int64_t x = x0 + k * step;
      if (x >= all_pages) continue;
      const uint32_t have = plan_pages(context[k], p.block_size);
      p.table[owner[k] * p.table_stride + have + (x - taken[owner[k]])] = id[k];
    }
  }
  // ---- slots and positions: a page that was taken just now is read off the stack, not from the table -------
  for (int64_t x0 = first; x0 < p.room; x0 += kPlanBatch * step) {
    int64_t slot[kPlanBatch], at[kPlanBatch];
    const uint32_t bs = p.block_size;
#pragma unroll
    for (int k = 0; k < kPlanBatch; ++k) {
      const int64_t x = x0 + k * step;
      slot[k] = at[k] = -1;
      if (x >= all_tokens) continue;
      const int i = plan_owner(starts, some, int32_t(x));
      const uint32_t context = p.context[i], position = context + uint32_t(x - starts[i]);
      const uint32_t page = position / bs, have = plan_pages(context, bs);
      const int32_t id = page < have ? p.table[i * p.table_stride + page]
                                     : p.free_pages[height - 1 - (taken[i] + int64_t(page - have))];
      slot[k] = int64_t(id) * bs + (position - page * bs);
      at[k] = position;
    }
#pragma unroll
    for (int k = 0; k < kPlanBatch; ++k) {
      const int64_t x = x0 + k * step;
      if (x >= p.room) break;
      p.slots[x] = slot[k];
      p.positions[x] = at[k];
    }
  }
  cluster_barrier();  // (of one CTA, unless free_count is count_out)
  if (cta == 0 && tid == 0) *p.count_out = int32_t(height - all_pages);
}

struct ReleaseArgs {
  const uint8_t* finished;
  const int32_t* context;
  const int32_t* table;
  int64_t table_stride;
  int width, requests, block_size;
  int32_t* free_pages;
  int64_t capacity;
  const int32_t* free_count;
  int32_t* count_out;
};

__global__ void __launch_bounds__(kPlanThreads) release_pages_kernel(const ReleaseArgs p) {
  extern __shared__ int32_t plan_smem[];
  int32_t* const starts = plan_smem;  // [requests]
  __shared__ int64_t sums[kPlanThreads / 32][2];
  __shared__ int64_t all_pages;
  const int tid = threadIdx.x;
  const int ctas = gridDim.x, cta = blockIdx.x;
  int64_t height = *p.free_count;
  height = height < 0 ? 0 : (height > p.capacity ? p.capacity : height);
  auto pages_of = [&](int i) -> int64_t {
    const int32_t context = p.context[i];
    if (!p.finished[i] || context <= 0) return 0;
    return min(plan_pages(context, p.block_size), uint32_t(p.width));
  };
  const int each = (p.requests + kPlanThreads - 1) / kPlanThreads;
  const int i0 = min(tid * each, p.requests), i1 = min(i0 + each, p.requests);
  int64_t pages = 0, unused = 0;
  for (int i = i0; i < i1; ++i) pages += pages_of(i);
  const int64_t mine = pages;
  plan_before(pages, unused, sums, tid);
  if (tid == kPlanThreads - 1) all_pages = pages + mine;
  const int64_t space = p.capacity - height;
  for (int i = i0; i < i1; ++i) {
    starts[i] = int32_t(pages < space ? pages : space);
    pages += pages_of(i);
  }
  __syncthreads();
  const int64_t total = all_pages < space ? all_pages : space;
  const int64_t step = int64_t(ctas) * kPlanThreads;
  for (int64_t x0 = int64_t(cta) * kPlanThreads + tid; x0 < total; x0 += kPlanBatch * step) {
    int32_t id[kPlanBatch];
#pragma unroll
    for (int k = 0; k < kPlanBatch; ++k) {
      const int64_t x = x0 + k * step;
      if (x >= total) continue;
      const int i = plan_owner(starts, p.requests, int32_t(x));
      id[k] = p.table[i * p.table_stride + (x - starts[i])];
    }
#pragma unroll
    for (int k = 0; k < kPlanBatch; ++k) {
      const int64_t x = x0 + k * step;
      if (x < total) p.free_pages[height + x] = id[k];
    }
  }
  cluster_barrier();
  if (cta == 0 && tid == 0) *p.count_out = int32_t(height + total);
}

// (64 prompts, 39 000 tokens: 10.1 us by a cluster of eight CTAs, 5.9 by one to 1024; 128 000 pages released: 14.9, 4.6)
constexpr int kPlanCluster = 8, kPlanMaxCtas = 148;
// `work`: pages or tokens
template <typename Args>
static int launch_plan(void (*kernel)(Args), const Args& p, int64_t work, size_t smem, const char* what,
                       cudaStream_t stream) {
  int ctas = int(std::min<int64_t>(std::max<int64_t>(1, (work + kPlanThreads - 1) / kPlanThreads), kPlanMaxCtas));
  const bool in_place = p.count_out == p.free_count;
  if (in_place && ctas > 1) ctas = kPlanCluster;
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(ctas);
  config.blockDim = dim3(kPlanThreads);
  config.dynamicSmemBytes = smem;
  config.stream = stream;
  cudaLaunchAttribute cluster;
  cluster.id = cudaLaunchAttributeClusterDimension;
  cluster.val.clusterDim.x = ctas;
  cluster.val.clusterDim.y = cluster.val.clusterDim.z = 1;
  config.attrs = &cluster;
  config.numAttrs = in_place && ctas > 1 ? 1 : 0;
  const cudaError_t e = cudaLaunchKernelEx(&config, kernel, p);
  if (e != cudaSuccess) return fail(FQ_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
  return check_launch(what);
}

}  // namespace fq

using namespace fq;

static int plan_check(int requests, int width, int64_t table_stride, int block_size, int64_t capacity) {
  FQ_REQUIRE(requests >= 0 && width >= 0 && capacity >= 0 && block_size > 0 && (width == 0 || table_stride >= width),
             FQ_ERR_INVALID_ARGUMENT, "step plan: bad size");
  FQ_REQUIRE(requests <= kPlanMaxRequests, FQ_ERR_UNSUPPORTED, "step plan: at most %d requests (got %d)",
             kPlanMaxRequests, requests);
  FQ_REQUIRE(capacity <= 0x7fffffff && int64_t(width) * block_size <= 0x7fffffff, FQ_ERR_UNSUPPORTED,
             "step plan: more than 2^31 pages, or tokens to a request");
  return FQ_OK;
}

extern "C" int fq_plan_paged_step(const int32_t* context_lens, const int32_t* query_lens, int num_requests,
                                  int32_t* block_table, int64_t block_table_stride, int block_table_width,
                                  int block_size, const int32_t* free_blocks, int64_t free_capacity,
                                  const int32_t* free_count, int64_t max_tokens, int32_t* seq_lens,
                                  int32_t* cu_seqlens_q, int64_t* slot_mapping, int64_t* positions, uint8_t* served,
                                  int32_t* free_count_out, fq_stream_t stream) {
  FQ_RANGE("fq_plan_paged_step");
  if (const int rc = plan_check(num_requests, block_table_width, block_table_stride, block_size, free_capacity)) return rc;
  FQ_REQUIRE(max_tokens >= 0 && max_tokens <= 0x7fffffff, FQ_ERR_INVALID_ARGUMENT, "step plan: max_tokens");
  FQ_REQUIRE(cu_seqlens_q && free_count && free_count_out && (free_capacity == 0 || free_blocks) &&
                 (max_tokens == 0 || (slot_mapping && positions)) &&
                 (num_requests == 0 || (context_lens && query_lens && seq_lens && served &&
                                        (block_table_width == 0 || block_table))),
             FQ_ERR_INVALID_ARGUMENT, "step plan: null pointer");
  PlanArgs p;
  p.context = context_lens; p.query = query_lens;
  p.table = block_table; p.table_stride = block_table_stride; p.width = block_table_width;
  p.requests = num_requests; p.block_size = block_size;
  p.free_pages = free_blocks; p.capacity = free_capacity; p.free_count = free_count;
  p.room = max_tokens;
  p.seq_lens = seq_lens; p.starts = cu_seqlens_q;
  p.slots = slot_mapping; p.positions = positions;
  p.served = served; p.count_out = free_count_out;
  return launch_plan(plan_step_kernel, p, max_tokens, 2 * size_t(num_requests) * sizeof(int32_t), "step plan", stream);
}

extern "C" int fq_release_pages(const uint8_t* finished, const int32_t* context_lens, int num_requests,
                                const int32_t* block_table, int64_t block_table_stride, int block_table_width,
                                int block_size, int32_t* free_blocks, int64_t free_capacity, const int32_t* free_count,
                                int32_t* free_count_out, fq_stream_t stream) {
  FQ_RANGE("fq_release_pages");
  if (const int rc = plan_check(num_requests, block_table_width, block_table_stride, block_size, free_capacity)) return rc;
  FQ_REQUIRE(free_count && free_count_out && (free_capacity == 0 || free_blocks) &&
                 (num_requests == 0 || (finished && context_lens && (block_table_width == 0 || block_table))),
             FQ_ERR_INVALID_ARGUMENT, "release: null pointer");
  ReleaseArgs p;
  p.finished = finished; p.context = context_lens;
  p.table = block_table; p.table_stride = block_table_stride; p.width = block_table_width;
  p.requests = num_requests; p.block_size = block_size;
  p.free_pages = free_blocks; p.capacity = free_capacity; p.free_count = free_count;
  p.count_out = free_count_out;
  return launch_plan(release_pages_kernel, p, std::min(int64_t(num_requests) * block_table_width, free_capacity),
                     size_t(num_requests) * sizeof(int32_t), "release", stream);
}
