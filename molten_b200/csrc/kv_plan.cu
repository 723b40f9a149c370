// Bookkeeping of the paged cache on the device: which pages a step's tokens
// go to (mc_kv_plan) and giving a finished request's pages back
// (mc_kv_release). No host round trip: a decode step can be captured once and
// replayed while requests grow at different paces.
//
// With bs tokens a page, a request holding L tokens and adding n needs
// ceil((L+n)/bs) - ceil(L/bs) fresh pages. The free list is a stack:
// requests take pages from its top in request order, so request r's first
// fresh page is entry n_free - 1 - (the fresh pages of the requests before
// it). That is a prefix sum, and so is each request's first token row; one
// CTA does both (a request a thread, chunks of the block's width, 64-bit
// running sums). A request is admitted whole or not at all.
//
// The work is a few hundred bytes to a few hundred KB, bound by latency: one
// CTA (of as many threads as there are requests or rows to map, up to the
// most), with what the maps need in shared memory; above kMapsInPlan rows the
// maps (20 bytes a token) go to a second, chained launch. The first launch writes the map
// entries of each request's first token; their position and kv_len tell the
// second launch the request's old length and whether it was admitted, so
// `seq_lens` may be `lens` itself.
#include "kv_common.cuh"

namespace {

constexpr int kThreads = 1024;  // most threads; requests of a chunk
constexpr int kWarpsP = kThreads / 32;

struct PlanParams {
  const int32_t* lens;
  const int32_t* new_lens;  // null: one token each
  int n_req, block_size;
  int32_t* table;
  int width;
  const int32_t* free_list;
  const int32_t* n_free;
  int free_len;
  int32_t* seq_lens;
  int32_t* n_free_out;
  int32_t* row_start;
  int32_t* positions;
  int32_t* token_req;
  int32_t* kv_lens;
  unsigned long long* slots;
  int max_tokens;
  uint32_t* status;
};

// Inclusive sum over the block; `total` is the block's sum.
__device__ __forceinline__ long long block_scan(long long v, long long* warp_sums,
                                                long long& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const long long o = __shfl_up_sync(0xffffffffu, v, d);
    if (lane >= d) v += o;
  }
  if (lane == 31) warp_sums[warp] = v;
  __syncthreads();
  if (warp == 0) {
    const int warps = blockDim.x >> 5;
    long long w = lane < warps ? warp_sums[lane] : 0;
#pragma unroll
    for (int d = 1; d < kWarpsP; d <<= 1) {
      const long long o = __shfl_up_sync(0xffffffffu, w, d);
      if (lane >= d) w += o;
    }
    if (lane < warps) warp_sums[lane] = w;
  }
  __syncthreads();
  if (warp > 0) v += warp_sums[warp - 1];
  total = warp_sums[(blockDim.x >> 5) - 1];
  __syncthreads();
  return v;
}

// First index in a[0..n) whose value is above x (a ascending).
template <typename T>
__device__ __forceinline__ int upper_bound(const T* a, int n, T x) {
  int lo = 0, hi = n;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (a[mid] <= x) lo = mid + 1;
    else hi = mid;
  }
  return lo;
}

// Shares out the pages of a chunk's requests: fn(i, j, n) for page j of the n
// pages of request i, this thread's being request threadIdx.x with n pages.
// One or two are done by the request's own thread, up to kWarpPages by one warp
// together, more by the whole block. Every thread of the block calls it. (By
// warps only up to 64, or up to 16384: a step of 256 requests with a release,
// lists of up to 512 pages, 17.1 us, 8.6 as it is, 8.6; 64 requests of up to
// 8192 pages 12.0, 12.3, 22.6; 4 prompts of up to 4096 pages 8.4, 8.7, 11.0.)
constexpr int kWarpPages = 1024;
template <typename F>
__device__ __forceinline__ void share_pages(int n, int* lists, int* count_s, F&& fn) {
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5, threads = blockDim.x;
  // who they are and how many pages: for a warp from the front, for the block from the back
  int* who = lists;
  int* pages_of = lists + threads;
  if (t < 2) count_s[t] = 0;
  __syncthreads();
  int at = -1;
  if (n > kWarpPages) at = threads - 1 - atomicAdd(count_s + 1, 1);
  else if (n > 2) at = atomicAdd(count_s, 1);
  if (at >= 0) {
    who[at] = t;
    pages_of[at] = n;
  }
  if (n == 1 || n == 2) {
    fn(t, 0, n);
    if (n == 2) fn(t, 1, n);
  }
  __syncthreads();
  const int n_warp = count_s[0], n_block = count_s[1];
  for (int k = warp; k < n_warp; k += threads >> 5) {
    const int i = who[k], pages = pages_of[k];
#pragma unroll 4
    for (int j = lane; j < pages; j += 32) fn(i, j, pages);
  }
  for (int k = 0; k < n_block; ++k) {
    const int i = who[threads - 1 - k], pages = pages_of[threads - 1 - k];
#pragma unroll 4
    for (int j = t; j < pages; j += threads) fn(i, j, pages);
  }
  __syncthreads();
}

// The maps of token row t (row_start and the first rows' entries written).
__device__ __forceinline__ void map_token(const PlanParams& P, int t) {
  const int total = P.row_start[P.n_req];
  if (t >= total) {
    P.positions[t] = 0;
    P.token_req[t] = -1;
    P.kv_lens[t] = 0;
    P.slots[t] = MC_KV_SLOT_NONE;
    return;
  }
  const int r = upper_bound(P.row_start, P.n_req + 1, t) - 1;
  const int first = P.row_start[r];
  const int pos = (int)min((long long)P.positions[first] + (t - first), (long long)INT32_MAX);
  const bool ok = P.kv_lens[first] != 0;
  unsigned long long slot = MC_KV_SLOT_NONE;
  if (ok) {
    const int page = P.table[(size_t)r * P.width + pos / P.block_size];
    if (page >= 0)  // a page that is not the cache's is left to the calls that use the slot
      slot = (unsigned long long)page * P.block_size + pos % P.block_size;
  }
  if (t != first) {
    P.positions[t] = pos;
    P.kv_lens[t] = ok ? pos + 1 : 0;
  }
  P.token_req[t] = r;
  P.slots[t] = slot;
}

// MAPS: at most kThreads requests and kMapsInPlan rows, whose maps are written too.
template <bool MAPS>
__global__ void __launch_bounds__(kThreads) plan_kernel(const PlanParams P) {
  __shared__ long long warp_sums[kWarpsP];
  __shared__ long long taken_s[kThreads];  // inclusive fresh-page sums of the chunk
  __shared__ int have_s[kThreads];         // pages held; -1: not admitted
  __shared__ int start_s[MAPS ? kThreads + 1 : 1], len_s[MAPS ? kThreads : 1];
  __shared__ int lists_s[2 * kThreads], count_s[2];
  __shared__ unsigned long long used_s;
  __shared__ uint32_t status_s;
  const int t = threadIdx.x, threads = blockDim.x;
  if (t == 0) {
    used_s = 0;
    status_s = 0;
  }
  mc_pdl_launch_dependents();
  mc_pdl_wait();
  const long long bs = P.block_size;
  const int nf = min(max(*P.n_free, 0), P.free_len);
  long long rows = 0, pages = 0;  // sums of the chunks before
  for (int r0 = 0; r0 < P.n_req; r0 += threads) {
    const int r = r0 + t;
    const bool in = r < P.n_req;
    long long len = in ? P.lens[r] : 0, add = in ? (P.new_lens ? P.new_lens[r] : 1) : 0;
    uint32_t st = 0;
    if (len < 0 || add < 0) {
      st = MC_KV_BAD_LENGTH;
      add = 0;
      len = len < 0 ? 0 : len;
    }
    long long total;
    const long long row_end = rows + block_scan(add, warp_sums, total);
    rows += total;
    const long long have = (len + bs - 1) / bs, want = (len + add + bs - 1) / bs;
    bool ok = st == 0;
    if (ok && (want > P.width || len + add > INT32_MAX)) {
      st = MC_KV_TABLE_FULL;
      ok = false;
    }
    if (ok && row_end > P.max_tokens) {
      st = MC_KV_ROWS_FULL;
      ok = false;
    }
    const long long need = ok ? want - have : 0;
    const long long taken = block_scan(need, warp_sums, total);
    if (ok && need > 0 && pages + taken > nf) {
      st = MC_KV_NO_PAGES;
      ok = false;
    }
    taken_s[t] = taken;
    have_s[t] = ok ? (int)have : -1;
    const int end32 = (int)min(row_end, (long long)INT32_MAX);
    if (MAPS) {
      start_s[t + 1] = end32;
      len_s[t] = (int)len;
    }
    if (in) {
      if (ok && need > 0) atomicMax(&used_s, (unsigned long long)(pages + taken));
      if (st) atomicOr(&status_s, st);
      const long long first = row_end - add;
      if (r == 0) P.row_start[0] = 0;
      P.row_start[r + 1] = end32;
      P.seq_lens[r] = (int)(ok ? len + add : len);
      if (!MAPS && add > 0 && first < P.max_tokens) {
        P.positions[first] = (int)len;
        P.kv_lens[first] = ok ? (int)len + 1 : 0;
      }
    }
    __syncthreads();
    share_pages(ok ? (int)need : 0, lists_s, count_s, [&](int i, int j, int n) {
      const long long e = pages + taken_s[i] - n + j;
      P.table[(size_t)(r0 + i) * P.width + have_s[i] + j] = __ldg(P.free_list + (nf - 1 - e));
    });
    pages += total;
    __syncthreads();
  }
  if (t == 0) {
    *P.n_free_out = nf - (int)used_s;
    if (P.status && status_s) atomicOr(P.status, status_s);
  }
  if (!MAPS) return;
  // the table entries written above are seen behind the barrier
  for (int i = t; i < P.max_tokens; i += threads) {
    int pos = 0, req = -1, kv_len = 0;
    unsigned long long slot = MC_KV_SLOT_NONE;
    if (i < rows) {
      req = upper_bound(start_s + 1, P.n_req, i);
      const long long at = (long long)len_s[req] + i - (req ? start_s[req] : 0);
      pos = (int)min(at, (long long)INT32_MAX);
      if (have_s[req] >= 0) {
        kv_len = pos + 1;
        const int page = P.table[(size_t)req * P.width + pos / P.block_size];
        if (page >= 0) slot = (unsigned long long)page * P.block_size + pos % P.block_size;
      }
    }
    P.positions[i] = pos;
    P.token_req[i] = req;
    P.kv_lens[i] = kv_len;
    P.slots[i] = slot;
  }
}

__global__ void __launch_bounds__(256) map_kernel(const PlanParams P) {
  mc_pdl_launch_dependents();
  mc_pdl_wait();
  const int t = blockIdx.x * 256 + threadIdx.x;
  if (t < P.max_tokens) map_token(P, t);
}

struct ReleaseParams {
  const uint32_t* done;
  const int32_t* lens;
  int n_req, block_size;
  const int32_t* table;
  int width;
  int32_t* free_list;
  const int32_t* n_free;
  int free_len;
  int32_t* lens_out;
  int32_t* n_free_out;
  uint32_t* status;
};

__global__ void __launch_bounds__(kThreads) release_kernel(const ReleaseParams P) {
  mc_pdl_launch_dependents();
  mc_pdl_wait();
  __shared__ long long warp_sums[kWarpsP];
  __shared__ long long given_s[kThreads];
  __shared__ int lists_s[2 * kThreads], count_s[2];
  const int t = threadIdx.x;
  const int threads = blockDim.x;
  const long long nf = min(max(*P.n_free, 0), P.free_len);
  long long pages = 0;
  for (int r0 = 0; r0 < P.n_req; r0 += threads) {
    const int r = r0 + t;
    long long held = 0;
    if (r < P.n_req) {
      const int len = P.lens[r];
      const bool done = P.done[r] != 0;
      if (done && len > 0)
        held = min(((long long)len + P.block_size - 1) / P.block_size, (long long)P.width);
      P.lens_out[r] = done ? 0 : len;
    }
    long long total;
    given_s[t] = block_scan(held, warp_sums, total);
    __syncthreads();
    share_pages((int)held, lists_s, count_s, [&](int i, int j, int n) {
      const long long at = nf + pages + given_s[i] - n + j;
      if (at < P.free_len) P.free_list[at] = __ldg(P.table + (size_t)(r0 + i) * P.width + j);
    });
    pages += total;
    __syncthreads();
  }
  if (t == 0) {
    const long long now = nf + pages;
    *P.n_free_out = (int)min(now, (long long)P.free_len);
    if (now > P.free_len && P.status) atomicOr(P.status, MC_KV_LIST_FULL);
  }
}

// Above this many token rows the maps go to a launch of their own: 16 requests
// with 512 rows take 4.1 us in one launch and 6.0 in two, with 2048 6.5 and 6.9,
// with 4096 7.5 and 7.0, with 16384 13.4 and 7.2.
constexpr int kMapsInPlan = 2048;

// A thread for each request and row, whole warps.
int plan_threads(int n_req, int rows) {
  const int n = n_req > rows ? n_req : rows;
  return n >= kThreads ? kThreads : (n + 31) / 32 * 32;
}

}  // namespace

extern "C" int mc_kv_plan(mc_ctx* ctx, const int32_t* lens, const int32_t* new_lens, int n_req,
                          int block_size, int32_t* block_table, int table_width,
                          const int32_t* free_list, const int32_t* n_free, int free_len,
                          int32_t* seq_lens, int32_t* n_free_out, int32_t* row_start,
                          int32_t* positions, int32_t* token_req, int32_t* kv_lens,
                          uint64_t* slots, int max_tokens, uint32_t* status) {
  MC_REQUIRE(n_req >= 1, "kv_plan: n_req %d", n_req);
  MC_REQUIRE(block_size >= 1 && table_width >= 1 && free_len >= 1,
             "kv_plan: block size %d, table width %d, free list of %d", block_size, table_width,
             free_len);
  MC_REQUIRE(max_tokens >= 1, "kv_plan: max_tokens %d", max_tokens);
  MC_REQUIRE(lens && block_table && free_list && n_free && seq_lens && n_free_out && row_start &&
                 positions && token_req && kv_lens && slots,
             "kv_plan: null pointer");
  MC_REQUIRE(mc_aligned(slots, 8), "kv_plan: slots must be 8-byte aligned");
  MC_REQUIRE(new_lens != seq_lens, "kv_plan: seq_lens must not be new_lens");
  MC_REQUIRE(ctx, "kv_plan: null context");
  McDeviceGuard dev(ctx->device);
  MC_CUDA(dev.error());
  const PlanParams P{lens, new_lens, n_req, block_size, block_table, table_width, free_list,
                     n_free, free_len, seq_lens, n_free_out, row_start, positions, token_req,
                     kv_lens, reinterpret_cast<unsigned long long*>(slots), max_tokens, status};
  if (max_tokens <= kMapsInPlan && n_req <= kThreads) {
    MC_CUDA(mc_launch_pdl(plan_kernel<true>, dim3(1), dim3(plan_threads(n_req, max_tokens)), 0,
                          ctx->stream, P));
    return mc_after_launch("plan_kernel");
  }
  MC_CUDA(mc_launch_pdl(plan_kernel<false>, dim3(1), dim3(kThreads), 0, ctx->stream, P));
  MC_CUDA(mc_launch_pdl(map_kernel, dim3((unsigned)(((size_t)max_tokens + 255) / 256)), dim3(256),
                        0, ctx->stream, P));
  return mc_after_launch("map_kernel");
}

extern "C" int mc_kv_release(mc_ctx* ctx, const uint32_t* done, const int32_t* lens, int n_req,
                             int block_size, const int32_t* block_table, int table_width,
                             int32_t* free_list, const int32_t* n_free, int free_len,
                             int32_t* lens_out, int32_t* n_free_out, uint32_t* status) {
  MC_REQUIRE(n_req >= 1, "kv_release: n_req %d", n_req);
  MC_REQUIRE(block_size >= 1 && table_width >= 1 && free_len >= 1,
             "kv_release: block size %d, table width %d, free list of %d", block_size, table_width,
             free_len);
  MC_REQUIRE(done && lens && block_table && free_list && n_free && lens_out && n_free_out,
             "kv_release: null pointer");
  MC_REQUIRE(ctx, "kv_release: null context");
  McDeviceGuard dev(ctx->device);
  MC_CUDA(dev.error());
  const ReleaseParams P{done, lens, n_req, block_size, block_table, table_width, free_list,
                        n_free, free_len, lens_out, n_free_out, status};
  MC_CUDA(mc_launch_pdl(release_kernel, dim3(1), dim3(kThreads), 0, ctx->stream, P));
  return mc_after_launch("release_kernel");
}
