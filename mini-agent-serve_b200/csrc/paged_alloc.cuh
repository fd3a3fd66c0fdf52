// paged_alloc.cuh -- page allocation and token maps of a paged KV cache, built on the GPU from request
// lengths (sm_100a).
//
// Allocation, for requests b = 0 .. B-1 with len[b] tokens cached and app[b] new ones:
//   need[b] = ceil((len + app) / page_size) - ceil(len / page_size)
//   the j-th page needed (requests ascending, pages ascending) is free_pages[num_free - 1 - j]
//   block_tables[b, ceil(len / page_size) + i] = the i-th page of b;  len[b] += app[b];
//   num_free -= sum(need)
//   token t of request b: batch_indices = b, positions = len[b] + (t - cum[b]), cum = exclusive sum of app
// Release is its inverse: with R pages past the kept lengths in all, the j-th of them (same order)
// goes to free_pages[num_free + R - 1 - j], so releasing what was just allocated restores the list.
//
// Nothing here is bandwidth: 8 bytes a token and 4 a page. What bounds a call is latency: one launch, one
// round trip for the lengths, one block scan, one round trip for the pages. So there is one launch and no
// scratch memory: every CTA scans all lengths itself (at most kMaxRequests, in shared memory) and then
// fills its share of the outputs, finding a token's request by bisection of the scanned lengths. The
// state (len, num_free) is updated in place, which needs every CTA to have read it first: the CTAs are
// one cluster, with one cluster barrier between the reads and the writes. A step whose outputs one
// CTA can fill alone (alloc_cluster below) launches a single CTA and skips the barrier.
#pragma once

#include "common.cuh"

namespace mas {

constexpr int kAllocThreads = 1024;
constexpr int kMaxRequests = 8192;  // scanned lengths in shared memory: 12 bytes a request
constexpr int kAllocClusterCtas = 8;
constexpr int kAllocSingleOutputs = 4096;  // tokens or pages that one CTA fills alone

struct AllocArgs {
  const int32_t* delta_lens;  // allocate: new tokens a request; release: tokens a request keeps
  int32_t* seq_lens;          // in, out
  int32_t* block_tables;      // [B, max_blocks], row stride table_stride
  int32_t* free_pages;        // [free_capacity], a stack: the last num_free[0] - 1 entry is popped first
  int32_t* num_free;          // in, out
  int32_t* cum_lens;          // [B + 1]         (allocate only, as the rest)
  int32_t* batch_indices;     // [max_tokens]
  int32_t* positions;         // [max_tokens]
  int32_t* last_page_len;     // [B]
  int64_t table_stride;
  int64_t max_tokens;
  int64_t free_capacity;
  int32_t B, max_blocks, page_size;
  int32_t* status;
};

__device__ __forceinline__ int32_t page_count(int32_t len, int32_t page_size) {
  return len / page_size + (len % page_size != 0);
}

// The last index i in [0, n) with cum[i] <= x; cum is ascending and cum[0] <= x.
__device__ __forceinline__ int bisect(const int32_t* cum, int n, int32_t x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (cum[mid] <= x) lo = mid; else hi = mid;
  }
  return lo;
}

__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// Exclusive scan over the block of one 64-bit value a thread; the total through *total.
__device__ __forceinline__ int64_t block_scan(int64_t v, int64_t* scratch, int64_t* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int64_t x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  if (lane == 31) scratch[warp] = x;
  __syncthreads();
  const int nwarps = blockDim.x >> 5;
  int64_t before = 0, all = 0;
  {
    const int64_t w = lane < nwarps ? scratch[lane] : 0;
    int64_t s = w;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t y = __shfl_up_sync(0xffffffffu, s, o);
      if (lane >= o) s += y;
    }
    before = __shfl_sync(0xffffffffu, s - w, warp);
    all = __shfl_sync(0xffffffffu, s, 31);
  }
  __syncthreads();  // scratch may be used again
  *total = all;
  return before + x - v;
}

// RELEASE: delta_lens are the kept lengths. Dynamic shared memory: 3 * (B + 1) int32.
template <bool RELEASE, bool CLUSTER>
__global__ void __launch_bounds__(kAllocThreads) paged_alloc_kernel(const AllocArgs a) {
  extern __shared__ int32_t alloc_smem[];
  __shared__ int64_t scratch[32];
  int32_t* cum_tok = alloc_smem;                // [B + 1]
  int32_t* cum_page = alloc_smem + (a.B + 1);   // [B + 1]
  int32_t* first_page = cum_page + (a.B + 1);   // [B]: allocate: old length; release: pages kept
  pdl_wait();
  const int tid = threadIdx.x;
  const int rank = CLUSTER ? blockIdx.x : 0;  // one cluster is the whole grid
  const int64_t ranks = CLUSTER ? gridDim.x : 1;
  const int per = (a.B + kAllocThreads - 1) / kAllocThreads;
  const int b0 = tid * per, b1 = min(a.B, b0 + per);
  const int64_t capacity = min((int64_t)a.max_blocks * a.page_size, (int64_t)INT32_MAX);

  int64_t tok = 0, pages = 0;
  int bad = 0;
  for (int b = b0; b < b1; ++b) {
    const int32_t len = a.seq_lens[b], d = a.delta_lens[b];
    if (len < 0 || d < 0 || len > capacity || (RELEASE ? d > len : (int64_t)len + d > capacity)) {
      bad = 1;
      continue;
    }
    tok += RELEASE ? 0 : d;
    pages += RELEASE ? page_count(len, a.page_size) - page_count(d, a.page_size)
                     : page_count(len + d, a.page_size) - page_count(len, a.page_size);
  }
  const int32_t num_free = *a.num_free;
  int64_t all_tok = 0, all_pages = 0;
  int64_t tok_before = RELEASE ? 0 : block_scan(tok, scratch, &all_tok);
  int64_t pages_before = block_scan(pages, scratch, &all_pages);
  if (num_free < 0 || num_free > a.free_capacity) bad = 1;
  if (RELEASE ? num_free + all_pages > a.free_capacity : all_pages > num_free || all_tok > a.max_tokens) bad = 1;
  bad = __syncthreads_or(bad);
  if (!bad) {
    for (int b = b0; b < b1; ++b) {
      const int32_t len = a.seq_lens[b], d = a.delta_lens[b];
      cum_tok[b] = (int32_t)tok_before;
      cum_page[b] = (int32_t)pages_before;
      first_page[b] = RELEASE ? page_count(d, a.page_size) : len;
      tok_before += RELEASE ? 0 : d;
      pages_before += RELEASE ? page_count(len, a.page_size) - page_count(d, a.page_size)
                              : page_count(len + d, a.page_size) - page_count(len, a.page_size);
    }
  }
  // Every CTA has read seq_lens and num_free: from here they may be overwritten.
  if (CLUSTER) cluster_barrier(); else __syncthreads();

  const int64_t gid = (int64_t)rank * kAllocThreads + tid, step = ranks * kAllocThreads;
  if (bad) {
    // Nothing is taken or given back; an allocation's maps say that no token has a place.
    if (gid == 0) flag_status(a.status, MAS_STATUS_KV_ALLOC_REFUSED);
    if (!RELEASE) {
      for (int64_t i = gid; i < a.max_tokens; i += step) {
        a.batch_indices[i] = -1;
        a.positions[i] = 0;
      }
      for (int64_t b = gid; b <= a.B; b += step) {
        a.cum_lens[b] = 0;
        if (b < a.B) {
          const int32_t len = a.seq_lens[b];
          a.last_page_len[b] = len > 0 ? (len - 1) % a.page_size + 1 : 0;
        }
      }
    }
    pdl_launch_dependents();
    return;
  }
  for (int64_t i = gid; i < all_pages; i += step) {
    const int b = bisect(cum_page, a.B, (int32_t)i);
    const int32_t within = (int32_t)i - cum_page[b];
    if (RELEASE) {
      a.free_pages[num_free + all_pages - 1 - i] = a.block_tables[b * a.table_stride + first_page[b] + within];
    } else {
      a.block_tables[b * a.table_stride + page_count(first_page[b], a.page_size) + within] =
          a.free_pages[num_free - 1 - i];
    }
  }
  if (!RELEASE) {
    for (int64_t i = gid; i < a.max_tokens; i += step) {
      int32_t batch = -1, pos = 0;  // entries behind the last token name no request
      if (i < all_tok) {
        batch = bisect(cum_tok, a.B, (int32_t)i);
        pos = first_page[batch] + (int32_t)i - cum_tok[batch];
      }
      a.batch_indices[i] = batch;
      a.positions[i] = pos;
    }
  }
  if (rank == 0) {
    for (int b = tid; b < a.B; b += kAllocThreads) {
      const int32_t d = a.delta_lens[b];
      if (RELEASE) {
        a.seq_lens[b] = d;
      } else {
        const int32_t len = first_page[b] + d;
        a.seq_lens[b] = len;
        a.cum_lens[b] = cum_tok[b];
        a.last_page_len[b] = len > 0 ? (len - 1) % a.page_size + 1 : 0;
      }
    }
    if (tid == 0) {
      *a.num_free = RELEASE ? num_free + (int32_t)all_pages : num_free - (int32_t)all_pages;
      if (!RELEASE) a.cum_lens[a.B] = (int32_t)all_tok;
    }
  }
  pdl_launch_dependents();
}

}  // namespace mas
