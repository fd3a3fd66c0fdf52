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
constexpr int kAllocSmallThreads = 256;
constexpr int kMaxRequests = 8192;  // scanned lengths in shared memory: 12 bytes a request
constexpr int kAllocClusterCtas = 8;
// Tokens or pages up to which one CTA fills them alone: allocating and releasing one token for each of 256 requests takes
// 6.6 us with one CTA and 8.2 with a cluster, 33 K tokens of 64 requests 27 and 10.3 (18 and 10.2 with four tokens a
// bisection). Few requests and tokens take 256 threads instead of 1024: 6.6 against 7.7 us.
constexpr int kAllocSingleOutputs = 2048;

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

// Exclusive scans over the block of two 64-bit values a thread, with their totals. One barrier.
struct ScanPair {
  int64_t tok, pages;
};
__device__ __forceinline__ ScanPair block_scan(ScanPair v, ScanPair* scratch, ScanPair* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nwarps = blockDim.x >> 5;
  ScanPair x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t y = __shfl_up_sync(0xffffffffu, x.tok, o), z = __shfl_up_sync(0xffffffffu, x.pages, o);
    if (lane >= o) {
      x.tok += y;
      x.pages += z;
    }
  }
  if (lane == 31) scratch[warp] = x;
  __syncthreads();
  ScanPair s = lane < nwarps ? scratch[lane] : ScanPair{0, 0};
  const ScanPair w = s;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t y = __shfl_up_sync(0xffffffffu, s.tok, o), z = __shfl_up_sync(0xffffffffu, s.pages, o);
    if (lane >= o) {
      s.tok += y;
      s.pages += z;
    }
  }
  *total = {__shfl_sync(0xffffffffu, s.tok, 31), __shfl_sync(0xffffffffu, s.pages, 31)};
  return {__shfl_sync(0xffffffffu, s.tok - w.tok, warp) + x.tok - v.tok,
          __shfl_sync(0xffffffffu, s.pages - w.pages, warp) + x.pages - v.pages};
}

// RELEASE: delta_lens are the kept lengths. Dynamic shared memory: 3 * (B + 1) int32.
template <bool RELEASE, bool CLUSTER>
__global__ void __launch_bounds__(kAllocThreads) paged_alloc_kernel(const AllocArgs a) {
  extern __shared__ int32_t alloc_smem[];
  __shared__ ScanPair scratch[32];
  int32_t* cum_tok = alloc_smem;                // [B + 1]
  int32_t* cum_page = alloc_smem + (a.B + 1);   // [B + 1]
  int32_t* first_page = cum_page + (a.B + 1);   // [B]: allocate: old length; release: pages kept
  pdl_wait();
  const int tid = threadIdx.x;
  const int rank = CLUSTER ? blockIdx.x : 0;  // one cluster is the whole grid
  const int64_t ranks = CLUSTER ? gridDim.x : 1;
  const int threads = blockDim.x;
  const int per = (a.B + threads - 1) / threads;
  const int b0 = tid * per, b1 = min(a.B, b0 + per);
  const int64_t capacity = min((int64_t)a.max_blocks * a.page_size, (int64_t)INT32_MAX);

  const int32_t num_free = *a.num_free;
  ScanPair mine = {0, 0};
  int bad = 0;
  int32_t first_len = 0, first_delta = 0;  // of the thread's first request: all there is up to a thread each
  for (int b = b0; b < b1; ++b) {
    const int32_t len = a.seq_lens[b], d = a.delta_lens[b];
    if (b == b0) {
      first_len = len;
      first_delta = d;
    }
    if (len < 0 || d < 0 || len > capacity || (RELEASE ? d > len : (int64_t)len + d > capacity)) {
      bad = 1;
      continue;
    }
    mine.tok += RELEASE ? 0 : d;
    mine.pages += RELEASE ? page_count(len, a.page_size) - page_count(d, a.page_size)
                     : page_count(len + d, a.page_size) - page_count(len, a.page_size);
  }
  ScanPair all;
  ScanPair before = block_scan(mine, scratch, &all);
  const int64_t all_tok = all.tok, all_pages = all.pages;
  if (num_free < 0 || num_free > a.free_capacity) bad = 1;
  if (RELEASE ? num_free + all_pages > a.free_capacity : all_pages > num_free || all_tok > a.max_tokens) bad = 1;
  bad = __syncthreads_or(bad);
  if (!bad) {
    for (int b = b0; b < b1; ++b) {
      const int32_t len = b == b0 ? first_len : a.seq_lens[b], d = b == b0 ? first_delta : a.delta_lens[b];
      cum_tok[b] = (int32_t)before.tok;
      cum_page[b] = (int32_t)before.pages;
      first_page[b] = RELEASE ? page_count(d, a.page_size) : len;
      before.tok += RELEASE ? 0 : d;
      before.pages += RELEASE ? page_count(len, a.page_size) - page_count(d, a.page_size)
                              : page_count(len + d, a.page_size) - page_count(len, a.page_size);
    }
  }
  // Every CTA has read seq_lens and num_free: from here they may be overwritten.
  if (CLUSTER) cluster_barrier(); else __syncthreads();

  const int64_t gid = (int64_t)rank * threads + tid, step = ranks * threads;
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
    // Where a thread has several tokens they are four in a row: one bisection, then at most a step on each.
    const int run = a.max_tokens > 2 * step ? 4 : 1;
    const bool vec = run == 4 && ((reinterpret_cast<uintptr_t>(a.batch_indices) | reinterpret_cast<uintptr_t>(a.positions)) & 15) == 0;
    for (int64_t i = gid * run; i < a.max_tokens; i += step * run) {
      int32_t batch[4] = {-1, -1, -1, -1}, pos[4] = {0, 0, 0, 0};  // entries behind the last token name no request
      if (i < all_tok) {
        int b = bisect(cum_tok, a.B, (int32_t)i);
        int32_t shift = first_page[b] - cum_tok[b], next = b + 1 < a.B ? cum_tok[b + 1] : INT32_MAX;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (j >= run || i + j >= all_tok) break;
          while (i + j >= next) {
            ++b;
            shift = first_page[b] - cum_tok[b];
            next = b + 1 < a.B ? cum_tok[b + 1] : INT32_MAX;
          }
          batch[j] = b;
          pos[j] = (int32_t)(i + j) + shift;
        }
      }
      if (vec && i + 4 <= a.max_tokens) {
        *reinterpret_cast<int4*>(a.batch_indices + i) = make_int4(batch[0], batch[1], batch[2], batch[3]);
        *reinterpret_cast<int4*>(a.positions + i) = make_int4(pos[0], pos[1], pos[2], pos[3]);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (j < run && i + j < a.max_tokens) {
            a.batch_indices[i + j] = batch[j];
            a.positions[i + j] = pos[j];
          }
      }
    }
  }
  if (rank == 0) {
    for (int b = tid; b < a.B; b += threads) {
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
