// attn_int4.cuh -- attention of ragged query rows over the 4-bit paged KV cache (sm_100a).
//
// With k_t = ck_t sk_t + mk_t and v_t = cv_t sv_t + mv_t (kv_int4.cuh), a query row q sees
//   S_t = scale * (sk_t * sum_d q_d ck_td + mk_t * sum_d q_d)            (t up to the row's causal limit)
//   o_d = (sum_t p_t sv_t (cv_td - 8) + sum_t p_t (mv_t + 8 sv_t)) / sum_t p_t,   p_t = exp(S_t - max S)
// so the matrix products run on the bare codes, exact in 16 bits, and the pairs enter per token in fp32:
// no key or value is ever rounded. p_t sv_t is rounded to bf16 for the second product (two bf16 terms, high and
// low, when the queries are fp16, whose 11 bits one bf16 term would not serve); bf16 and not fp16
// because sv_t may be anything. Maxima, sums and products are accumulated in fp32. The values' codes are centred
// (c - 8) so that long sums do not grow one-sidedly and cancel against the minimum's part.
//
// Work split. The rows of a request that share a kv head (tokens x group, token-major) are cut into tiles of
// 16, the tile's keys into units of 128 tokens; all units of a launch, requests outermost, form one line that the
// CTAs cut into equal shares, whatever the lengths are (they are only known on the device). A share that
// covers a tile's keys writes the output; the others leave (sum, maximum, unnormalised o) in the
// workspace, and a second kernel joins them in a fixed order, so results do not change from run to run.
//
// A CTA is 4 warps that share the tile's queries; each takes every fourth run of 32 tokens, with a ring of
// cp.async stages of its own, an online softmax of its own, and no barrier until the tile ends. A lane's
// operands of mma.m16n8k16 come straight from the staged bytes: the D axis of the first product and the columns of
// the second are permuted so that a lane's codes are 16 (8) consecutive bytes of a row.
#pragma once

#include <type_traits>

#include "common.cuh"
#include "kv_int4.cuh"

namespace mas {

constexpr int kAttnThreads = 128;
constexpr int kAttnWarps = kAttnThreads / 32;
constexpr int kAttnStages = 3;
constexpr int kAttnRows = 16;
constexpr int kAttnRun = 32;                       // tokens of one stage of one warp
constexpr int kAttnUnit = kAttnRun * kAttnWarps;   // tokens of a unit of work
constexpr int kAttnCtasPerSm = 4;

struct AttnInt4Args {
  const void* q;
  void* out;
  float* lse;  // nullable
  KVInt4Args kv;
  const int32_t* block_tables;
  const int32_t* seq_lens;
  const int32_t* cum_q;  // nullable: one query a request
  int64_t T;
  int64_t table_stride;
  int64_t qsn, qsh, osn, osh;  // elements
  float* part;                 // [grid][2][16 * D + 32]
  int32_t* desc;               // [grid][kAttnDescInts]
  float scale_log2;            // softmax scale * log2(e)
  int32_t B, max_blocks, group;
  int32_t page_shift;          // log2(page_size), or -1
  int32_t causal;
  int32_t* status;
};

// What the joining kernel needs of a tile that was split: written by the CTA whose share starts the tile.
// {number of parts (0: nothing to join), request, the tile's first row within it, kv head}
constexpr int kAttnDescInts = 4;

__host__ __device__ constexpr int attn_part_floats(int D) { return kAttnRows * D + 2 * kAttnRows; }

template <int D>
struct AttnInt4Shape {
  static constexpr int kRowBytes = D / 2;
  static constexpr int kKeys = 0;
  static constexpr int kValues = kAttnRun * kRowBytes;
  static constexpr int kPairs = 2 * kAttnRun * kRowBytes;
  static constexpr int kStage = kPairs + kAttnRun * 8;
  static constexpr int kWarpRing = kAttnStages * kStage;
  static constexpr int kQFrag = D / 16 * 32 * 16;
  static constexpr int kMerge = kAttnWarps * (D / 2) * 32 * 4;  // the warps' o; their statistics follow
  static constexpr int kRing = kAttnWarps * kWarpRing;
  static constexpr int kStats = kAttnWarps * kAttnRows * 2 * 4;
  static constexpr int kSmem = kQFrag + (kRing > kMerge ? kRing : kMerge) + kStats;
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool valid) {
  const int bytes = valid ? 16 : 0;  // the rest of the 16 bytes becomes zero
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async8(uint32_t dst, const void* src, bool valid) {
  const int bytes = valid ? 8 : 0;
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ uint4 lds128(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
  return v;
}
__device__ __forceinline__ uint2 lds64(uint32_t a) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a));
  return v;
}
__device__ __forceinline__ uint32_t lds32(uint32_t a) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(a));
  return v;
}

__device__ __forceinline__ void mma_bf16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                         uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_fp16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                         uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// (w & mask) | magic in one instruction.
__device__ __forceinline__ uint32_t and_or(uint32_t w, uint32_t mask, uint32_t magic) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(w), "r"(mask), "r"(magic));
  return r;
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// The key codes of a word as 16-bit pairs (e0, e4), (e1, e5), (e2, e6), (e3, e7). bf16: 128 + c (the bias
// leaves with the sum of q, in the accumulator's start value); fp16: c - 8.
template <typename T>
struct KeyCodes;
template <>
struct KeyCodes<__nv_bfloat16> {
  static constexpr float kStart = -128.0f;  // accumulators start at this times sum q
  static constexpr float kCentre = 0.0f;    // a product is sum q (c - kCentre)
  static __device__ __forceinline__ void unpack(uint32_t w, uint32_t (&p)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) p[i] = and_or(w >> (4 * i), 0x000f000fu, 0x43004300u);
  }
  static __device__ __forceinline__ void mma(float (&c)[4], const uint4& a, uint32_t b0, uint32_t b1) {
    mma_bf16(c, a.x, a.y, a.z, a.w, b0, b1);
  }
};
template <>
struct KeyCodes<__half> {
  static constexpr float kStart = 0.0f;
  static constexpr float kCentre = 8.0f;
  static __device__ __forceinline__ void unpack(uint32_t w, uint32_t (&p)[4]) {
    const __half2 off = __floats2half2_rn(1032.0f, 1032.0f), sixteenth = __floats2half2_rn(0.0625f, 0.0625f);
    const __half2 off16 = __floats2half2_rn(-72.0f, -72.0f);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      uint32_t lo = and_or(w >> (8 * i), 0x000f000fu, 0x64006400u);  // 1024 + c
      uint32_t hi = and_or(w >> (8 * i), 0x00f000f0u, 0x64006400u);  // 1024 + 16 c
      __half2 x = __hsub2(*reinterpret_cast<__half2*>(&lo), off);
      __half2 y = __hfma2(*reinterpret_cast<__half2*>(&hi), sixteenth, off16);
      p[2 * i] = *reinterpret_cast<uint32_t*>(&x);
      p[2 * i + 1] = *reinterpret_cast<uint32_t*>(&y);
    }
  }
  static __device__ __forceinline__ void mma(float (&c)[4], const uint4& a, uint32_t b0, uint32_t b1) {
    mma_fp16(c, a.x, a.y, a.z, a.w, b0, b1);
  }
};

// Code pair i of a word whose halves hold two tokens' codes, as bf16 c - 8 (exact).
__device__ __forceinline__ uint32_t value_codes(uint32_t x, int i) {
  uint32_t u = and_or(x >> (4 * i), 0x000f000fu, 0x43004300u);  // 128 + c
  const __nv_bfloat162 off = __floats2bfloat162_rn(136.0f, 136.0f);
  __nv_bfloat162 y = __hsub2(*reinterpret_cast<__nv_bfloat162*>(&u), off);
  return *reinterpret_cast<uint32_t*>(&y);
}

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  return Elem<__nv_bfloat16>::from_f2(lo, hi);
}

// Where a staged value row's 16-byte chunk lies: rows are reordered (and at D = 128 chunks exchanged) so that the
// four rows 2t (or 2t + 1) that a warp reads at once fall into different banks.
template <int D>
__device__ __forceinline__ uint32_t value_offset(int row, int byte) {
  if (D == 128) {
    const int phys = (row & ~3) | ((row & 1) << 1) | ((row >> 1) & 1);
    return phys * 64 + (byte ^ (((row >> 2) & 1) << 5));
  }
  const int phys = (row & ~7) | ((row & 1) << 2) | ((row >> 1) & 3);
  return phys * 32 + byte;
}

// A request's extent, with every length that does not fit its buffers cut to them.
struct AttnRequest {
  int32_t q0, qlen;  // first query row, queries
  int32_t n;         // tokens in the cache
  int32_t tiles, units;
  __device__ __forceinline__ int64_t work(int heads) const { return (int64_t)tiles * heads * units; }
};

__device__ __forceinline__ AttnRequest attn_request(const AttnInt4Args& a, int b, int32_t* status) {
  AttnRequest r;
  int64_t q0 = b, q1 = b + 1;
  if (a.cum_q != nullptr) {
    q0 = a.cum_q[b];
    q1 = a.cum_q[b + 1];
  }
  const int64_t capacity = min((int64_t)a.max_blocks * a.kv.page_size, (int64_t)INT32_MAX - kAttnUnit);
  int64_t n = a.seq_lens[b];
  if (q0 < 0 || q1 < q0 || q1 > a.T || n < 0 || n > capacity) {
    flag_status(status, MAS_STATUS_KV_SLOT_OUT_OF_RANGE);
    q0 = min(max(q0, (int64_t)0), a.T);
    q1 = min(max(q1, q0), a.T);
    n = min(max(n, (int64_t)0), capacity);
  }
  r.q0 = (int32_t)q0;
  r.qlen = (int32_t)(q1 - q0);
  r.n = (int32_t)n;
  r.tiles = (int32_t)(((int64_t)r.qlen * a.group + kAttnRows - 1) / kAttnRows);
  r.units = max(1, (r.n + kAttnUnit - 1) / kAttnUnit);
  return r;
}

template <typename T, int D>
__global__ void __launch_bounds__(kAttnThreads, kAttnCtasPerSm) attn_int4_kernel(const AttnInt4Args a) {
  using Sh = AttnInt4Shape<D>;
  using Keys = KeyCodes<T>;
  constexpr int kNt = D / 8;        // column tiles of the second product
  constexpr int kWords = D / 32;    // key words a lane and token
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ int64_t s_scan[kAttnWarps + 2];
  __shared__ int32_t s_b;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, t = lane & 3;
  uint8_t* ring = smem + Sh::kQFrag;
  const uint32_t qfrag_u = smem_u32(smem);
  const uint32_t ring_u = smem_u32(ring) + warp * Sh::kWarpRing;
  float* merge = reinterpret_cast<float*>(ring);
  float* stats = reinterpret_cast<float*>(smem + Sh::kSmem - Sh::kStats);  // [warp][row][max, sum]
  int32_t* desc = a.desc + (int64_t)blockIdx.x * kAttnDescInts;
  pdl_wait();

  // This CTA's share of the line of units: total by a block sum, the request it starts in by the scan.
  const int heads = a.kv.heads;
  const int per = (a.B + kAttnThreads - 1) / kAttnThreads;
  const int rb0 = min(a.B, tid * per), rb1 = min(a.B, rb0 + per);
  int64_t mine = 0;
  for (int b = rb0; b < rb1; ++b) mine += attn_request(a, b, blockIdx.x == 0 ? a.status : nullptr).work(heads);
  int64_t incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t y = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += y;
  }
  if (lane == 31) s_scan[warp] = incl;
  __syncthreads();
  int64_t total = 0, before = incl - mine;
#pragma unroll
  for (int w = 0; w < kAttnWarps; ++w) {
    if (w < warp) before += s_scan[w];
    total += s_scan[w];
  }
  const int64_t share = max((total + gridDim.x - 1) / gridDim.x, (int64_t)1);
  int64_t at = (int64_t)blockIdx.x * share;
  const int64_t end = min(at + share, total);
  if (at >= end) {
    if (tid == 0 && a.desc != nullptr) desc[0] = 0;
    pdl_launch_dependents();
    return;
  }
  if (at >= before && at < before + mine) {
    int64_t rem = at - before;
    int b = rb0;
    for (; b < rb1; ++b) {
      const int64_t w = attn_request(a, b, nullptr).work(heads);
      if (rem < w) break;
      rem -= w;
    }
    s_b = b;
    s_scan[kAttnWarps] = rem;
  }
  __syncthreads();
  int b = s_b;
  AttnRequest rq = attn_request(a, b, nullptr);
  int unit, head, tile;
  {
    int64_t rem = s_scan[kAttnWarps];
    unit = (int)(rem % rq.units);
    rem /= rq.units;
    head = (int)(rem % heads);
    tile = (int)(rem / heads);
  }
  int desc_parts = 0, desc_request = 0, desc_row = 0, desc_head = 0;

  while (at < end) {
    const int seg_units = (int)min((int64_t)(rq.units - unit), end - at);
    const int rows_here = min(kAttnRows, rq.qlen * a.group - tile * kAttnRows);
    const int row0 = tile * kAttnRows;
    // Keys visible to a row: those before its limit. Rows past the tile's last take the last one's limit.
    const int last_tok = (row0 + rows_here - 1) / a.group;
    const int tile_end = a.causal ? min(rq.n, max(0, rq.n - rq.qlen + last_tok + 1)) : rq.n;
    const int t0 = unit * kAttnUnit;
    const int t1 = min((unit + seg_units) * kAttnUnit, tile_end);
    int lim0 = tile_end, lim1 = tile_end, lim_first = tile_end;
    if (a.causal) {
      lim_first = max(0, rq.n - rq.qlen + row0 / a.group + 1);
      if (g < rows_here) lim0 = max(0, rq.n - rq.qlen + (row0 + g) / a.group + 1);
      if (g + 8 < rows_here) lim1 = max(0, rq.n - rq.qlen + (row0 + g + 8) / a.group + 1);
    }

    // Queries into shared memory in the order the first product takes them: k step 2i of lane (g, t) holds
    // elements 0, 4 and 1, 5 of 32-bit code word i of the lane's stretch of the row, step 2i + 1 the rest.
    for (int e = tid; e < D / 16 * 32; e += kAttnThreads) {
      const int step = e >> 5, l = e & 31;
      const int d = (D / 4) * (l & 3) + 8 * (step >> 1) + 2 * (step & 1);
      uint32_t v[4];
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int r = row0 + (l >> 2) + 8 * half;
        const bool here = (l >> 2) + 8 * half < rows_here;
        const int tok = r / a.group, sub = r - tok * a.group;
        const uint16_t* src = static_cast<const uint16_t*>(a.q) + (int64_t)(rq.q0 + tok) * a.qsn +
                              ((int64_t)head * a.group + sub) * a.qsh + d;
        v[half] = here ? src[0] | ((uint32_t)src[4] << 16) : 0u;
        v[2 + half] = here ? src[1] | ((uint32_t)src[5] << 16) : 0u;
      }
      *reinterpret_cast<uint4*>(smem + e * 16) = make_uint4(v[0], v[1], v[2], v[3]);
    }

    // The warp's runs: t0 + 32 (warp + 4 i).
    const int runs_all = t1 > t0 ? (t1 - t0 + kAttnRun - 1) / kAttnRun : 0;
    const int runs = runs_all > warp ? (runs_all - warp + kAttnWarps - 1) / kAttnWarps : 0;
    const int32_t* table = a.block_tables + (int64_t)b * a.table_stride;
    auto load_page = [&](int i) {
      const int tok = t0 + kAttnRun * (warp + kAttnWarps * i) + lane;
      if (i >= runs || tok >= t1) return -1;
      const int block = a.page_shift >= 0 ? tok >> a.page_shift : tok / (int)a.kv.page_size;
      const int page = table[block];  // block < max_blocks: tok < n <= capacity
      if (page < 0 || page >= a.kv.num_pages) {
        flag_status(a.status, MAS_STATUS_KV_SLOT_OUT_OF_RANGE);
        return -1;  // its tokens read as zeros
      }
      return page;
    };
    auto issue = [&](int i, int page) {
      if (i < runs) {
        const int tok = t0 + kAttnRun * (warp + kAttnWarps * i) + lane;
        const int entry = a.page_shift >= 0 ? tok & ((1 << a.page_shift) - 1) : tok % (int)a.kv.page_size;
        const uint32_t stage = ring_u + (i % kAttnStages) * Sh::kStage;
        int64_t off = -1;
        if (page >= 0)
          off = page * a.kv.stride_page + entry * a.kv.stride_entry + head * a.kv.stride_head;
        constexpr int kChunks = Sh::kRowBytes / 16;
        constexpr int kRowsAtOnce = 32 / kChunks;
#pragma unroll
        for (int it = 0; it < kAttnRun / kRowsAtOnce; ++it) {
          const int row = it * kRowsAtOnce + lane / kChunks, byte = lane % kChunks * 16;
          const int64_t o = __shfl_sync(0xffffffffu, off, row);
          const bool ok = o >= 0;
          const int64_t src = ok ? o + byte : 0;
          cp_async16(stage + Sh::kKeys + row * Sh::kRowBytes + byte, a.kv.k_codes + src, ok);
          cp_async16(stage + Sh::kValues + value_offset<D>(row, byte), a.kv.v_codes + src, ok);
        }
        const int64_t pair = page >= 0 ? page * a.kv.pair_stride_page + ((int64_t)head * a.kv.page_size + entry) * 4 : 0;
        cp_async8(stage + Sh::kPairs + lane * 8, a.kv.pairs + pair, page >= 0);
      }
      cp_async_commit();
    };
    int page = load_page(0);
#pragma unroll
    for (int i = 0; i < kAttnStages - 1; ++i) {
      const int next = load_page(i + 1);
      issue(i, page);
      page = next;
    }
    __syncthreads();  // the queries are in shared memory

    float qsum0 = 0.0f, qsum1 = 0.0f;
#pragma unroll
    for (int s = 0; s < D / 16; ++s) {
      const uint4 v = lds128(qfrag_u + (s * 32 + lane) * 16);
      const float2 x = Elem<T>::to_f2(v.x), y = Elem<T>::to_f2(v.y), z = Elem<T>::to_f2(v.z), w = Elem<T>::to_f2(v.w);
      qsum0 += (x.x + x.y) + (z.x + z.y);
      qsum1 += (y.x + y.y) + (w.x + w.y);
    }
    qsum0 += __shfl_xor_sync(0xffffffffu, qsum0, 1);
    qsum0 += __shfl_xor_sync(0xffffffffu, qsum0, 2);
    qsum1 += __shfl_xor_sync(0xffffffffu, qsum1, 1);
    qsum1 += __shfl_xor_sync(0xffffffffu, qsum1, 2);

    float o[kNt][4];
#pragma unroll
    for (int j = 0; j < kNt; ++j)
#pragma unroll
      for (int c = 0; c < 4; ++c) o[j][c] = 0.0f;
    float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.0f, l1 = 0.0f, r0 = 0.0f, r1 = 0.0f;

    for (int i = 0; i < runs; ++i) {
      cp_async_wait<kAttnStages - 2>();
      __syncwarp();  // run i has landed, and every lane has read run i - 1, whose stage is filled next
      {
        const int next = load_page(i + kAttnStages);
        issue(i + kAttnStages - 1, page);
        page = next;
      }
      const uint32_t stage = ring_u + (i % kAttnStages) * Sh::kStage;
      const int tb = t0 + kAttnRun * (warp + kAttnWarps * i);

      float s[4][4];
      uint32_t kw[4][kWords];
#pragma unroll
      for (int nt = 0; nt < 4; ++nt) {
        const uint32_t at_row = stage + Sh::kKeys + (nt * 8 + g) * Sh::kRowBytes + t * (D / 8);
        if (D == 128) {
          const uint4 v = lds128(at_row);
          kw[nt][0] = v.x; kw[nt][1] = v.y; kw[nt][kWords - 2] = v.z; kw[nt][kWords - 1] = v.w;
        } else {
          const uint2 v = lds64(at_row);
          kw[nt][0] = v.x; kw[nt][1] = v.y;
        }
        s[nt][0] = s[nt][1] = Keys::kStart * qsum0;
        s[nt][2] = s[nt][3] = Keys::kStart * qsum1;
      }
#pragma unroll
      for (int w = 0; w < kWords; ++w) {
        const uint4 qa = lds128(qfrag_u + (2 * w * 32 + lane) * 16);
        const uint4 qb = lds128(qfrag_u + ((2 * w + 1) * 32 + lane) * 16);
#pragma unroll
        for (int nt = 0; nt < 4; ++nt) {
          uint32_t p[4];
          Keys::unpack(kw[nt][w], p);
          Keys::mma(s[nt], qa, p[0], p[1]);
          Keys::mma(s[nt], qb, p[2], p[3]);
        }
      }

      // The pairs: logits in units of log2, and what the values need of each token.
      float vs[4][2], vm[4][2];
#pragma unroll
      for (int nt = 0; nt < 4; ++nt) {
        const uint4 v = lds128(stage + Sh::kPairs + nt * 64 + t * 16);
        const uint32_t kp[2] = {v.x, v.z}, vp[2] = {v.y, v.w};
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const float sk = __uint_as_float(kp[c] << 16);
          const float km = __uint_as_float(kp[c] & 0xffff0000u);
          const float ks = sk * a.scale_log2, kb = fmaf(Keys::kCentre, sk, km) * a.scale_log2;
          vs[nt][c] = __uint_as_float(vp[c] << 16);
          vm[nt][c] = fmaf(8.0f, vs[nt][c], __uint_as_float(vp[c] & 0xffff0000u));
          s[nt][c] = fmaf(s[nt][c], ks, qsum0 * kb);
          s[nt][2 + c] = fmaf(s[nt][2 + c], ks, qsum1 * kb);
        }
      }
      const bool edge = tb + kAttnRun > min(lim_first, t1);
      if (edge) {
#pragma unroll
        for (int nt = 0; nt < 4; ++nt)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const int tok = tb + nt * 8 + 2 * t + c;
            if (tok >= lim0 || tok >= t1) s[nt][c] = -INFINITY;
            if (tok >= lim1 || tok >= t1) s[nt][2 + c] = -INFINITY;
          }
      }
      float x0 = -INFINITY, x1 = -INFINITY;
#pragma unroll
      for (int nt = 0; nt < 4; ++nt) {
        x0 = fmaxf(x0, fmaxf(s[nt][0], s[nt][1]));
        x1 = fmaxf(x1, fmaxf(s[nt][2], s[nt][3]));
      }
      x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, 1));
      x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, 2));
      x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, 1));
      x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, 2));
      // The reference point of the exponentials moves only when a logit passes it by 8 (a factor of 256,
      // harmless in fp32 and bf16): the accumulators are then rescaled, which most runs need not do.
      if (__any_sync(0xffffffffu, x0 > m0 + 8.0f || x1 > m1 + 8.0f)) {
        const float n0 = fmaxf(m0, x0), n1 = fmaxf(m1, x1);
        const float f0 = n0 == m0 ? 1.0f : ex2(m0 - n0), f1 = n1 == m1 ? 1.0f : ex2(m1 - n1);
        m0 = n0;
        m1 = n1;
        l0 *= f0; r0 *= f0;
        l1 *= f1; r1 *= f1;
#pragma unroll
        for (int j = 0; j < kNt; ++j) {
          o[j][0] *= f0; o[j][1] *= f0;
          o[j][2] *= f1; o[j][3] *= f1;
        }
      }
      const float ref0 = m0 == -INFINITY ? 0.0f : m0, ref1 = m1 == -INFINITY ? 0.0f : m1;
      // A hidden token's terms are left out, not multiplied by its zero weight: its pair may be NaN.
      auto weigh = [&](auto masked) {
#pragma unroll
        for (int nt = 0; nt < 4; ++nt)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const bool in0 = !masked.value || s[nt][c] != -INFINITY, in1 = !masked.value || s[nt][2 + c] != -INFINITY;
            const float p0 = ex2(s[nt][c] - ref0), p1 = ex2(s[nt][2 + c] - ref1);
            l0 += p0;
            l1 += p1;
            r0 = in0 ? fmaf(p0, vm[nt][c], r0) : r0;
            r1 = in1 ? fmaf(p1, vm[nt][c], r1) : r1;
            s[nt][c] = in0 ? p0 * vs[nt][c] : 0.0f;
            s[nt][2 + c] = in1 ? p1 * vs[nt][c] : 0.0f;
          }
      };
      if (edge) weigh(std::true_type{}); else weigh(std::false_type{});

#pragma unroll
      for (int kk = 0; kk < 2; ++kk) {
        float (&sa)[4] = s[2 * kk];
        float (&sb)[4] = s[2 * kk + 1];
        const uint4 hi = make_uint4(pack_bf16(sa[0], sa[1]), pack_bf16(sa[2], sa[3]), pack_bf16(sb[0], sb[1]),
                                    pack_bf16(sb[2], sb[3]));
        uint4 lo = make_uint4(0, 0, 0, 0);
        if (sizeof(T) == 2 && Keys::kCentre != 0.0f) {  // fp16 queries: the rest of p sv
          const float2 h0 = Elem<__nv_bfloat16>::to_f2(hi.x), h1 = Elem<__nv_bfloat16>::to_f2(hi.y);
          const float2 h2 = Elem<__nv_bfloat16>::to_f2(hi.z), h3 = Elem<__nv_bfloat16>::to_f2(hi.w);
          lo = make_uint4(pack_bf16(sa[0] - h0.x, sa[1] - h0.y), pack_bf16(sa[2] - h1.x, sa[3] - h1.y),
                          pack_bf16(sb[0] - h2.x, sb[1] - h2.y), pack_bf16(sb[2] - h3.x, sb[3] - h3.y));
        }
        constexpr int kVWords = D / 64;
        uint32_t vw[4][kVWords];
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const int row = 16 * kk + 2 * t + (x & 1) + 8 * (x >> 1);
          const uint32_t src = stage + Sh::kValues + value_offset<D>(row, (g * (D / 16)) & ~15) + ((g * (D / 16)) & 15);
          if (D == 128) {
            const uint2 v = lds64(src);
            vw[x][0] = v.x;
            vw[x][kVWords - 1] = v.y;
          } else {
            vw[x][0] = lds32(src);
          }
        }
#pragma unroll
        for (int w = 0; w < kVWords; ++w) {
          const uint32_t ab[2] = {__byte_perm(vw[0][w], vw[1][w], 0x5410), __byte_perm(vw[0][w], vw[1][w], 0x7632)};
          const uint32_t cd[2] = {__byte_perm(vw[2][w], vw[3][w], 0x5410), __byte_perm(vw[2][w], vw[3][w], 0x7632)};
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const uint32_t b0 = value_codes(ab[e >> 2], e & 3), b1 = value_codes(cd[e >> 2], e & 3);
            mma_bf16(o[8 * w + e], hi.x, hi.y, hi.z, hi.w, b0, b1);
            if (sizeof(T) == 2 && Keys::kCentre != 0.0f) mma_bf16(o[8 * w + e], lo.x, lo.y, lo.z, lo.w, b0, b1);
          }
        }
      }
    }
    cp_async_wait<0>();

    l0 += __shfl_xor_sync(0xffffffffu, l0, 1);
    l0 += __shfl_xor_sync(0xffffffffu, l0, 2);
    l1 += __shfl_xor_sync(0xffffffffu, l1, 1);
    l1 += __shfl_xor_sync(0xffffffffu, l1, 2);
    r0 += __shfl_xor_sync(0xffffffffu, r0, 1);
    r0 += __shfl_xor_sync(0xffffffffu, r0, 2);
    r1 += __shfl_xor_sync(0xffffffffu, r1, 1);
    r1 += __shfl_xor_sync(0xffffffffu, r1, 2);

    // Join the warps: statistics, then o (with the minima's part added), lane by lane.
    if (t == 0) {
      stats[(warp * kAttnRows + g) * 2] = m0;
      stats[(warp * kAttnRows + g) * 2 + 1] = l0;
      stats[(warp * kAttnRows + g + 8) * 2] = m1;
      stats[(warp * kAttnRows + g + 8) * 2 + 1] = l1;
    }
    __syncthreads();  // all rings are drained: their memory may be overwritten
#pragma unroll
    for (int j = 0; j < kNt; ++j) {
      merge[((warp * kNt + j) * 4 + 0) * 32 + lane] = o[j][0] + r0;
      merge[((warp * kNt + j) * 4 + 1) * 32 + lane] = o[j][1] + r0;
      merge[((warp * kNt + j) * 4 + 2) * 32 + lane] = o[j][2] + r1;
      merge[((warp * kNt + j) * 4 + 3) * 32 + lane] = o[j][3] + r1;
    }
    __syncthreads();
    const bool starts = unit == 0, ends = unit + seg_units == rq.units;
    const int slot = starts && !ends ? 1 : 0;
    float* part = a.part + ((int64_t)blockIdx.x * 2 + slot) * attn_part_floats(D);
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int r = g + 8 * half;
      float top = -INFINITY, sum = 0.0f, f[kAttnWarps];
#pragma unroll
      for (int w = 0; w < kAttnWarps; ++w) top = fmaxf(top, stats[(w * kAttnRows + r) * 2]);
#pragma unroll
      for (int w = 0; w < kAttnWarps; ++w) {
        const float mw = stats[(w * kAttnRows + r) * 2];
        f[w] = mw == top ? 1.0f : ex2(mw - top);
        sum = fmaf(f[w], stats[(w * kAttnRows + r) * 2 + 1], sum);
      }
      if (r < rows_here) {
        const int tok = (row0 + r) / a.group, sub = (row0 + r) - tok * a.group;
        const float inv = sum != 0.0f ? 1.0f / sum : 0.0f;  // a row that sees no key is zero
        // This warp's quarter of the columns: kNt / 4 consecutive elements of each of the lane's two stretches.
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float v[kNt / 4];
#pragma unroll
          for (int jj = 0; jj < kNt / 4; ++jj) {
            const int j = warp * (kNt / 4) + jj;
            float x = 0.0f;
#pragma unroll
            for (int w = 0; w < kAttnWarps; ++w)
              x = fmaf(f[w], merge[((w * kNt + j) * 4 + 2 * half + c) * 32 + lane], x);
            v[jj] = x;
          }
          const int d0 = (D / 8) * (2 * t + c) + warp * (kNt / 4);
          if (starts && ends) {
            uint16_t* dst = static_cast<uint16_t*>(a.out) + (int64_t)(rq.q0 + tok) * a.osn +
                            ((int64_t)head * a.group + sub) * a.osh + d0;
#pragma unroll
            for (int jj = 0; jj < kNt / 4; ++jj) dst[jj] = Elem<T>::from_f(v[jj] * inv);
          } else {
#pragma unroll
            for (int jj = 0; jj < kNt / 4; ++jj) part[r * D + d0 + jj] = v[jj];
          }
        }
        if (warp == 0 && t == 0) {
          if (starts && ends) {
            if (a.lse != nullptr)
              a.lse[(int64_t)(rq.q0 + tok) * heads * a.group + (int64_t)head * a.group + sub] =
                  sum != 0.0f ? top + __log2f(sum) : -INFINITY;
          } else {
            part[kAttnRows * D + 2 * r] = top;
            part[kAttnRows * D + 2 * r + 1] = sum;
          }
        }
      }
    }
    if (starts && !ends) {
      // The tile goes on in the following CTAs, up to the one that holds its last unit.
      const int64_t last = (at + rq.units - 1) / share;
      desc_parts = (int)(last - blockIdx.x) + 1;
      desc_request = b;
      desc_row = tile * kAttnRows;
      desc_head = head;
    }
    __syncthreads();  // merge and the queries may be overwritten

    at += seg_units;
    unit += seg_units;
    if (unit == rq.units && at < end) {
      unit = 0;
      if (++head == heads) {
        head = 0;
        if (++tile == rq.tiles) {
          tile = 0;
          do rq = attn_request(a, ++b, nullptr); while (rq.tiles == 0);  // at < end: there is one
        }
      }
    }
  }
  if (tid == 0 && a.desc != nullptr) {
    desc[0] = desc_parts;
    desc[1] = desc_request;
    desc[2] = desc_row;
    desc[3] = desc_head;
  }
  pdl_launch_dependents();
}

// Joins the parts of the tiles that were split: CTA (c, y) takes rows 4y .. 4y + 3 of the tile that the
// main kernel's CTA c started, a warp a row, in the order of the parts.
template <typename T, int D>
__global__ void __launch_bounds__(kAttnThreads) attn_int4_join_kernel(const AttnInt4Args a) {
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int r = blockIdx.y * kAttnWarps + (threadIdx.x >> 5);
  const int32_t* desc = a.desc + (int64_t)blockIdx.x * kAttnDescInts;
  const int parts = desc[0];
  if (parts > 0) {
    const AttnRequest rq = attn_request(a, desc[1], nullptr);
    const int row = desc[2] + r, head = desc[3];
    if (row < rq.qlen * a.group) {
      constexpr int kPer = D / 32;
      const int64_t stride = 2 * attn_part_floats(D);
      // part 0 is slot 1 of CTA c, part i slot 0 of CTA c + i
      const float* first = a.part + ((int64_t)blockIdx.x * 2 + 1) * attn_part_floats(D);
      const float* rest = a.part + (int64_t)blockIdx.x * stride;
      float top = -INFINITY;
      for (int i = lane; i < parts; i += 32)
        top = fmaxf(top, (i == 0 ? first : rest + i * stride)[kAttnRows * D + 2 * r]);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      float sum = 0.0f, acc[kPer];
#pragma unroll
      for (int j = 0; j < kPer; ++j) acc[j] = 0.0f;
#pragma unroll 4
      for (int i = 0; i < parts; ++i) {
        const float* p = i == 0 ? first : rest + i * stride;
        const float m = p[kAttnRows * D + 2 * r], l = p[kAttnRows * D + 2 * r + 1];
        const float f = m == top ? 1.0f : ex2(m - top);
        sum = fmaf(f, l, sum);
#pragma unroll
        for (int j = 0; j < kPer; ++j) acc[j] = fmaf(f, p[r * D + j * 32 + lane], acc[j]);
      }
      const int tok = row / a.group, sub = row - tok * a.group;
      const float inv = sum != 0.0f ? 1.0f / sum : 0.0f;
      uint16_t* dst = static_cast<uint16_t*>(a.out) + (int64_t)(rq.q0 + tok) * a.osn +
                      ((int64_t)head * a.group + sub) * a.osh;
#pragma unroll
      for (int j = 0; j < kPer; ++j) dst[j * 32 + lane] = Elem<T>::from_f(acc[j] * inv);
      if (lane == 0 && a.lse != nullptr)
        a.lse[(int64_t)(rq.q0 + tok) * a.kv.heads * a.group + (int64_t)head * a.group + sub] =
            sum != 0.0f ? top + __log2f(sum) : -INFINITY;
    }
  }
  pdl_launch_dependents();
}

}  // namespace mas
