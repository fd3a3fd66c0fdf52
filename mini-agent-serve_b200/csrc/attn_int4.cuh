// attn_int4.cuh -- attention of ragged query rows over the 4-bit paged KV cache (sm_100a).
//
// With k_t = ck_t sk_t + mk_t and v_t = cv_t sv_t + mv_t (kv_int4.cuh), a query row q sees
//   S_t = scale * (sk_t * sum_d q_d ck_td + mk_t * sum_d q_d)            (t up to the row's causal limit)
//   o_d = (sum_t p_t sv_t (cv_td - z) + sum_t p_t (mv_t + z sv_t)) / sum_t p_t,   p_t = exp(S_t - max S)
// so the matrix products run on the bare codes, exact in 16 bits, and the pairs enter per token in fp32:
// no key or value is ever rounded. The weights w_t = p_t sv_t are rounded to fp16 for the second product (11 bits
// where bf16 has 8, whatever the queries' type); their own running reference, apart from the logits', keeps the
// largest of a row near 1 down to the least scale, 2^-126 (2^-14 there). p stays below 2^14, so the sums hold values up to
// 2^90. Maxima, sums and products are accumulated in fp32. z is 0 for bf16 results and 7.5 for fp16 ones, where the weights'
// rounding counts: it then meets codes of half the size.
//
// Work split. The rows of a request that share a kv head (tokens x group, token-major) are cut into tiles of
// 8 or 16, the tile's keys into units; all units of a launch, requests outermost, form one line that the
// CTAs cut into equal shares, whatever the lengths are (they are only known on the device). A share that
// covers a tile's keys writes the output; the others leave (sum, maximum, unnormalised o) in the
// workspace, and a second kernel joins them in a fixed order, so results do not change from run to run.
//
// A CTA is 4 warps. Where the number of kv heads is even, two take one head and two the next: under the NHD layout
// a token's codes of two heads are one 128-byte line, and fetched apart in time they came from DRAM twice (1.085 GB
// read for 0.572 GB at 256 requests x 2048 tokens). A head's warps take its runs of 32 tokens in turn, each with a
// ring of cp.async stages of its own, an online softmax of its own, and no barrier until the tile ends.
//
// Both products have the tokens' codes as the A operand of mma.m16n8k16 (16 tokens x D, then D x 16 tokens) and
// the rows as its 8 columns, so tiles come in steps of 8 rows and a lane's operands come straight from the
// staged bytes: the D axis is permuted so that a lane's codes are 16 (8) consecutive bytes of a row. The weights
// leave the first product's layout for the second's operand by one 8x8 transpose (movmatrix) each.
//
// Measured (96/8 heads of 128, graph replays): 256 requests of up to 4 K tokens, a query each, 186 us against a floor of 88
// (bytes); 48 of up to 8 K with 2 to 8 drafts each (32/8 heads, fp16) 141 (37); what bounds it is issue: 740 warp instructions a run of 32 tokens of a head, 51 % of the
// slots with 12 warps an SM, ALU 42 %, tensor pipe 35 %, DRAM 37 %. 12 heads of 64 with one row each: 27 us (6), latency.
#pragma once

#include <type_traits>

#include "common.cuh"
#include "kv_int4.cuh"

namespace mas {

constexpr int kAttnThreads = 128;
constexpr int kAttnWarps = kAttnThreads / 32;
constexpr int kAttnStages = 2;
constexpr int kAttnRun = 32;  // tokens of one stage of one warp
constexpr int kAttnMaxHeads = 2;  // kv heads a CTA takes at once
// What starting on a tile costs (its queries, the first loads' latency, the joining of the warps), in units of work:
// without it the shares with many short requests finish last. 256 requests of 1 to 4096 tokens, 96 / 8 heads: 310 us
// with 0, 271 with 2, 255 with 4, 256 with 6 (before the products were all fp16).
constexpr int kAttnLead = 4;

// How far a logit (log2), and so a p, may lie past its row's reference before the reference moves.
constexpr float kAttnFarLogit = 12.0f, kAttnFarP = 4096.0f;

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
  float* part;                 // [grid][2][heads a CTA][rows a tile * (D + 2)]
  int32_t* desc;               // [grid][kAttnDescInts]; nullptr: no tile can be split
  // softmax scale * log2(e): its sign (0 for 0) enters with the keys' pairs, its size with a query row's scale, so that no
  // product on the way to a logit is far larger than the larger of the logit and the key
  float key_sign, row_scale;
  int32_t B, max_blocks, group;
  int32_t page_shift;          // log2(page_size), or -1
  int32_t causal;
  int32_t cta_heads;           // 1 or 2
  int32_t q_vec, o_vec;        // rows of queries, of results are 16-byte aligned
  int32_t split_rows;          // requests with more rows are the prompt kernel's
  uint32_t page16, entry16;    // the codes' strides in units of 16 bytes
  int32_t* status;
};

// What the joining kernel needs of a tile that was split: written by the CTA whose share starts the tile.
// {number of parts (0: nothing to join), the request's first query and queries, the tile's first row within it, first kv head}
constexpr int kAttnDescInts = 5;

// A part of a tile: its rows' unnormalised o, then {maximum, sum} of each.
__host__ __device__ constexpr int attn_part_floats(int D, int rows) { return rows * (D + 2); }

// NT: the tile's rows in eights.
template <int D, int NT>
struct AttnInt4Shape {
  static constexpr int kRows = 8 * NT;
  static constexpr int kPass = 2;  // 16-token steps a warp computes at once: with one, 204 us where two take 196
  // By registers (128 and 168 a thread). At 16 rows four CTAs of 128 registers took 211 us where three take 196
  // (spills, or half the independent products a warp), two of 255 took 221.
  static constexpr int kCtasPerSm = NT == 1 ? 4 : 3;
  static constexpr int kRowBytes = D / 2;
  static constexpr int kKeys = 0;
  static constexpr int kValues = kAttnRun * kRowBytes;
  static constexpr int kPairs = 2 * kAttnRun * kRowBytes;
  static constexpr int kFactors = kPairs + kAttnRun * 8;         // the pairs as fp32 factors
  static constexpr int kStage = kFactors + kAttnRun * 16;
  static constexpr int kWarpRing = kAttnStages * kStage;
  static constexpr int kQHead = D / 32 * NT * 512;               // a head's queries as operands
  static constexpr int kQFrag = kAttnMaxHeads * kQHead;
  static constexpr int kMerge = kAttnWarps * (D / 4 * NT) * 32 * 4;  // the warps' o
  static constexpr int kRing = kAttnWarps * kWarpRing;
  static constexpr int kStats = kAttnWarps * kRows * 3 * 4;
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
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
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
__device__ __forceinline__ void sts128(uint32_t a, float x, float y, float z, float w) {
  asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(a), "f"(x), "f"(y), "f"(z), "f"(w) : "memory");
}
__device__ __forceinline__ float2 lds_float2(uint32_t a) {
  const uint2 v = lds64(a);
  return make_float2(__uint_as_float(v.x), __uint_as_float(v.y));
}
__device__ __forceinline__ uint32_t lds32(uint32_t a) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(a));
  return v;
}

#define MAS_MMA(NAME, SHAPE)                                                                                     \
  __device__ __forceinline__ void NAME(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,         \
                                       uint32_t b0, uint32_t b1) {                                               \
    asm volatile("mma.sync.aligned." SHAPE " {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"     \
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])                                                \
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));                                        \
  }                                                                                                              \
  __device__ __forceinline__ void NAME##_first(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, \
                                               uint32_t b0, uint32_t b1) {                                       \
    asm volatile("mma.sync.aligned." SHAPE " {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};" \
                 : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])                                                \
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));                             \
  }
MAS_MMA(mma_fp16, "m16n8k16.row.col.f32.f16.f16.f32")
#undef MAS_MMA

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// A code word's nibbles at bits 0, 4, 8, 12 of each half as fp16 pairs. A nibble c at the foot of a half IS the
// fp16 denormal c * 2^-24, one nibble up c * 2^-20: two masks a byte, no arithmetic.
constexpr float kEvenUnit = 16777216.0f, kOddUnit = 1048576.0f;  // 2^24, 2^20: what undoes that
// A row's sums are kept at 2^-22 of what its scaled queries give, next to a key's size: a key's scale then meets a factor of 4, where
// one of 2^24 took scales above 2^104 out of fp32.
constexpr float kSumUnit = 2.38418579e-7f;
__device__ __forceinline__ void nibbles_fp16(uint32_t w, uint32_t (&p)[4]) {
  p[0] = w & 0x000f000fu;
  p[1] = w & 0x00f000f0u;
  p[2] = (w >> 8) & 0x000f000fu;
  p[3] = (w >> 8) & 0x00f000f0u;
}

// One lane's 8 query elements that meet one code word, as the first product's operand: elements that meet odd
// nibbles are divided by 16. The row has been scaled by a power of two to a largest element of 2^15 to 2^16 (fp16 ends at 65504,
// which holds 11 bits there), where fp16 holds a bf16 row's 8 bits down to 2^-29 of that largest, and an fp16 row's elements to
// within 2^-36 of it.
__device__ __forceinline__ uint4 query_operand(const float (&f)[8]) {
  constexpr float kOdd = 0.0625f;
  return make_uint4(Elem<__half>::from_f2(f[0], f[4]), Elem<__half>::from_f2(f[1] * kOdd, f[5] * kOdd),
                    Elem<__half>::from_f2(f[2], f[6]), Elem<__half>::from_f2(f[3] * kOdd, f[7] * kOdd));
}

// What takes a row's sums back to logits: 2^exponent times the softmax scale, kept among the normal numbers (a hidden key's
// -infinity has to survive it; at the upper end, queries above 2^123 under the usual scales, any difference of logits is past any softmax).
__device__ __forceinline__ float row_unscale(float power, float scale) {
  return fminf(fmaxf(power * scale, 1.17549435e-38f), 3.40282347e38f);
}

// The 8x8 matrix of 16-bit elements held as pairs (row lane / 4, columns 2 (lane % 4), + 1), transposed.
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

__device__ __forceinline__ uint32_t max_nan_half2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

// Where a staged value row's 16-byte chunk lies: exchanged so that one chunk of eight consecutive rows, which a matrix
// load reads at once, covers all banks.
template <int D>
__device__ __forceinline__ uint32_t value_offset(int row, int chunk) {
  return D == 128 ? row * 64 + ((chunk ^ ((row >> 1) & 3)) << 4) : row * 32 + ((chunk ^ ((row >> 2) & 1)) << 4);
}

// Four 8x8 matrices of 16-bit units, transposed: matrix i's rows are the 16 bytes at lanes 8i .. 8i + 7's addresses; lane
// (g, t) receives column g of rows 2t, 2t + 1 of each.
__device__ __forceinline__ void load_transposed(uint32_t (&r)[4], uint32_t a) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(a));
}

// A request's extent, with every length that does not fit its buffers cut to them.
struct AttnRequest {
  int32_t q0, qlen;  // first query row, queries
  int32_t n;         // tokens in the cache
  int32_t tiles, units;
  __device__ __forceinline__ int64_t work(int head_groups) const { return (int64_t)tiles * head_groups * (units + kAttnLead); }
};

template <int ROWS>
__device__ __forceinline__ AttnRequest attn_request(const AttnInt4Args& a, int b, int32_t* status, bool few = true) {
  const int unit = kAttnRun * (kAttnWarps / a.cta_heads);
  AttnRequest r;
  int64_t q0 = b, q1 = b + 1;
  if (a.cum_q != nullptr) {
    q0 = a.cum_q[b];
    q1 = a.cum_q[b + 1];
  }
  const int64_t capacity = min((int64_t)a.max_blocks * a.kv.page_size, (int64_t)INT32_MAX - 2 * kAttnRun * kAttnWarps);
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
  const int64_t rows = (int64_t)r.qlen * a.group;
  r.tiles = few && rows > a.split_rows ? 0 : (int32_t)((rows + ROWS - 1) / ROWS);
  r.units = max(1, (r.n + unit - 1) / unit);
  return r;
}

template <typename T, int D, int NT>
__global__ void __launch_bounds__(kAttnThreads, AttnInt4Shape<D, NT>::kCtasPerSm)
    attn_int4_kernel(const AttnInt4Args a) {
  using Sh = AttnInt4Shape<D, NT>;
  // fp16 results: the second product's codes are centred (c - 7.5), through one more product with ones that sums the
  // rounded weights; their rounding then meets codes of half the size. bf16 results are rounded 8 times coarser.
  constexpr bool kCentred = std::is_same<T, __half>::value;
  constexpr float kCentre = kCentred ? 7.5f : 0.0f;
  constexpr int kRows = Sh::kRows;
  constexpr int kMt = D / 16;     // 16-row tiles of the second product's D axis
  constexpr int kWords = D / 32;  // key code words a lane and token
  constexpr int kPass = Sh::kPass;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ int64_t s_scan[kAttnWarps + 2];
  __shared__ int32_t s_b;
  __shared__ AttnRequest s_rq;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, t = lane & 3;
  uint8_t* ring = smem + Sh::kQFrag;
  const uint32_t ring_u = smem_u32(ring) + warp * Sh::kWarpRing;
  float* merge = reinterpret_cast<float*>(ring);
  float* stats = reinterpret_cast<float*>(smem + Sh::kSmem - Sh::kStats);  // [warp][row][m, l]
  float* qrow = stats + kAttnWarps * kRows * 2;                            // [head][pair of rows][2 sums of q, 2 scales]
  int32_t* desc = a.desc + (int64_t)blockIdx.x * kAttnDescInts;
  pdl_wait();

  // This CTA's share of the line of units: total by a block sum, the request it starts in by the scan.
  const int cta_heads = a.cta_heads, head_warps = kAttnWarps / cta_heads, head_groups = a.kv.heads / cta_heads;
  const int unit_tokens = kAttnRun * head_warps;
  const int which = warp / head_warps, sub_warp = warp % head_warps;  // this warp's head of the CTA's, its place there
  const int per = (a.B + kAttnThreads - 1) / kAttnThreads;
  const int rb0 = min(a.B, tid * per), rb1 = min(a.B, rb0 + per);
  int64_t mine = 0;
  AttnRequest first_rq = {};
  for (int b = rb0; b < rb1; ++b) {
    const AttnRequest x = attn_request<kRows>(a, b, blockIdx.x == 0 ? a.status : nullptr);
    if (b == rb0) first_rq = x;
    mine += x.work(head_groups);
  }
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
    AttnRequest mine_rq = first_rq;
    for (; b < rb1; ++b) {
      if (b > rb0) mine_rq = attn_request<kRows>(a, b, nullptr);
      const int64_t w = mine_rq.work(head_groups);
      if (rem < w) break;
      rem -= w;
    }
    s_b = b;
    s_rq = mine_rq;
    s_scan[kAttnWarps] = rem;
  }
  __syncthreads();
  int b = s_b;
  AttnRequest rq = s_rq;
  int unit, head_group, tile;
  {
    int64_t rem = s_scan[kAttnWarps];
    unit = (int)(rem % (rq.units + kAttnLead)) - kAttnLead;  // below 0: the start's cost
    rem /= rq.units + kAttnLead;
    head_group = (int)(rem % head_groups);
    tile = (int)(rem / head_groups);
  }
  int desc_parts = 0, desc_q0 = 0, desc_qlen = 0, desc_row = 0, desc_head = 0;

  while (at < end) {
    // Of this share, the start's cost is passed over. A share may hold nothing but (a part of) that.
    const int lead = (int)min((int64_t)max(-unit, 0), end - at);
    at += lead;
    unit += lead;
    if (at == end) break;
    const int seg_units = (int)min((int64_t)(rq.units - unit), end - at);
    const int row0 = tile * kRows;
    const int rows_here = min(kRows, rq.qlen * a.group - row0);
    const int head = head_group * cta_heads + which;
    // Tokens visible to row r of the tile: those before its limit. Rows past the last take the last one's limit.
    auto limit = [&](int r) {
      const int tok = (row0 + min(r, rows_here - 1)) / a.group;
      return a.causal ? min(rq.n, max(0, rq.n - rq.qlen + tok + 1)) : rq.n;
    };
    const int t0 = unit * unit_tokens;
    const int t1 = min((unit + seg_units) * unit_tokens, limit(kRows - 1));
    const int lim_first = limit(0);
    const uint32_t head16 = (uint32_t)(head * a.kv.stride_head >> 4);

    const uint32_t qfrag_u = smem_u32(smem) + which * Sh::kQHead + lane * 16;

    // The warp's runs: t0 + 32 (sub_warp + head_warps * i).
    const int runs_all = t1 > t0 ? (t1 - t0 + kAttnRun - 1) / kAttnRun : 0;
    const int runs = runs_all > sub_warp ? (runs_all - sub_warp + head_warps - 1) / head_warps : 0;
    const int32_t* table = a.block_tables + (int64_t)b * a.table_stride;
    auto load_page = [&](int i) {
      const int tok = t0 + kAttnRun * (sub_warp + head_warps * i) + lane;
      if (i >= runs || tok >= t1) return -1;
      const int block = a.page_shift >= 0 ? tok >> a.page_shift : tok / (int)a.kv.page_size;
      const int page = table[block];  // block < max_blocks: tok < n <= capacity
      if (page < 0 || page >= a.kv.num_pages) {
        flag_status(a.status, MAS_STATUS_KV_SLOT_OUT_OF_RANGE);
        return -1;  // its tokens read as zeros
      }
      return page;
    };
    // Offsets travel in units of 16 bytes: 32 bits reach 64 GB (checked by the host).
    auto issue = [&](int i, int page) {
      if (i < runs) {
        const int tok = t0 + kAttnRun * (sub_warp + head_warps * i) + lane;
        const int entry = a.page_shift >= 0 ? tok & ((1 << a.page_shift) - 1) : tok % (int)a.kv.page_size;
        const uint32_t stage = ring_u + (i % kAttnStages) * Sh::kStage;
        const uint32_t valid = __ballot_sync(0xffffffffu, page >= 0);
        const uint32_t off = page >= 0 ? (uint32_t)page * a.page16 + (uint32_t)entry * a.entry16 + head16 : 0u;
        constexpr int kChunks = Sh::kRowBytes / 16;
        constexpr int kRowsAtOnce = 32 / kChunks;
        const int chunk = lane % kChunks;
#pragma unroll
        for (int it = 0; it < kAttnRun / kRowsAtOnce; ++it) {
          const int row = it * kRowsAtOnce + lane / kChunks;
          const uint64_t src = (uint64_t)(__shfl_sync(0xffffffffu, off, row) + chunk) * 16;
          const uint32_t to_k = stage + Sh::kKeys + row * Sh::kRowBytes + chunk * 16;
          const uint32_t to_v = stage + Sh::kValues + value_offset<D>(row, chunk);
          if (valid == 0xffffffffu) {
            cp_async16(to_k, a.kv.k_codes + src);
            cp_async16(to_v, a.kv.v_codes + src);
          } else {
            const bool ok = (valid >> row) & 1u;
            cp_async16(to_k, a.kv.k_codes + src, ok);
            cp_async16(to_v, a.kv.v_codes + src, ok);
          }
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
    // Queries into shared memory as the first product takes them, a warp for eight rows of a head: lane (g, t) has
    // elements (D / 4) t and on of row g. Beside them the rows' sums and scales, two rows (2t, 2t + 1) together.
    for (int c = warp; c < cta_heads * NT; c += kAttnWarps) {
      const int nt = c % NT, hd = c / NT, rr = nt * 8 + g;
      float f[D / 32][8], sum = 0.0f, most = 0.0f;
      const int tok = (row0 + min(rr, rows_here - 1)) / a.group, sub = row0 + min(rr, rows_here - 1) - tok * a.group;
      const uint16_t* src = static_cast<const uint16_t*>(a.q) + (int64_t)(rq.q0 + tok) * a.qsn +
                            ((int64_t)(head_group * cta_heads + hd) * a.group + sub) * a.qsh + (D / 4) * t;
#pragma unroll
      for (int i = 0; i < D / 32; ++i) {
        unpack8<T>(a.q_vec ? kv_load8<true>(src + 8 * i) : kv_load8<false>(src + 8 * i), f[i]);
#pragma unroll
        for (int x = 0; x < 8; ++x) {
          f[i][x] = rr < rows_here ? f[i][x] : 0.0f;
          // as bits, so that a NaN is the most
          most = __uint_as_float(max(__float_as_uint(most), __float_as_uint(fabsf(f[i][x]))));
        }
      }
#pragma unroll
      for (int z = 1; z < 4; z <<= 1)
        most = __uint_as_float(max(__float_as_uint(most), __shfl_xor_sync(0xffffffffu, __float_as_uint(most), z)));
      const uint32_t exponent = min(max(__float_as_uint(most) >> 23, 16u), 254u);
      const float scale = __uint_as_float((269u - exponent) << 23);
#pragma unroll
      for (int i = 0; i < D / 32; ++i) {
#pragma unroll
        for (int x = 0; x < 8; ++x) {
          f[i][x] *= scale;
          sum += f[i][x];
        }
        *reinterpret_cast<uint4*>(smem + hd * Sh::kQHead + ((i * NT + nt) * 32 + lane) * 16) = query_operand(f[i]);
      }
#pragma unroll
      for (int z = 1; z < 4; z <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, z);
      if (t == 0) {
        float* dst = qrow + (hd * kRows + nt * 8 + (g & ~1)) * 2 + (g & 1);
        dst[0] = sum * kSumUnit;
        dst[2] = row_unscale(__uint_as_float((exponent - 15u) << 23), a.row_scale * (1.0f / kSumUnit));
      }
    }
    __syncthreads();  // the queries are in shared memory

    const uint32_t qrow_u = smem_u32(qrow) + which * kRows * 8 + t * 16;

    // o: tile j of the D axis holds elements 32 (j / 2) + 4g + 2 (j % 2) and the next, of rows 2t, 2t + 1. l and r (the
    // minima's part) are relative to 2^-nref, o to 2^-nref / wscale, wscale a power of two; l == 0: the row has seen no key
    // and nref means nothing.
    float o[kMt][NT][4];
    float2 nref[NT], wscale[NT], l[NT], r[NT];
    float wsum[kCentred ? NT : 1][4];  // the sum of the rounded weights, of rows 2t, 2t + 1 (twice)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int j = 0; j < kMt; ++j)
#pragma unroll
        for (int c = 0; c < 4; ++c) o[j][nt][c] = 0.0f;
      wscale[nt] = both(1.0f);
      nref[nt] = l[nt] = r[nt] = both(0.0f);
      if (kCentred) wsum[nt][0] = wsum[nt][1] = wsum[nt][2] = wsum[nt][3] = 0.0f;
    }

    // Run i has landed: each lane turns its token's pairs into what the logits and the values need.
    auto make_factors = [&](int i) {
      const uint32_t stage = ring_u + (i % kAttnStages) * Sh::kStage;
      const uint2 pr = lds64(stage + Sh::kPairs + lane * 8);
      const float sk = __uint_as_float(pr.x << 16), km = __uint_as_float(pr.x & 0xffff0000u);
      const float sv = __uint_as_float(pr.y << 16), vm = __uint_as_float(pr.y & 0xffff0000u);
      sts128(stage + Sh::kFactors + lane * 16, sk * (a.key_sign * (kEvenUnit * kSumUnit)), km * a.key_sign, sv,
             fmaf(kCentre, sv, vm));
      __syncwarp();
    };
    // The first product and the keys' pairs: the logits (over the row's scale) of kPass 16-token steps from p0 on,
    // s[x][nt] = tokens g, g + 8 of step p0 + x, rows 2t, 2t + 1.
    auto logits = [&](int i, int p0, float (&s)[kPass][NT][4]) {
      const uint32_t stage = ring_u + (i % kAttnStages) * Sh::kStage;
      uint32_t kw[kPass][2][kWords];
#pragma unroll
      for (int x = 0; x < kPass; ++x)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const uint32_t at_row = stage + Sh::kKeys + ((p0 + x) * 16 + half * 8 + g) * Sh::kRowBytes + t * (D / 8);
          if (D == 128) {
            const uint4 v = lds128(at_row);
            kw[x][half][0] = v.x; kw[x][half][1] = v.y;
            kw[x][half][kWords - 2] = v.z; kw[x][half][kWords - 1] = v.w;
          } else {
            const uint2 v = lds64(at_row);
            kw[x][half][0] = v.x; kw[x][half][1] = v.y;
          }
        }
#pragma unroll
      for (int w = 0; w < kWords; ++w) {
        uint32_t ka[kPass][2][4];
#pragma unroll
        for (int x = 0; x < kPass; ++x)
#pragma unroll
          for (int half = 0; half < 2; ++half) nibbles_fp16(kw[x][half][w], ka[x][half]);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const uint4 qb = lds128(qfrag_u + (w * NT + nt) * 512);
#pragma unroll
          for (int x = 0; x < kPass; ++x) {
            if (w == 0) mma_fp16_first(s[x][nt], ka[x][0][0], ka[x][1][0], ka[x][0][1], ka[x][1][1], qb.x, qb.y);
            else mma_fp16(s[x][nt], ka[x][0][0], ka[x][1][0], ka[x][0][1], ka[x][1][1], qb.x, qb.y);
            mma_fp16(s[x][nt], ka[x][0][2], ka[x][1][2], ka[x][0][3], ka[x][1][3], qb.z, qb.w);
          }
        }
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const float2 qs = lds_float2(qrow_u + nt * 64);
#pragma unroll
        for (int x = 0; x < kPass; ++x)
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const float2 f = lds_float2(stage + Sh::kFactors + ((p0 + x) * 16 + half * 8 + g) * 16);
            const float2 y = fma2_f32(make_float2(s[x][nt][2 * half], s[x][nt][2 * half + 1]), both(f.x), mul2_f32(qs, both(f.y)));
            s[x][nt][2 * half] = y.x;
            s[x][nt][2 * half + 1] = y.y;
          }
      }
    };
    // One step: weights of the logits s, the running sums, the second product.
    const int mat_row = ((lane >> 3) & 1) * 8 + (lane & 7);
    const uint32_t v_lane = Sh::kValues + value_offset<D>(mat_row, lane >> 4);
    auto step = [&](int i, int p0, float (&s)[kPass][NT][4]) {
      const uint32_t stage = ring_u + (i % kAttnStages) * Sh::kStage;
      const int tb = t0 + kAttnRun * (sub_warp + head_warps * i) + p0 * 16;
      float2 unscale[NT];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) unscale[nt] = lds_float2(qrow_u + nt * 64 + 8);
      float2 vf[kPass][2];  // a token's value scale, and its minimum
#pragma unroll
      for (int x = 0; x < kPass; ++x)
#pragma unroll
        for (int half = 0; half < 2; ++half)
          vf[x][half] = lds_float2(stage + Sh::kFactors + ((p0 + x) * 16 + half * 8 + g) * 16 + 8);
      bool apart = false;
      if (tb + kPass * 16 > min(lim_first, t1)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const int lim = min(limit(nt * 8 + 2 * t + c), t1);
#pragma unroll
            for (int x = 0; x < kPass; ++x)
#pragma unroll
              for (int half = 0; half < 2; ++half)
                if (tb + x * 16 + half * 8 + g >= lim) s[x][nt][2 * half + c] = -INFINITY;
          }
        // A hidden token's zero weight hides its value, unless that is a NaN or an infinity.
        float odd = 0.0f;
#pragma unroll
        for (int x = 0; x < kPass; ++x)
#pragma unroll
          for (int half = 0; half < 2; ++half) odd = fmaf(vf[x][half].x, 0.0f, fmaf(vf[x][half].y, 0.0f, odd));
        apart = __any_sync(0xffffffffu, odd != 0.0f);
      }

      float2 p_sum[NT], r_new[NT];
      uint32_t wh[kPass][NT][2];
      uint32_t top;  // the largest weights, a NaN before all (0 * infinity, of a logit far past the reference, is one)
      auto weigh = [&](auto masked) {
        top = 0;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          p_sum[nt] = both(0.0f);
          r_new[nt] = r[nt];
#pragma unroll
          for (int x = 0; x < kPass; ++x)
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              const float2 sv = make_float2(s[x][nt][2 * half], s[x][nt][2 * half + 1]);
              const float2 dv = fma2_f32(sv, unscale[nt], nref[nt]);
              const float2 p = make_float2(ex2(dv.x), ex2(dv.y));
              // In this order, as p * wscale is finite and zero where p is: wscale * sv may overflow beside a p of zero.
              float2 w = mul2_f32(mul2_f32(p, wscale[nt]), both(vf[x][half].x));
              float2 vmh = both(vf[x][half].y);
              if (masked.value) {
                w.x = sv.x == -INFINITY ? 0.0f : w.x;
                w.y = sv.y == -INFINITY ? 0.0f : w.y;
                vmh.x = sv.x == -INFINITY ? 0.0f : vmh.x;
                vmh.y = sv.y == -INFINITY ? 0.0f : vmh.y;
              }
              p_sum[nt] = add2_f32(p_sum[nt], p);
              r_new[nt] = fma2_f32(p, vmh, r_new[nt]);
              wh[x][nt][half] = Elem<__half>::from_f2(w.x, w.y);
              top = max_nan_half2(top, wh[x][nt][half]);
            }
        }
      };
      weigh(std::false_type{});
      if (apart) weigh(std::true_type{});
      const bool first = i == 0 && p0 == 0;
      // The references move only when a weight passes 1024 (fp32 sums and fp16 weights have that much room), when a p passes
      // 2^12 (the weights of values of next to no spread never grow, but their minima enter with p alone: r stays finite for
      // values up to 2^90 and more tokens than fit), and with the first step: the accumulators are then rescaled, which most
      // steps need not do. A half above 1024 (0x6400), an infinity or a NaN carries into its sign bit.
      bool far = false;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) far |= fmaxf(p_sum[nt].x, p_sum[nt].y) > kAttnFarP * (2 * kPass);
      if (first || __any_sync(0xffffffffu, ((top + 0x1bff1bffu) & 0x80008000u) || far)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float hi[2] = {-INFINITY, -INFINITY}, hw[2] = {-INFINITY, -INFINITY}, seen[2] = {l[nt].x, l[nt].y};
#pragma unroll
          for (int x = 0; x < kPass; ++x)
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              const float lv = __log2f(vf[x][half].x);
#pragma unroll
              for (int c = 0; c < 2; ++c) {
                const float logit = s[x][nt][2 * half + c] * (c == 0 ? unscale[nt].x : unscale[nt].y);
                hi[c] = fmaxf(hi[c], logit);
                hw[c] = fmaxf(hw[c], logit + lv);  // fmaxf passes over a NaN
              }
            }
#pragma unroll
          for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int z = 4; z < 32; z <<= 1) {
              hi[c] = fmaxf(hi[c], __shfl_xor_sync(0xffffffffu, hi[c], z));
              hw[c] = fmaxf(hw[c], __shfl_xor_sync(0xffffffffu, hw[c], z));
              seen[c] = fmaxf(seen[c], __shfl_xor_sync(0xffffffffu, seen[c], z));
            }
          float fl[2], fo[2], nr[2] = {nref[nt].x, nref[nt].y}, ws[2] = {wscale[nt].x, wscale[nt].y};
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            // Only rows that need it move, so that no row's rounding depends on another's values. Then the largest
            // weight of the row so far (at most 1024 by the scale it has) or of this step becomes at most 1.
            const float old = seen[c] == 0.0f ? -INFINITY : -nr[c];
            const float was = old - __log2f(ws[c]);
            fl[c] = fo[c] = 1.0f;
            if (!(hw[c] > was + 10.0f || hi[c] > old + kAttnFarLogit)) continue;
            const float now = fmaxf(old, hi[c]);
            const float room = floorf(now - fmaxf(was, hw[c]));
            // At most 2^112: p * wscale stays finite (p is below 2^14 where the references stand), and the least scale,
            // 2^-126, still gives a weight that fp16 holds with all its bits.
            const float grow = fminf(fmaxf(room, -126.0f), 112.0f);
            const float nws = now == -INFINITY ? 1.0f : __uint_as_float((uint32_t)(grow + 127.0f) << 23);
            fl[c] = now == old ? 1.0f : ex2(old - now);
            fo[c] = ex2((now == old ? 0.0f : old - now) + (__log2f(nws) - __log2f(ws[c])));  // as one power: its parts leave fp32
            nr[c] = now == -INFINITY ? 0.0f : -now;
            ws[c] = nws;
          }
          nref[nt] = make_float2(nr[0], nr[1]);
          wscale[nt] = make_float2(ws[0], ws[1]);
          l[nt].x *= fl[0]; l[nt].y *= fl[1];
          r[nt].x *= fl[0]; r[nt].y *= fl[1];
#pragma unroll
          for (int j = 0; j < kMt; ++j) {
            o[j][nt][0] *= fo[0]; o[j][nt][1] *= fo[1];
            o[j][nt][2] *= fo[0]; o[j][nt][3] *= fo[1];
          }
          if (kCentred) {
            wsum[nt][0] *= fo[0]; wsum[nt][1] *= fo[1];
            wsum[nt][2] *= fo[0]; wsum[nt][3] *= fo[1];
          }
        }
        if (apart) weigh(std::true_type{}); else weigh(std::false_type{});
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        l[nt] = add2_f32(l[nt], p_sum[nt]);
        r[nt] = r_new[nt];
      }
#pragma unroll
      for (int x = 0; x < kPass; ++x)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int half = 0; half < 2; ++half) wh[x][nt][half] = transpose8x8(wh[x][nt][half]);
      if (kCentred) {
        constexpr uint32_t kOnes = 0x3c003c00u;
#pragma unroll
        for (int x = 0; x < kPass; ++x)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
            mma_fp16(wsum[nt], kOnes, kOnes, kOnes, kOnes, wh[x][nt][0], wh[x][nt][1]);
      }

      // The second product, D x rows over 16 tokens: a unit of four codes of tokens 2t, 2t + 1 (ab) and 2t + 8, 2t + 9 (cd)
      // comes transposed from shared memory, 32 elements of D a chunk.
#pragma unroll
      for (int x = 0; x < kPass; ++x)
#pragma unroll
        for (int c = 0; c < D / 32; c += 2) {
          uint32_t u[4];
          load_transposed(u, (stage + v_lane + (p0 + x) * 16 * Sh::kRowBytes) ^ (c * 16));
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            uint32_t ab[4], cd[4];
            nibbles_fp16(u[2 * k], ab);
            nibbles_fp16(u[2 * k + 1], cd);
#pragma unroll
            for (int e = 0; e < 2; ++e)
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
                mma_fp16(o[2 * (c + k) + e][nt], ab[2 * e], ab[2 * e + 1], cd[2 * e], cd[2 * e + 1], wh[x][nt][0], wh[x][nt][1]);
          }
        }
    };

    for (int i = 0; i < runs; ++i) {
      cp_async_wait<kAttnStages - 2>();
      __syncwarp();  // run i has landed, and every lane has read run i - 1, whose stage is filled next
      {
        const int next = load_page(i + kAttnStages);
        issue(i + kAttnStages - 1, page);
        page = next;
      }
      make_factors(i);
#pragma unroll
      for (int p0 = 0; p0 < 2; p0 += kPass) {
        float s[kPass][NT][4];
        logits(i, p0, s);
        step(i, p0, s);
      }
    }
    cp_async_wait<0>();

    // A row's sums over the lanes that hold its other tokens.
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int z = 4; z < 32; z <<= 1) {
        l[nt].x += __shfl_xor_sync(0xffffffffu, l[nt].x, z);
        l[nt].y += __shfl_xor_sync(0xffffffffu, l[nt].y, z);
        r[nt].x += __shfl_xor_sync(0xffffffffu, r[nt].x, z);
        r[nt].y += __shfl_xor_sync(0xffffffffu, r[nt].y, z);
      }

    // Join a head's warps, o and r of each relative to its own reference m.
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      if (g == 0) {
        float* st = stats + (warp * kRows + nt * 8 + 2 * t) * 2;
        st[0] = l[nt].x == 0.0f ? -INFINITY : -nref[nt].x; st[1] = l[nt].x;
        st[2] = l[nt].y == 0.0f ? -INFINITY : -nref[nt].y; st[3] = l[nt].y;
      }
    }
    __syncthreads();  // all rings are drained: their memory may be overwritten
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const float b0 = 1.0f / wscale[nt].x, b1 = 1.0f / wscale[nt].y;
      const float w0 = kCentred ? kCentre * wsum[nt][0] : 0.0f, w1 = kCentred ? kCentre * wsum[nt][1] : 0.0f;
#pragma unroll
      for (int j = 0; j < kMt; ++j) {
        float* dst = merge + ((warp * kMt + j) * NT + nt) * 128 + lane;
        dst[0] = fmaf(fmaf(o[j][nt][0], kEvenUnit, -w0), b0, r[nt].x);
        dst[32] = fmaf(fmaf(o[j][nt][1], kEvenUnit, -w1), b1, r[nt].y);
        dst[64] = fmaf(fmaf(o[j][nt][2], kOddUnit, -w0), b0, r[nt].x);
        dst[96] = fmaf(fmaf(o[j][nt][3], kOddUnit, -w1), b1, r[nt].y);
      }
    }
    __syncthreads();
    const bool starts = unit == 0, ends = unit + seg_units == rq.units;
    const int slot = starts && !ends ? 1 : 0;
    float* part = a.part + (((int64_t)blockIdx.x * 2 + slot) * cta_heads + which) * attn_part_floats(D, kRows);
    const int first_warp = which * head_warps;
    // This warp's share of the D tiles.
    const int tiles_here = kMt / head_warps;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int rr = nt * 8 + 2 * t + c;
        float top = -INFINITY, sum = 0.0f, f[kAttnWarps];
#pragma unroll
        for (int w = 0; w < kAttnWarps; ++w)
          if (w < head_warps) top = fmaxf(top, stats[((first_warp + w) * kRows + rr) * 2]);
#pragma unroll
        for (int w = 0; w < kAttnWarps; ++w) {
          f[w] = 0.0f;
          if (w < head_warps) {
            const float mw = stats[((first_warp + w) * kRows + rr) * 2];
            f[w] = mw == top ? 1.0f : ex2(mw - top);
            sum = fmaf(f[w], stats[((first_warp + w) * kRows + rr) * 2 + 1], sum);
          }
        }
        if (rr < rows_here) {
          const int tok = (row0 + rr) / a.group, sub = (row0 + rr) - tok * a.group;
          const float inv = sum != 0.0f ? 1.0f / sum : 0.0f;  // a row that sees no key is zero
          uint16_t* dst = static_cast<uint16_t*>(a.out) + (int64_t)(rq.q0 + tok) * a.osn +
                          ((int64_t)head * a.group + sub) * a.osh;
          for (int jj = 0; jj < tiles_here; ++jj) {
            const int j = sub_warp * tiles_here + jj;
            float v0 = 0.0f, v1 = 0.0f;
#pragma unroll
            for (int w = 0; w < kAttnWarps; ++w)
              if (w < head_warps) {
                const float* src = merge + (((first_warp + w) * kMt + j) * NT + nt) * 128 + c * 32 + lane;
                v0 = fmaf(f[w], src[0], v0);
                v1 = fmaf(f[w], src[64], v1);
              }
            const int d = 32 * (j >> 1) + 4 * g + 2 * (j & 1);
            if (starts && ends) {
              dst[d] = Elem<T>::from_f(v0 * inv);
              dst[d + 1] = Elem<T>::from_f(v1 * inv);
            } else {
              *reinterpret_cast<float2*>(part + rr * D + d) = make_float2(v0, v1);
            }
          }
          if (sub_warp == 0 && g == 0) {
            if (starts && ends) {
              if (a.lse != nullptr)
                a.lse[(int64_t)(rq.q0 + tok) * a.kv.heads * a.group + (int64_t)head * a.group + sub] =
                    sum != 0.0f ? top + __log2f(sum) : -INFINITY;
            } else {
              part[kRows * D + 2 * rr] = top;
              part[kRows * D + 2 * rr + 1] = sum;
            }
          }
        }
      }
    if (starts && !ends) {
      // The tile goes on in the following CTAs, up to the one that holds its last unit.
      const int64_t last = (at + rq.units - 1) / share;
      desc_parts = (int)(last - blockIdx.x) + 1;
      desc_q0 = rq.q0;
      desc_qlen = rq.qlen;
      desc_row = row0;
      desc_head = head_group * cta_heads;
    }
    __syncthreads();  // merge and the queries may be overwritten

    at += seg_units;
    unit += seg_units;
    if (unit == rq.units && at < end) {
      unit = -kAttnLead;
      if (++head_group == head_groups) {
        head_group = 0;
        if (++tile == rq.tiles) {
          tile = 0;
          do rq = attn_request<kRows>(a, ++b, nullptr); while (rq.tiles == 0);  // at < end: there is one
        }
      }
    }
  }
  if (tid == 0 && a.desc != nullptr) {
    desc[0] = desc_parts;
    desc[1] = desc_q0;
    desc[2] = desc_qlen;
    desc[3] = desc_row;
    desc[4] = desc_head;
  }
  pdl_launch_dependents();
}

// Joins the parts of the tiles that were split: CTAs (c, y) take the (head, row) pairs of the tile that the
// main kernel's CTA c started, a warp each, in the order of the parts.
template <typename T, int D, int kRows>
__global__ void __launch_bounds__(kAttnThreads) attn_int4_join_kernel(const AttnInt4Args a) {
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int32_t* desc = a.desc + (int64_t)blockIdx.x * kAttnDescInts;
  const int parts = desc[0];
  for (int hr = blockIdx.y * kAttnWarps + (threadIdx.x >> 5); parts > 0 && hr < a.cta_heads * kRows; hr += gridDim.y * kAttnWarps) {
    const int which = hr / kRows, r = hr % kRows;
    const int q0 = desc[1], row = desc[3] + r, head = desc[4] + which;
    if (row < desc[2] * a.group) {
      constexpr int kPer = D / 32;
      const int64_t slot = (int64_t)a.cta_heads * attn_part_floats(D, kRows);
      // part 0 is slot 1 of CTA c, part i slot 0 of CTA c + i
      const float* rest = a.part + blockIdx.x * 2 * slot + which * attn_part_floats(D, kRows);
      const float* first = rest + slot;
      float top = -INFINITY;
      for (int i = lane; i < parts; i += 32)
        top = fmaxf(top, (i == 0 ? first : rest + i * 2 * slot)[kRows * D + 2 * r]);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      float sum = 0.0f, acc[kPer];
#pragma unroll
      for (int j = 0; j < kPer; ++j) acc[j] = 0.0f;
#pragma unroll 4
      for (int i = 0; i < parts; ++i) {
        const float* p = i == 0 ? first : rest + i * 2 * slot;
        const float m = p[kRows * D + 2 * r], l = p[kRows * D + 2 * r + 1];
        // l by the root twice: beside a reference far below (a prompt part of next to no scales) it may be as far above 1.
        const float root = m == top ? 1.0f : ex2(0.5f * (m - top)), f = root * root;
        sum = fmaf(l * root, root, sum);
#pragma unroll
        for (int j = 0; j < kPer; ++j) acc[j] = fmaf(f, p[r * D + j * 32 + lane], acc[j]);
      }
      const int tok = row / a.group, sub = row - tok * a.group;
      const float inv = sum != 0.0f ? 1.0f / sum : 0.0f;
      uint16_t* dst = static_cast<uint16_t*>(a.out) + (int64_t)(q0 + tok) * a.osn +
                      ((int64_t)head * a.group + sub) * a.osh;
#pragma unroll
      for (int j = 0; j < kPer; ++j) dst[j * 32 + lane] = Elem<T>::from_f(acc[j] * inv);
      if (lane == 0 && a.lse != nullptr)
        a.lse[(int64_t)(q0 + tok) * a.kv.heads * a.group + (int64_t)head * a.group + sub] =
            sum != 0.0f ? top + __log2f(sum) : -INFINITY;
    }
  }
  pdl_launch_dependents();
}

}  // namespace mas
