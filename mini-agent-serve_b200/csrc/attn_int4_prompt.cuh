// attn_int4_prompt.cuh -- attention of many query rows a request (prompt chunks) over the 4-bit paged KV cache, on the
// fifth-generation tensor cores (sm_100a).
//
// The same mathematics as attn_int4.cuh, with another bound: a request's rows (tokens x group) outnumber what a key
// brings in, so the products decide, 4 * D flops a row and key, and each key is unpacked once for 256 rows. Here, too, the products
// run on bare codes (c - 8 in fp16, exact) and the pairs enter in fp32, between them:
//   y = S' ks + (sum q) kb,  p = 2^(y - M),  l += p,  r += p (mv + 8 sv),  w = fp16(p sv),  O += w (cv - 8),  o = (O + r) / l
// (ks, kb the key's scale and minimum + 8 scales; the row's scale holds the softmax scale and log2 e). M is one reference for all: the row's
// largest log2 of a p g, moved when one passes it by 8. g is what a key may add to a sum: its scale, or its minimum (+ 8 scales) over 2^60,
// or 2^-96. So weights stay within fp16, r within 2^68 a key whatever the values are (a constant row's scale is 2^-126), l within 2^104,
// and scales down to 2^-110, or to 2^-74 of their minimum, keep their weights' bits.
//
// Measured: 911 and 1511 new tokens of 6 K (96/8 heads of 128) take 1290 us against a floor of 393
// (products); 1385 with the items dealt to the SMs whole. What bounds it is the softmax warps, two a scheduler, which issue in 36 % of the cycles: of the 1385, their arithmetic is 636 us, exponentials alone 91,
// factor loads 172. Sixteen softmax warps of half a row a thread took 1798 (104 registers spill), two S buffers of 64 keys a
// tile 15 % more than this. Keys and values rounded to bf16 on the way in, two instructions less a (row, key), took 924, but were
// 0.0051 of the result off where this is 0.0017.
//
// A CTA takes 256 rows of one kv head (two tiles of 128, the height of an MMA) and walks the keys in steps of 128:
//   warps 8-15   unpack a step's codes into shared memory, a thread a key: K [key][D] (8-11) and V [key][D] (12-15), 128-byte
//                rows of 64 elements, 16-byte chunks exchanged by the row's last three bits (the 128-byte swizzle), two stages
//   warps 0-7    softmax, a thread a row, 64 keys of a step at a time: S from tensor memory, the logits y and their maximum, the
//                weights, over the first half of S as 16-bit pairs; while one tile's rows are at it the other tile's products
//                run. A thread of each tile's first warp issues them: S = Q K^T (both operands from shared
//                memory, K-major), then O += P V (P from tensor memory, V from shared memory, MN-major)
// Tensor memory: S0 S1 O0 O1, 128 fp32 columns each, all 512. When M moves, the thread rescales its row of O, which no
// product touches between the two barriers it stands between. The keys' and values' factors travel through shared memory, four
// steps deep: a step's are overwritten four steps on, when the products of two steps on, which followed its rows' softmax, are done.
// Every wait is bounded; one that runs out sets the fault word and all roles leave.
#pragma once

#include <math_constants.h>

#include <type_traits>

#include "attn_int4.cuh"
#include "common.cuh"

namespace mas {

constexpr int kPromptThreads = 512;
// Registers of the roles: 8 warps x 168 + 8 warps x 88 = 16 warps x 128, what the block is launched with (on every quarter of
// the SM, too).
constexpr int kPromptSoftmaxRegs = 168, kPromptUnpackRegs = 88;
constexpr int kPromptRows = 256;  // rows of a CTA's item
constexpr int kPromptKeys = 128;  // keys of a step
// Requests with more rows a kv head go to this kernel, in calls with enough rows (over all heads) an SM to pay for the launches.
// This kernel / tiles of 16 rows, us, 96/8 heads of 128 (32/8: within 7 %), over contexts of 600, 4 K and 15 K tokens:
//   requests x rows a kv head    rows an SM        600            4 K             15 K
//   1 x 504                          27          53 /  27       66 /  59       113 /  153
//   4 x 132                          29          45 /  27       71 /  62       148 /  170
//   4 x 240                          52          52 /  35       83 /  91       164 /  271
//   4 x 504                         109          64 /  53      114 / 169       276 /  551
//   16 x 132                        114          49 /  59      167 / 189       492 /  624
//   16 x 240                        208          53 /  85      186 / 303       508 / 1025
// 64 rows an SM lies between the break-even over 4 K tokens and that over 600. What a rule on rows gives away is at the other lengths: up to
// 1.65 times below it over 15 K, 1.2 times above it over 600. (The lengths are the device's; the host knows the tables' width, a bound.)
// Rows a kv head, 16 requests over 4 K tokens: 72 rows 131 / 116 and 96 rows 151 / 136 with the items whole, 100 rows (32/8 heads) 134 / 151 with
// the shares equal. A call with many rows and no such request pays 6 to 9 us for nothing.
constexpr int kAttnSplitRows = 96, kPromptRowsPerSm = 64;
constexpr int kPromptJoinCtas = 16;  // a CTA's item in the joining kernel (64 cost an empty launch 10 us more)

template <int D>
struct PromptShape {
  static constexpr int kTile = 128 * D * 2;  // bytes of a 128-row operand
  static constexpr int kQ = 0;               // two tiles
  static constexpr int kK = 2 * kTile;       // two stages
  static constexpr int kV = 4 * kTile;       // two stages
  static constexpr int kKeyFactors = 6 * kTile;              // [4][64 pairs of keys] {ks, ks, kb, kb}
  static constexpr int kValueFactors = kKeyFactors + 4096;   // [4][64 pairs of keys] {sv, sv, mv + 8 sv, mv + 8 sv}
  static constexpr int kLogs = kValueFactors + 4096;         // [4][128] log2 g
  static constexpr int kSpread = kLogs + 2048;               // [4][4 warps] {largest, smallest log2 g}
  static constexpr int kBars = kSpread + 128;
  static constexpr int kSmem = kBars + 256 + 1024;  // the operands are aligned to 1024 bytes by hand
};

enum PromptBar { kKFull = 0, kKEmpty = 2, kVFull = 4, kVEmpty = 6, kSFull = 8, kPFull = 10, kQFull = 12, kOFull = 14, kKeyFac = 16, kValueFac = 20,
                 kDrain = 24, kPromptBars = 26 };
// The keys' pairs are taken at 2^-16, exact for any bf16 scale, so that a logit's terms, of 128 elements of up to 2^9 each, stay
// below twice the key's size; the row's scale gives it back.
constexpr float kPromptSumUnit = 1.52587891e-5f;
// Up to this spread of log2 g in a step, the largest stands for all in the choice of M.
constexpr float kPromptSpread = 10.0f;

// Shared-memory operand descriptor, 128-byte swizzle. K-major: rows of 128 bytes, groups of eight rows `sbo` bytes apart.
// MN-major: `lbo` bytes between blocks of 64 elements of the long axis, `sbo` between groups of eight of the other.
__device__ __forceinline__ uint64_t umma_desc(uint32_t addr, uint32_t lbo, uint32_t sbo) {
  return (uint64_t)((addr & 0x3ffffu) >> 4) | ((uint64_t)(lbo >> 4) << 16) | ((uint64_t)(sbo >> 4) << 32) | (1ull << 46) |
         (2ull << 61);
}
// Instruction descriptor of kind::f16: fp32 accumulators, both operands fp16.
__device__ __forceinline__ constexpr uint32_t umma_idesc(int m, int n, bool b_mn_major) {
  return (1u << 4) | ((b_mn_major ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}
__device__ __forceinline__ void umma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)accumulate)
      : "memory");
}
__device__ __forceinline__ void umma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"((uint32_t)accumulate)
      : "memory");
}
// Arrives on `bar` once every product issued by this thread so far has completed.
__device__ __forceinline__ void umma_commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void tmem_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tmem_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// 32 columns of this thread's lane; the wait is part of the statement, so that nothing uses the registers before it.
__device__ __forceinline__ void tmem_ld32(uint32_t (&r)[32], uint32_t addr) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, "
      "%18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]),
        "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]),
        "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(addr));
}
// 64 columns of this thread's lane; the wait is part of the statement, so that nothing uses the registers before it.
__device__ __forceinline__ void tmem_ld64(uint32_t (&r)[64], uint32_t addr) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x64.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, "
      "%32, %33, %34, %35, %36, %37, %38, %39, %40, %41, %42, %43, %44, %45, %46, %47, "
      "%48, %49, %50, %51, %52, %53, %54, %55, %56, %57, %58, %59, %60, %61, %62, %63}, [%64];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31]), "=r"(r[32]),
        "=r"(r[33]), "=r"(r[34]), "=r"(r[35]), "=r"(r[36]), "=r"(r[37]), "=r"(r[38]), "=r"(r[39]), "=r"(r[40]),
        "=r"(r[41]), "=r"(r[42]), "=r"(r[43]), "=r"(r[44]), "=r"(r[45]), "=r"(r[46]), "=r"(r[47]), "=r"(r[48]),
        "=r"(r[49]), "=r"(r[50]), "=r"(r[51]), "=r"(r[52]), "=r"(r[53]), "=r"(r[54]), "=r"(r[55]), "=r"(r[56]),
        "=r"(r[57]), "=r"(r[58]), "=r"(r[59]), "=r"(r[60]), "=r"(r[61]), "=r"(r[62]), "=r"(r[63])
      : "r"(addr));
}
__device__ __forceinline__ void tmem_st32(uint32_t addr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, "
      "%18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(addr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
      "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]),
      "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]),
      "r"(r[31])
      : "memory");
}

// (w & mask) | magic in one instruction.
__device__ __forceinline__ uint32_t and_or(uint32_t w, uint32_t mask, uint32_t magic) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(w), "r"(mask), "r"(magic));
  return r;
}

// One key's codes into its row of a 128-row operand as fp16 c - 8, each eight elements in the order 0 4 1 5 2 6 3 7 they
// unpack in (the queries and the results take the same one): 1024 + c and 1024 + 16 c are exact, and so is what follows.
template <int D>
__device__ __forceinline__ void unpack_row(uint32_t base, int row, const uint32_t (&w)[D / 8]) {
  const __half2 off = __float2half2_rn(1032.0f), sixteenth = __float2half2_rn(0.0625f), off16 = __float2half2_rn(-72.0f);
#pragma unroll
  for (int c = 0; c < D / 8; ++c) {
    uint32_t v[4];  // pairs (0, 4), (1, 5), (2, 6), (3, 7)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      uint32_t lo = and_or(w[c] >> (8 * i), 0x000f000fu, 0x64006400u), hi = and_or(w[c] >> (8 * i), 0x00f000f0u, 0x64006400u);
      const __half2 x = __hsub2(*reinterpret_cast<__half2*>(&lo), off);
      const __half2 y = __hfma2(*reinterpret_cast<__half2*>(&hi), sixteenth, off16);
      v[2 * i] = *reinterpret_cast<const uint32_t*>(&x);
      v[2 * i + 1] = *reinterpret_cast<const uint32_t*>(&y);
    }
    const uint32_t dst = base + (c >> 3) * 16384 + row * 128 + (((c & 7) ^ (row & 7)) << 4);
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]) : "memory");
  }
}

// What starting on an item costs (its queries, the first loads' latency), in steps (0, 1, 4 instead: 1295, 1295, 1288 us where 2 took
// 1292), and the least share: one step past that (132 rows over 600 tokens: 47 us, 53 with 4, 70 with 8).
constexpr int kPromptLead = 2, kPromptMinShare = 3;

// A stretch of the line of work: steps u0 .. u1 of an item, 256 rows of one kv head of one request.
struct PromptItem {
  AttnRequest rq;
  int32_t b, head, block;  // the block of rows
  int32_t row0, rows, u0, u1;
  int32_t starts, ends;    // the item's first, last step is in it
};

// Steps of 128 keys that a block of rows sees.
__device__ __forceinline__ int prompt_steps(const AttnInt4Args& a, const AttnRequest& rq, int block) {
  const int rows = min((block + 1) * kPromptRows, rq.qlen * a.group);
  const int seen = a.causal ? min(rq.n, max(0, rq.n - rq.qlen + (rows - 1) / a.group + 1)) : rq.n;
  return (seen + kPromptKeys - 1) / kPromptKeys;
}
__device__ __forceinline__ int prompt_blocks(const AttnInt4Args& a, const AttnRequest& rq) {
  const int64_t rows = (int64_t)rq.qlen * a.group;
  return rows > a.split_rows ? (int)((rows + kPromptRows - 1) / kPromptRows) : 0;
}
// A kv head's work of a request: of each block its steps, at least one, and the lead.
__device__ __forceinline__ int64_t prompt_work(const AttnInt4Args& a, const AttnRequest& rq) {
  int64_t work = 0;
  for (int k = prompt_blocks(a, rq) - 1; k >= 0; --k) work += max(1, prompt_steps(a, rq, k)) + kPromptLead;
  return work;
}

template <typename T, int D>
__global__ void __launch_bounds__(kPromptThreads, 1) attn_int4_prompt_kernel(const AttnInt4Args a, int32_t* fault) {
  using Sh = PromptShape<D>;
  extern __shared__ uint8_t raw[];
  __shared__ uint32_t s_tmem;
  __shared__ volatile int s_stop;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t base = (smem_u32(raw) + 1023u) & ~1023u;
  uint8_t* shared = raw + (base - smem_u32(raw));
  uint64_t* bars = reinterpret_cast<uint64_t*>(shared + Sh::kBars);
  __shared__ int64_t s_scan[kPromptThreads / 32];
  __shared__ PromptItem s_item;
  __shared__ int s_unit;
  pdl_wait();
  // The items, requests outermost, then heads, then row blocks (the last rows, which see the most keys under a causal mask, first),
  // form one line of steps that the CTAs cut into equal shares. Total and place by a block scan over the requests.
  const int heads = a.kv.heads;
  int32_t* desc = a.desc + (int64_t)blockIdx.x * kAttnDescInts;
  const int per = (a.B + kPromptThreads - 1) / kPromptThreads;
  const int rb0 = min(a.B, tid * per), rb1 = min(a.B, rb0 + per);
  int64_t mine = 0;
  for (int b = rb0; b < rb1; ++b) mine += prompt_work(a, attn_request<8>(a, b, nullptr, false)) * heads;
  int64_t incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t y = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += y;
  }
  if (lane == 31) s_scan[warp] = incl;
  __syncthreads();
  int64_t total = 0, before = incl - mine;
  for (int w = 0; w < kPromptThreads / 32; ++w) {
    if (w < warp) before += s_scan[w];
    total += s_scan[w];
  }
  const int64_t share = max((total + gridDim.x - 1) / gridDim.x, (int64_t)kPromptMinShare);
  int64_t at = (int64_t)blockIdx.x * share;
  const int64_t end = min(at + share, total);
  if (at >= end) {  // nothing for this CTA
    if (tid == 0) desc[0] = 0;
    pdl_launch_dependents();
    return;
  }
  if (at >= before && at < before + mine) {
    int64_t rem = at - before;
    PromptItem x;
    for (x.b = rb0;; ++x.b) {
      x.rq = attn_request<8>(a, x.b, nullptr, false);
      const int64_t w = prompt_work(a, x.rq);
      if (rem < w * heads) {
        x.head = (int)(rem / w);
        rem %= w;
        break;
      }
      rem -= w * heads;
    }
    for (x.block = prompt_blocks(a, x.rq) - 1;; --x.block) {
      const int w = max(1, prompt_steps(a, x.rq, x.block)) + kPromptLead;
      if (rem < w) break;
      rem -= w;
    }
    s_item = x;
    s_unit = (int)rem - kPromptLead;  // below 0: the start's cost
  }
  __syncthreads();
  PromptItem it = s_item;
  int unit = s_unit;
  int32_t parts = 0, part_q0 = 0, part_qlen = 0, part_row = 0, part_head = 0;  // of an item that goes on in the next CTA
  // The next stretch of this share, into `it`; every warp walks the share for itself.
  auto next_item = [&]() {
    if (at >= end) return false;
    int steps = prompt_steps(a, it.rq, it.block), units = max(1, steps);
    if (unit == units) {
      unit = -kPromptLead;
      if (--it.block < 0) {
        if (++it.head == heads) {
          it.head = 0;
          do it.rq = attn_request<8>(a, ++it.b, nullptr, false); while (prompt_blocks(a, it.rq) == 0);  // at < end: there is one
        }
        it.block = prompt_blocks(a, it.rq) - 1;
      }
      steps = prompt_steps(a, it.rq, it.block);
      units = max(1, steps);
    }
    const int lead = (int)min((int64_t)max(-unit, 0), end - at);
    at += lead;
    unit += lead;
    if (at == end) return false;
    const int take = (int)min((int64_t)(units - unit), end - at);
    it.row0 = it.block * kPromptRows;
    it.rows = min(kPromptRows, it.rq.qlen * a.group - it.row0);
    it.u0 = min(unit, steps);
    it.u1 = min(unit + take, steps);
    it.starts = unit == 0;
    it.ends = unit + take == units;
    if (it.starts && !it.ends) {
      parts = (int)((at + units - 1) / share - blockIdx.x) + 1;
      part_q0 = it.rq.q0;
      part_qlen = it.rq.qlen;
      part_row = it.row0;
      part_head = it.head;
    }
    at += take;
    unit += take;
    return true;
  };

  if (tid == 0) {
    s_stop = 0;
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bars[kKFull + i], 128);
      mbar_init(&bars[kKEmpty + i], 2);  // each tile's products
      mbar_init(&bars[kVFull + i], 128);
      mbar_init(&bars[kVEmpty + i], 2);
      mbar_init(&bars[kSFull + i], 1);
      mbar_init(&bars[kPFull + i], 128);
      mbar_init(&bars[kQFull + i], 128);
      mbar_init(&bars[kOFull + i], 1);
      mbar_init(&bars[kDrain + i], 1);
    }
    for (int i = 0; i < 4; ++i) {
      mbar_init(&bars[kKeyFac + i], 128);
      mbar_init(&bars[kValueFac + i], 128);
    }
    fence_barrier_init();
  }
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&s_tmem)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    tmem_fence_before();
  }
  __syncthreads();
  tmem_fence_after();
  const uint32_t tmem = s_tmem;

  // A wait that gives up (or finds that another has) ends its role; true means go on.
  auto wait = [&](int bar, uint32_t parity) {
    if (mbar_try_wait(&bars[bar], parity)) return true;
    const uint64_t t0 = global_timer_ns();
    for (uint32_t polls = 1; polls < kWaitMaxPolls; ++polls) {
      if (mbar_try_wait(&bars[bar], parity)) return true;
      if ((polls & 255u) == 0u && (s_stop || global_timer_ns() - t0 > kWaitLimitNs)) break;
    }
    s_stop = 1;
    flag_status(fault, MAS_STATUS_COPY_TIMEOUT);
    return false;
  };

  if (warp < 8) {
    // ---------------- softmax: thread = row ----------------
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kPromptSoftmaxRegs));
    const int tile = warp >> 2, r = tid & 127;
    const uint32_t row_sel = (uint32_t)(warp & 3) << 21;  // this warp's 32 lanes of tensor memory
    const uint32_t s_addr = tmem + row_sel + tile * 128, o_addr = tmem + row_sel + 256 + tile * 128;
    // Columns from `left` on are hidden from the row.
    auto hide = [&](uint32_t (&s)[64], int left) {
#pragma unroll
      for (int i = 0; i < 64; ++i) s[i] = i < left ? s[i] : 0xff800000u;
    };
    // Products, by one thread a tile. Step d (of all items) uses stage d & 1.
    constexpr uint32_t kIdescS = umma_idesc(128, kPromptKeys, false), kIdescO = umma_idesc(128, D, true);
    const bool issuer = lane == 0 && (warp & 3) == 0;
    auto issue_scores = [&](uint32_t d) {
      const int stage = d & 1;
      if (!wait(kKFull + stage, (d >> 1) & 1)) return;
      tmem_fence_after();
      const uint32_t q = base + Sh::kQ + tile * Sh::kTile, k = base + Sh::kK + stage * Sh::kTile;
#pragma unroll
      for (int x = 0; x < D / 16; ++x) {
        const uint32_t off = (x >> 2) * 16384 + (x & 3) * 32;  // 16 elements of D
        umma_ss(tmem + tile * 128, umma_desc(q + off, 16, 1024), umma_desc(k + off, 16, 1024), kIdescS, x > 0);
      }
      umma_commit(&bars[kSFull + tile]);
      umma_commit(&bars[kKEmpty + stage]);
    };
    auto issue_values = [&](uint32_t d, bool accumulate) {
      const int stage = d & 1;
      if (!wait(kVFull + stage, (d >> 1) & 1)) return;
      tmem_fence_after();
#pragma unroll
      for (int x = 0; x < kPromptKeys / 16; ++x)
        umma_ts(tmem + 256 + tile * 128, tmem + tile * 128 + x * 8,
                umma_desc(base + Sh::kV + stage * Sh::kTile + x * 2048, 16384, 1024), kIdescO, accumulate || x > 0);
      umma_commit(&bars[kVEmpty + stage]);
    };
    uint32_t s_phase = 0, o_phase = 0, p_phase = 0, q_phase = 0;
    uint32_t done = 0;  // steps so far, over all items, this tile's rows at work or not
    bool go = true;
    while (go && next_item()) {
      if (tile * 128 >= it.rows) {
        // No rows: the tile still takes and gives back each stage, or it would meet the next item's barriers phases early.
        for (int j = 0; issuer && j < it.u1 - it.u0; ++j) {
          const int stage = (done + j) & 1;
          const uint32_t parity = ((done + j) >> 1) & 1;
          if (!wait(kKFull + stage, parity)) break;
          mbar_arrive(&bars[kKEmpty + stage]);
          if (!wait(kVFull + stage, parity)) break;
          mbar_arrive(&bars[kVEmpty + stage]);
        }
        __syncwarp();
        done += it.u1 - it.u0;
        continue;
      }
      const int row = it.row0 + tile * 128 + r;
      const bool here = tile * 128 + r < it.rows;
      const int tok = (it.row0 + min(tile * 128 + r, it.rows - 1)) / a.group;
      const int sub = row - tok * a.group;
      const int lim = a.causal ? min(it.rq.n, max(0, it.rq.n - it.rq.qlen + tok + 1)) : it.rq.n;
      float qsum = 0.0f, unscale = 0.0f;
      if (it.u1 > it.u0) {
        // The row as fp16, a bf16 one scaled by a power of two to a largest element of 2^8 to 2^9 (8 bits down to 2^-22 of that
        // largest, to within 2^-33 of it below): its sums stay next to a key's size (see kPromptSumUnit).
        const uint16_t* src = static_cast<const uint16_t*>(a.q) + (int64_t)(it.rq.q0 + tok) * a.qsn +
                              ((int64_t)it.head * a.group + (here ? sub : 0)) * a.qsh;
        float scale = 1.0f, power = 1.0f;
        if (std::is_same<T, __nv_bfloat16>::value) {
          uint32_t most = 0;
#pragma unroll 4
          for (int c = 0; c < D / 8; ++c) {
            float f[8];
            unpack8<T>(a.q_vec ? kv_load8<true>(src + 8 * c) : kv_load8<false>(src + 8 * c), f);
#pragma unroll
            for (int x = 0; x < 8; ++x) most = max(most, __float_as_uint(fabsf(f[x])));
          }
          const uint32_t exponent = min(max(most >> 23, 12u), 254u);
          scale = __uint_as_float((262u - exponent) << 23);
          power = __uint_as_float((exponent - 8u) << 23);
        }
        unscale = row_unscale(power, a.row_scale * (1.0f / kPromptSumUnit));
#pragma unroll 4
        for (int c = 0; c < D / 8; ++c) {
          float f[8];
          unpack8<T>(a.q_vec ? kv_load8<true>(src + 8 * c) : kv_load8<false>(src + 8 * c), f);
#pragma unroll
          for (int x = 0; x < 8; ++x) {
            f[x] = here ? f[x] * scale : 0.0f;
            qsum += f[x];
          }
          const uint32_t dst = base + Sh::kQ + tile * Sh::kTile + (c >> 3) * 16384 + r * 128 + (((c & 7) ^ (r & 7)) << 4);
          asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst), "r"(Elem<__half>::from_f2(f[0], f[4])),
                       "r"(Elem<__half>::from_f2(f[1], f[5])), "r"(Elem<__half>::from_f2(f[2], f[6])),
                       "r"(Elem<__half>::from_f2(f[3], f[7]))
                       : "memory");
        }
        fence_proxy_async_smem();
        mbar_arrive(&bars[kQFull + tile]);
        if (issuer && wait(kQFull + tile, q_phase)) issue_scores(done);
        __syncwarp();
        q_phase ^= 1;
      }
      float m = -INFINITY, l = 0.0f;
      float2 r2 = both(0.0f);
      for (int j = it.u0; go && j < it.u1; ++j, ++done) {
        const int buf = done & 3;
        const uint32_t parity = (done >> 2) & 1;
        go = wait(kSFull + tile, s_phase) && wait(kKeyFac + buf, parity) && wait(kValueFac + buf, parity);
        s_phase ^= 1;
        if (!__all_sync(0xffffffffu, go)) {
          go = false;
          break;
        }
        tmem_fence_after();
        const int left = lim - j * kPromptKeys;  // keys of this step that the row sees
        const bool edge = __any_sync(0xffffffffu, left < kPromptKeys);
        const uint32_t kf = base + Sh::kKeyFactors + buf * 1024, vf = base + Sh::kValueFactors + buf * 1024;
        float lv_max = -INFINITY, lv_min = INFINITY;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 x = lds_float2(base + Sh::kSpread + buf * 32 + i * 8);
          lv_max = fmaxf(lv_max, x.x);
          lv_min = fminf(lv_min, x.y);
        }
        const bool alike = lv_max - lv_min <= kPromptSpread;
        // 64 keys at a time: logits, the reference, weights.
#pragma unroll 1
        for (int c = 0; c < 2; ++c) {
          uint32_t s[64];
          tmem_ld64(s, s_addr + c * 64);
#pragma unroll
          for (int i = 0; i < 64; i += 2) {
            const uint4 f = lds128(kf + (c * 64 + i) * 8);
            const float2 y = fma2_f32(make_float2(__uint_as_float(s[i]), __uint_as_float(s[i + 1])),
                                      make_float2(__uint_as_float(f.x), __uint_as_float(f.y)),
                                      mul2_f32(both(qsum), make_float2(__uint_as_float(f.z), __uint_as_float(f.w))));
            s[i] = __float_as_uint(y.x);
            s[i + 1] = __float_as_uint(y.y);
          }
          if (edge) hide(s, left - c * 64);
          float t0 = -INFINITY, t1 = -INFINITY;
#pragma unroll
          for (int i = 0; i < 64; i += 4) {
            t0 = fmaxf(t0, fmaxf(__uint_as_float(s[i]), __uint_as_float(s[i + 1])));
            t1 = fmaxf(t1, fmaxf(__uint_as_float(s[i + 2]), __uint_as_float(s[i + 3])));
          }
          const float top = fmaxf(t0, t1) * unscale;
          // The largest p g's log2: the largest logit and the largest g where the g are alike, each key's own where they are
          // not (a hidden key's must not set the reference of rows that do not see it).
          float cand = top + lv_max;
          if (!alike) {
            cand = -INFINITY;
#pragma unroll
            for (int i = 0; i < 64; i += 2) {
              const float2 lv = lds_float2(base + Sh::kLogs + buf * 512 + (c * 64 + i) * 4);
              cand = fmaxf(cand, fmaxf(fmaf(__uint_as_float(s[i]), unscale, lv.x), fmaf(__uint_as_float(s[i + 1]), unscale, lv.y)));
            }
          }
          const bool up = cand > m + 8.0f;
          if (__any_sync(0xffffffffu, up)) {
            const float was = m;
            m = up ? cand : m;
            const float factor = was == m || was == -INFINITY ? 1.0f : ex2(was - m);  // before its first key the row of O is zeros
            if (j > it.u0) {
#pragma unroll 1
              for (int d = 0; d < D / 32; ++d) {
                uint32_t o[32];
                tmem_ld32(o, o_addr + d * 32);
#pragma unroll
                for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * factor);
                tmem_st32(o_addr + d * 32, o);
              }
            }
            if (c > 0) {  // the first half's weights are relative to the old reference: rounded to 11 bits a second time
              uint32_t w[32];
              tmem_ld32(w, s_addr);
              const __half2 by = __float2half2_rn(factor);
#pragma unroll
              for (int i = 0; i < 32; ++i) {
                const __half2 x = __hmul2(*reinterpret_cast<__half2*>(&w[i]), by);
                w[i] = *reinterpret_cast<const uint32_t*>(&x);
              }
              tmem_st32(s_addr, w);
            }
            // M may rise by more than fp32's exponents while l, of up to 2^104 a key, still counts: by its root, twice.
            const float root = was == m || was == -INFINITY ? 1.0f : ex2(0.5f * (was - m));
            l = l * root * root;
            r2.x *= factor;
            r2.y *= factor;
          }
          const float ref = m == -INFINITY ? 0.0f : -m;
          float2 part = both(0.0f);
          uint32_t w[32];
#pragma unroll
          for (int i = 0; i < 64; i += 2) {
            const uint4 f = lds128(vf + (c * 64 + i) * 8);
            const float2 x = fma2_f32(make_float2(__uint_as_float(s[i]), __uint_as_float(s[i + 1])), both(unscale), both(ref));
            const float2 p = make_float2(ex2(x.x), ex2(x.y));
            part = add2_f32(part, p);
            r2 = fma2_f32(p, make_float2(__uint_as_float(f.z), __uint_as_float(f.w)), r2);
            const float2 v = mul2_f32(p, make_float2(__uint_as_float(f.x), __uint_as_float(f.y)));
            w[i / 2] = Elem<__half>::from_f2(v.x, v.y);
          }
          tmem_st32(s_addr + c * 32, w);  // columns that this thread has read
          l += part.x + part.y;
        }
        tmem_wait_st();
        tmem_fence_before();
        mbar_arrive(&bars[kPFull + tile]);
        if (issuer && wait(kPFull + tile, p_phase)) {
          issue_values(done, j > it.u0);
          if (j + 1 < it.u1) issue_scores(done + 1);
          else umma_commit(&bars[kOFull + tile]);
        }
        __syncwarp();
        p_phase ^= 1;
      }
      if (!go) break;
      if (it.u1 > it.u0) {
        go = wait(kOFull + tile, o_phase);
        o_phase ^= 1;
        if (!__all_sync(0xffffffffu, go)) {
          go = false;
          break;
        }
        tmem_fence_after();
      }
      const bool whole = it.starts && it.ends;
      const float inv = whole ? (l != 0.0f ? 1.0f / l : 0.0f) : 1.0f, rest = r2.x + r2.y;
      float* part = a.part + ((int64_t)blockIdx.x * 2 + (it.starts && !it.ends ? 1 : 0)) * attn_part_floats(D, kPromptRows);
      float* part_row_at = part + (tile * 128 + r) * D;
      uint16_t* dst = static_cast<uint16_t*>(a.out) + (int64_t)(it.rq.q0 + tok) * a.osn +
                      ((int64_t)it.head * a.group + sub) * a.osh;
#pragma unroll 1
      for (int c = 0; c < D / 32; ++c) {
        uint32_t o[32];
        if (it.u1 > it.u0) tmem_ld32(o, o_addr + c * 32);
#pragma unroll
        for (int i = 0; i < 32; i += 8) {
          float f[8];
#pragma unroll
          for (int x = 0; x < 8; ++x) f[x] = l != 0.0f ? (__uint_as_float(o[i + (x < 4 ? 2 * x : 2 * x - 7)]) + rest) * inv : 0.0f;
          if (here && !whole) {
            *reinterpret_cast<float4*>(part_row_at + c * 32 + i) = make_float4(f[0], f[1], f[2], f[3]);
            *reinterpret_cast<float4*>(part_row_at + c * 32 + i + 4) = make_float4(f[4], f[5], f[6], f[7]);
          } else if (here) {
            if (a.o_vec) kv_store8<true>(dst + c * 32 + i, pack8<T>(f));
            else kv_store8<false>(dst + c * 32 + i, pack8<T>(f));
          }
        }
      }
      tmem_fence_before();
      if (here && !whole) *reinterpret_cast<float2*>(part + kPromptRows * D + 2 * (tile * 128 + r)) = make_float2(m, l);
      if (here && whole && a.lse != nullptr)
        a.lse[(int64_t)(it.rq.q0 + tok) * heads * a.group + (int64_t)it.head * a.group + sub] =
            l != 0.0f ? m + __log2f(l) : -INFINITY;
    }
    if (!go && issuer) {
      // Products may be in flight over shared and tensor memory: let them end (bounded) before anything is freed.
      umma_commit(&bars[kDrain + tile]);
      (void)mbar_wait_bounded(&bars[kDrain + tile], 0, kWaitLimitNs / 4);
    }
  } else {
    // ---------------- unpacking: thread = key; warps 8-11 the keys, 12-15 the values ----------------
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kPromptUnpackRegs));
    const bool values = warp >= 12;
    const int r = tid & 127;
    const uint8_t* codes = values ? a.kv.v_codes : a.kv.k_codes;
    const uint32_t operand = base + (values ? Sh::kV : Sh::kK);
    const int full = values ? kVFull : kKFull, empty = values ? kVEmpty : kKEmpty;
    constexpr int kVecs = D / 32;  // 16-byte vectors of a row's codes
    uint32_t done = 0;             // steps unpacked so far, over all items
    bool go = true;
    while (go && next_item()) {
      const int32_t* table = a.block_tables + (int64_t)it.b * a.table_stride;
      // The page of this thread's key in step j, -1 past the cache's end and for a bad one.
      auto find = [&](int j) {
        const int tok = j * kPromptKeys + r;
        if (j >= it.u1 || tok >= it.rq.n) return -1;
        const int page = table[a.page_shift >= 0 ? tok >> a.page_shift : tok / (int)a.kv.page_size];
        if (page >= 0 && page < a.kv.num_pages) return page;
        if (!values) flag_status(a.status, MAS_STATUS_KV_SLOT_OUT_OF_RANGE);
        return -1;
      };
      // Its codes and pairs there; zeros without a page.
      auto load = [&](int j, int page, uint32_t (&w)[D / 8], uint2& pair) {
        pair = make_uint2(0, 0);
#pragma unroll
        for (int i = 0; i < D / 8; ++i) w[i] = 0;
        if (page >= 0) {
          const int tok = j * kPromptKeys + r;
          const int entry = a.page_shift >= 0 ? tok & ((1 << a.page_shift) - 1) : tok % (int)a.kv.page_size;
          const int64_t off = page * a.kv.stride_page + entry * a.kv.stride_entry + it.head * a.kv.stride_head;
          pair = *reinterpret_cast<const uint2*>(a.kv.pairs + page * a.kv.pair_stride_page +
                                                 ((int64_t)it.head * a.kv.page_size + entry) * 4);
#pragma unroll
          for (int i = 0; i < kVecs; ++i) {
            const Vec16 x = ld_ro(codes + off + 16 * i);
            w[4 * i] = x.a; w[4 * i + 1] = x.b; w[4 * i + 2] = x.c; w[4 * i + 3] = x.d;
          }
        }
      };
      // The codes of the next step and the page of the one after it are on their way while a step is unpacked.
      uint32_t w[D / 8];
      uint2 pair;
      load(it.u0, find(it.u0), w, pair);
      int page = find(it.u0 + 1);
      for (int j = it.u0; j < it.u1; ++j, ++done) {
        const int stage = done & 1;
        uint32_t w_next[D / 8];
        uint2 pair_next;
        load(j + 1, page, w_next, pair_next);
        page = find(j + 2);
        // The first use of a stage finds it free.
        go = __all_sync(0xffffffffu, wait(empty + stage, ((done >> 1) & 1) ^ 1));
        if (!go) break;
        unpack_row<D>(operand + stage * Sh::kTile, r, w);
        fence_proxy_async_smem();
        mbar_arrive(&bars[full + stage]);
        // A value row that is not finite may be hidden from some rows, whose zero weights would not hide it: its factors
        // are replaced by zeros and its key's by NaNs, which reach exactly the rows that see it.
        const float sv = __uint_as_float(pair.y << 16), mv = __uint_as_float(pair.y & 0xffff0000u);
        const bool bad = !(sv * 0.0f + mv * 0.0f == 0.0f);
        const int buf = done & 3;
        float x, y;
        if (values) {
          x = bad ? 0.0f : sv;
          y = bad ? 0.0f : fmaf(8.0f, sv, mv);
          const float lv = __log2f(fmaxf(fmaxf(x, fabsf(y) * 8.67361738e-19f), 1.26217745e-29f));  // log2 g: 2^-60, 2^-96
          const bool counts = !bad && j * kPromptKeys + r < it.rq.n;
          *reinterpret_cast<float*>(shared + Sh::kLogs + buf * 512 + r * 4) = lv;
          float hi = counts ? lv : -INFINITY, lo = counts ? lv : INFINITY;
#pragma unroll
          for (int z = 16; z > 0; z >>= 1) {
            hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, z));
            lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, z));
          }
          if (lane == 0) *reinterpret_cast<float2*>(shared + Sh::kSpread + buf * 32 + (warp & 3) * 8) = make_float2(hi, lo);
          __syncwarp();
        } else {
          const float sk = __uint_as_float(pair.x << 16), mk = __uint_as_float(pair.x & 0xffff0000u);
          const float unit = a.key_sign * kPromptSumUnit;
          x = bad ? CUDART_NAN_F : sk * unit;
          y = bad ? CUDART_NAN_F : fmaf(8.0f, sk, mk) * unit;
        }
        float* fac = reinterpret_cast<float*>(shared + (values ? Sh::kValueFactors : Sh::kKeyFactors) + buf * 1024 + (r >> 1) * 16);
        fac[r & 1] = x;
        fac[2 + (r & 1)] = y;
        mbar_arrive(&bars[(values ? kValueFac : kKeyFac) + buf]);
#pragma unroll
        for (int i = 0; i < D / 8; ++i) w[i] = w_next[i];
        pair = pair_next;
      }
    }
  }
  __syncwarp();
  tmem_fence_before();
  __syncthreads();
  if (tid == 0) {
    desc[0] = parts;
    desc[1] = part_q0;
    desc[2] = part_qlen;
    desc[3] = part_row;
    desc[4] = part_head;
  }
  if (warp == 0) {
    tmem_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
  }
  pdl_launch_dependents();
}

}  // namespace mas
