// attn_int4_prompt.cuh -- attention of many query rows a request (prompt chunks) over the 4-bit paged KV cache, on the
// fifth-generation tensor cores (sm_100a).
//
// The same mathematics as attn_int4.cuh, with another bound: a request's rows (tokens x group) outnumber what a key
// brings in, so the products decide, 4 * D flops a row and key, and each key is unpacked once for 256 rows. Keys and values
// enter the products as c * s + m rounded once to the queries' type, like a cache held in that type: the pair costs nothing per
// (row, key) then, where it would cost two of the five instructions the softmax spends on one.
//
// A CTA takes 256 rows of one kv head (two tiles of 128, the height of an MMA) and walks the keys in steps of 128:
//   warps 8-15   unpack a step's codes into shared memory, a thread a key: K [key][D] (8-11) and V [key][D] (12-15), 128-byte
//                rows of 64 elements, 16-byte chunks exchanged by the row's last three bits (the 128-byte swizzle), two stages
//   warp 16      one thread issues the products: S = Q K^T (both operands from shared memory, both K-major), then
//                O += P V (P from tensor memory, V from shared memory, MN-major)
//   warps 0-7    softmax, a thread a row: S from tensor memory, P = 2^(S c - m) back over S as 16-bit pairs; while one tile's
//                rows are at it the other tile's products run
// Tensor memory: S0 S1 O0 O1, 128 fp32 columns each, all 512. The reference m moves only when a logit passes it by 8, and
// then the thread rescales its row of O, which no product touches between the two barriers it stands between.
// Every wait is bounded; one that runs out sets the fault word and all roles leave.
#pragma once

#include <type_traits>

#include "attn_int4.cuh"
#include "common.cuh"

namespace mas {

constexpr int kPromptThreads = 544;
// Registers of the roles; 256 x 128 + 256 x 64 + 32 x 56 stay below the 544 x 96 that the block is launched with.
constexpr int kPromptSoftmaxRegs = 128, kPromptUnpackRegs = 64, kPromptIssueRegs = 56;
constexpr int kPromptRows = 256;  // rows of a CTA's item
constexpr int kPromptKeys = 128;  // keys of a step
constexpr int kAttnSplitRows = 64;  // requests with more rows a kv head go to this kernel

template <int D>
struct PromptShape {
  static constexpr int kTile = 128 * D * 2;  // bytes of a 128-row operand
  static constexpr int kQ = 0;               // two tiles
  static constexpr int kK = 2 * kTile;       // two stages
  static constexpr int kV = 4 * kTile;       // two stages
  static constexpr int kBars = 6 * kTile;
  static constexpr int kSmem = kBars + 256 + 1024;  // the operands are aligned to 1024 bytes by hand
};

enum PromptBar { kKFull = 0, kKEmpty = 2, kVFull = 4, kVEmpty = 6, kSFull = 8, kPFull = 10, kQFull = 12, kOFull = 14, kPromptBars = 16 };

// Shared-memory operand descriptor, 128-byte swizzle. K-major: rows of 128 bytes, groups of eight rows `sbo` bytes apart.
// MN-major: `lbo` bytes between blocks of 64 elements of the long axis, `sbo` between groups of eight of the other.
__device__ __forceinline__ uint64_t umma_desc(uint32_t addr, uint32_t lbo, uint32_t sbo) {
  return (uint64_t)((addr & 0x3ffffu) >> 4) | ((uint64_t)(lbo >> 4) << 16) | ((uint64_t)(sbo >> 4) << 32) | (1ull << 46) |
         (2ull << 61);
}
// Instruction descriptor of kind::f16: fp32 accumulators, both operands of one 16-bit type.
template <typename T>
__device__ __forceinline__ constexpr uint32_t umma_idesc(int m, int n, bool b_mn_major) {
  const uint32_t type = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
  return (1u << 4) | (type << 7) | (type << 10) | ((b_mn_major ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) |
         ((uint32_t)(m >> 4) << 24);
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
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(
          addr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
      "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
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

// The codes of one word (elements 8i .. 8i + 7, packed 0-4, 1-5, 2-6, 3-7) as values c * s + m in T, one rounding each.
template <typename T>
struct ValueUnpack;
template <>
struct ValueUnpack<__nv_bfloat16> {
  __nv_bfloat162 s, m;
  __device__ __forceinline__ ValueUnpack(uint32_t pair) {
    const uint32_t ss = __byte_perm(pair, pair, 0x1010), mm = __byte_perm(pair, pair, 0x3232);
    s = *reinterpret_cast<const __nv_bfloat162*>(&ss);
    m = *reinterpret_cast<const __nv_bfloat162*>(&mm);
  }
  __device__ __forceinline__ uint32_t operator()(uint32_t w, int i) const {
    uint32_t u = and_or(w >> (4 * i), 0x000f000fu, 0x43004300u);  // 128 + c
    const __nv_bfloat162 c = __hsub2(*reinterpret_cast<__nv_bfloat162*>(&u), __floats2bfloat162_rn(128.0f, 128.0f));
    const __nv_bfloat162 v = __hfma2(c, s, m);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
};
template <>
struct ValueUnpack<__half> {
  __half2 s, m;
  __device__ __forceinline__ ValueUnpack(uint32_t pair) {
    s = __float2half2_rn(__uint_as_float(pair << 16));
    m = __float2half2_rn(__uint_as_float(pair & 0xffff0000u));
  }
  __device__ __forceinline__ uint32_t operator()(uint32_t w, int i) const {
    uint32_t u = and_or(w >> (4 * i), 0x000f000fu, 0x64006400u);  // 1024 + c
    const __half2 c = __hsub2(*reinterpret_cast<__half2*>(&u), __float2half2_rn(1024.0f));
    const __half2 v = __hfma2(c, s, m);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
};

// One key's codes into its row of a 128-row operand, each eight elements in the order 0 4 1 5 2 6 3 7 they unpack in
// (the queries and the results take the same one). Values that leave T's range are kept at its end.
template <typename T, int D>
__device__ __forceinline__ void unpack_row(uint32_t base, int row, const uint32_t (&w)[D / 8], uint32_t pair) {
  const ValueUnpack<T> value(pair);
  const float s = __uint_as_float(pair << 16), m = __uint_as_float(pair & 0xffff0000u);
  const bool far = fmaf(15.0f, s, m) > kv_top<T>() || m < -kv_top<T>();
#pragma unroll
  for (int c = 0; c < D / 8; ++c) {
    uint32_t v[4];  // pairs (0, 4), (1, 5), (2, 6), (3, 7)
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = value(w[c], i);
    if (far) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float f[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          f[h] = fmaf((float)((w[c] >> (4 * (i + 4 * h))) & 15u), s, m);
          f[h] = fminf(fmaxf(f[h], -kv_top<T>()), kv_top<T>());
        }
        v[i] = Elem<T>::from_f2(f[0], f[1]);
      }
    }
    const uint32_t dst = base + (c >> 3) * 16384 + row * 128 + (((c & 7) ^ (row & 7)) << 4);
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]) : "memory");
  }
}

// An item of work: 256 rows of one kv head of one request.
struct PromptItem {
  AttnRequest rq;
  int32_t b, head, row0, rows, steps;
};

template <typename T, int D>
__global__ void __launch_bounds__(kPromptThreads, 1) attn_int4_prompt_kernel(const AttnInt4Args a, int32_t* fault) {
  using Sh = PromptShape<D>;
  extern __shared__ uint8_t raw[];
  __shared__ uint32_t s_tmem;
  __shared__ volatile int s_stop;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t base = (smem_u32(raw) + 1023u) & ~1023u;
  uint64_t* bars = reinterpret_cast<uint64_t*>(raw + (base - smem_u32(raw)) + Sh::kBars);
  pdl_wait();
  // Items in order: requests, heads, row blocks. Each warp walks them for itself, 32 requests at a time (a lane each);
  // all find the same ones.
  const int heads = a.kv.heads;
  PromptItem it;
  int window = -32;                          // first request of the window
  int64_t first = 0, window_items = 0;       // items before the window, and in it
  int64_t lane_items = 0, lane_before = 0;   // of this lane's request
  AttnRequest lane_rq = {};
  auto next_item = [&](int64_t index) {
    while (index >= first + window_items) {
      window += 32;
      if (window >= a.B) return false;
      first += window_items;
      lane_items = 0;
      if (window + lane < a.B) {
        lane_rq = attn_request<8>(a, window + lane, nullptr, false);
        const int64_t rows = (int64_t)lane_rq.qlen * a.group;
        if (rows > a.split_rows) lane_items = (rows + kPromptRows - 1) / kPromptRows * heads;
      }
      int64_t incl = lane_items;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int64_t y = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += y;
      }
      lane_before = incl - lane_items;
      window_items = __shfl_sync(0xffffffffu, incl, 31);
    }
    const int64_t at = index - first;
    const int src = __ffs(__ballot_sync(0xffffffffu, at >= lane_before && at < lane_before + lane_items)) - 1;
    it.b = window + src;
    it.rq.q0 = __shfl_sync(0xffffffffu, lane_rq.q0, src);
    it.rq.qlen = __shfl_sync(0xffffffffu, lane_rq.qlen, src);
    it.rq.n = __shfl_sync(0xffffffffu, lane_rq.n, src);
    const int blocks = (int)(__shfl_sync(0xffffffffu, lane_items, src) / heads);
    const int rest = (int)(at - __shfl_sync(0xffffffffu, lane_before, src));
    it.head = rest / blocks;
    // the longest first: under a causal mask the last rows see the most keys
    it.row0 = (blocks - 1 - rest % blocks) * kPromptRows;
    it.rows = min(kPromptRows, it.rq.qlen * a.group - it.row0);
    const int last = (it.row0 + it.rows - 1) / a.group;
    const int seen = a.causal ? min(it.rq.n, max(0, it.rq.n - it.rq.qlen + last + 1)) : it.rq.n;
    it.steps = (seen + kPromptKeys - 1) / kPromptKeys;
    return true;
  };
  if (!next_item(blockIdx.x)) {  // nothing for this CTA
    pdl_launch_dependents();
    return;
  }

  if (tid == 0) {
    s_stop = 0;
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bars[kKFull + i], 128);
      mbar_init(&bars[kKEmpty + i], 1);
      mbar_init(&bars[kVFull + i], 128);
      mbar_init(&bars[kVEmpty + i], 1);
      mbar_init(&bars[kSFull + i], 1);
      mbar_init(&bars[kPFull + i], 128);
      mbar_init(&bars[kQFull + i], 128);
      mbar_init(&bars[kOFull + i], 1);
    }
    fence_barrier_init();
  }
  if (warp == 16) {
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
    // A negative softmax scale becomes a positive one of negated queries, so that the largest product is the largest logit.
    const float scale = fmaxf(fabsf(a.scale_log2), 1e-37f);  // not 0, which would make NaNs of hidden columns
    const uint32_t flip = a.scale_log2 < 0.0f ? 0x80008000u : 0u;
    // Columns from `left` on are hidden from the row.
    auto hide = [&](uint32_t (&s)[64], int left) {
#pragma unroll
      for (int i = 0; i < 64; ++i) s[i] = i < left ? s[i] : 0xff800000u;
    };
    uint32_t s_phase = 0, o_phase = 0;
    bool go = true;
    for (int64_t item = blockIdx.x; go && next_item(item); item += gridDim.x) {
      if (tile * 128 >= it.rows) continue;
      const int row = it.row0 + tile * 128 + r;
      const bool here = tile * 128 + r < it.rows;
      const int tok = (it.row0 + min(tile * 128 + r, it.rows - 1)) / a.group;
      const int sub = row - tok * a.group;
      const int lim = a.causal ? min(it.rq.n, max(0, it.rq.n - it.rq.qlen + tok + 1)) : it.rq.n;
      if (it.steps > 0) {
        const uint16_t* src = static_cast<const uint16_t*>(a.q) + (int64_t)(it.rq.q0 + tok) * a.qsn +
                              ((int64_t)it.head * a.group + (here ? sub : 0)) * a.qsh;
#pragma unroll
        for (int c = 0; c < D / 8; ++c) {
          Vec16 v = {0, 0, 0, 0};
          if (here) v = a.q_vec ? kv_load8<true>(src + 8 * c) : kv_load8<false>(src + 8 * c);
          v = Vec16{__byte_perm(v.a, v.c, 0x5410), __byte_perm(v.a, v.c, 0x7632), __byte_perm(v.b, v.d, 0x5410),
                    __byte_perm(v.b, v.d, 0x7632)};
          const uint32_t dst = base + Sh::kQ + tile * Sh::kTile + (c >> 3) * 16384 + r * 128 + (((c & 7) ^ (r & 7)) << 4);
          asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst), "r"(v.a ^ flip), "r"(v.b ^ flip), "r"(v.c ^ flip),
                       "r"(v.d ^ flip)
                       : "memory");
        }
        fence_proxy_async_smem();
        mbar_arrive(&bars[kQFull + tile]);
      }
      float m = -INFINITY, l = 0.0f;
      for (int j = 0; go && j < it.steps; ++j) {
        go = wait(kSFull + tile, s_phase);
        s_phase ^= 1;
        if (!__all_sync(0xffffffffu, go)) {
          go = false;
          break;
        }
        tmem_fence_after();
        const int left = lim - j * kPromptKeys;  // keys of this step that the row sees
        const bool edge = __any_sync(0xffffffffu, left < kPromptKeys);
        // The row's largest logit first: P overwrites S, so nothing may be left to do again.
        float top = -INFINITY;
#pragma unroll 1
        for (int c = 0; c < 2; ++c) {
          uint32_t s[64];
          tmem_ld64(s, s_addr + c * 64);
          if (edge) {
            hide(s, left - c * 64);
          }
          float t0 = -INFINITY, t1 = -INFINITY;
#pragma unroll
          for (int i = 0; i < 64; i += 4) {
            t0 = fmaxf(t0, fmaxf(__uint_as_float(s[i]), __uint_as_float(s[i + 1])));
            t1 = fmaxf(t1, fmaxf(__uint_as_float(s[i + 2]), __uint_as_float(s[i + 3])));
          }
          top = fmaxf(top, fmaxf(t0, t1));
        }
        top *= scale;
        const bool up = top > m + 8.0f;
        if (__any_sync(0xffffffffu, up)) {
          const float was = m;
          m = up ? top : m;
          const float factor = was == m || was == -INFINITY ? 1.0f : ex2(was - m);  // before its first key the row of O is zeros
          if (j > 0) {
#pragma unroll 1
            for (int c = 0; c < D / 32; ++c) {
              uint32_t o[32];
              tmem_ld32(o, o_addr + c * 32);
#pragma unroll
              for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * factor);
              tmem_st32(o_addr + c * 32, o);
            }
          }
          l *= factor;
        }
        const float ref = m == -INFINITY ? 0.0f : -m;
        float2 part = make_float2(0.0f, 0.0f);
#pragma unroll 1
        for (int c = 0; c < 2; ++c) {
          uint32_t s[64], p[32];
          tmem_ld64(s, s_addr + c * 64);
          if (edge) hide(s, left - c * 64);
#pragma unroll
          for (int i = 0; i < 64; i += 2) {
            const float2 x = fma2_f32(make_float2(__uint_as_float(s[i]), __uint_as_float(s[i + 1])), both(scale), both(ref));
            const float2 e = make_float2(ex2(x.x), ex2(x.y));
            part = add2_f32(part, e);
            p[i / 2] = Elem<T>::from_f2(e.x, e.y);
          }
          tmem_st32(s_addr + c * 32, p);  // columns that this thread has read
        }
        l += part.x + part.y;
        tmem_wait_st();
        tmem_fence_before();
        mbar_arrive(&bars[kPFull + tile]);
      }
      if (!go) break;
      if (it.steps > 0) {
        go = wait(kOFull + tile, o_phase);
        o_phase ^= 1;
        if (!__all_sync(0xffffffffu, go)) {
          go = false;
          break;
        }
        tmem_fence_after();
      }
      const float inv = l != 0.0f ? 1.0f / l : 0.0f;
      uint16_t* dst = static_cast<uint16_t*>(a.out) + (int64_t)(it.rq.q0 + tok) * a.osn +
                      ((int64_t)it.head * a.group + sub) * a.osh;
#pragma unroll 1
      for (int c = 0; c < D / 32; ++c) {
        uint32_t o[32];
        if (it.steps > 0) {
          tmem_ld32(o, o_addr + c * 32);
        }
#pragma unroll
        for (int i = 0; i < 32; i += 8) {
          float f[8];
#pragma unroll
          for (int x = 0; x < 8; ++x) f[x] = l != 0.0f ? __uint_as_float(o[i + (x < 4 ? 2 * x : 2 * x - 7)]) * inv : 0.0f;
          if (here) {
            if (a.o_vec) kv_store8<true>(dst + c * 32 + i, pack8<T>(f));
            else kv_store8<false>(dst + c * 32 + i, pack8<T>(f));
          }
        }
      }
      tmem_fence_before();
      if (here && a.lse != nullptr)
        a.lse[(int64_t)(it.rq.q0 + tok) * heads * a.group + (int64_t)it.head * a.group + sub] =
            l != 0.0f ? m + __log2f(l) : -INFINITY;
    }
  } else if (warp < 16) {
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
    for (int64_t item = blockIdx.x; go && next_item(item); item += gridDim.x) {
      const int32_t* table = a.block_tables + (int64_t)it.b * a.table_stride;
      // The page of this thread's key in step j, -1 past the cache's end and for a bad one.
      auto find = [&](int j) {
        const int tok = j * kPromptKeys + r;
        if (j >= it.steps || tok >= it.rq.n) return -1;
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
      load(0, find(0), w, pair);
      int page = find(1);
      for (int j = 0; j < it.steps; ++j, ++done) {
        const int stage = done & 1;
        uint32_t w_next[D / 8];
        uint2 pair_next;
        load(j + 1, page, w_next, pair_next);
        page = find(j + 2);
        // The first use of a stage finds it free.
        go = __all_sync(0xffffffffu, wait(empty + stage, ((done >> 1) & 1) ^ 1));
        if (!go) break;
        // A value row that is not finite may be hidden from some rows, whose zero weights would not hide it: it is
        // replaced by zeros and its key by NaNs, which reach exactly the rows that see it.
        const float vf = fmaf(__uint_as_float(pair.y << 16), 0.0f, __uint_as_float(pair.y & 0xffff0000u) * 0.0f);
        const uint32_t mine = values ? (vf != 0.0f || vf != vf ? 0u : pair.y) : (vf != 0.0f || vf != vf ? 0x7fc07fc0u : pair.x);
        unpack_row<T, D>(operand + stage * Sh::kTile, r, w, mine);
        fence_proxy_async_smem();
        mbar_arrive(&bars[full + stage]);
#pragma unroll
        for (int i = 0; i < D / 8; ++i) w[i] = w_next[i];
        pair = pair_next;
      }
    }
  } else {
    // ---------------- products: lane 0 issues, the others walk along ----------------
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kPromptIssueRegs));
    constexpr uint32_t kIdescS = umma_idesc<T>(128, kPromptKeys, false), kIdescO = umma_idesc<T>(128, D, true);
    uint32_t done = 0, q_phase[2] = {0, 0}, p_phase[2] = {0, 0};
    bool go = true;
    auto scores = [&](int tile, int stage) {
      const uint32_t q = base + Sh::kQ + tile * Sh::kTile, k = base + Sh::kK + stage * Sh::kTile;
#pragma unroll
      for (int x = 0; x < D / 16; ++x) {
        const uint32_t off = (x >> 2) * 16384 + (x & 3) * 32;  // 16 elements of D
        umma_ss(tmem + tile * 128, umma_desc(q + off, 16, 1024), umma_desc(k + off, 16, 1024), kIdescS, x > 0);
      }
      umma_commit(&bars[kSFull + tile]);
    };
    auto run_item = [&] {
      bool ok = true;
      const int tiles = it.rows > 128 ? 2 : 1;
      ok = wait(kKFull + (done & 1), (done >> 1) & 1);
      for (int tile = 0; ok && tile < tiles; ++tile) {
        ok = wait(kQFull + tile, q_phase[tile]);
        q_phase[tile] ^= 1;
        if (!ok) break;
        tmem_fence_after();
        scores(tile, done & 1);
      }
      if (!ok) return false;
      umma_commit(&bars[kKEmpty + (done & 1)]);
      for (int j = 0; ok && j < it.steps; ++j, ++done) {
        const int stage = done & 1;
        const uint32_t parity = (done >> 1) & 1;
        ok = wait(kVFull + stage, parity);
        for (int tile = 0; ok && tile < tiles; ++tile) {
          ok = wait(kPFull + tile, p_phase[tile]);
          p_phase[tile] ^= 1;
          if (!ok) break;
          tmem_fence_after();
#pragma unroll
          for (int x = 0; x < kPromptKeys / 16; ++x)
            umma_ts(tmem + 256 + tile * 128, tmem + tile * 128 + x * 8,
                    umma_desc(base + Sh::kV + stage * Sh::kTile + x * 2048, 16384, 1024), kIdescO, j > 0 || x > 0);
          if (tile == tiles - 1) umma_commit(&bars[kVEmpty + stage]);
          if (j + 1 < it.steps) {
            if (tile == 0) ok = wait(kKFull + ((done + 1) & 1), ((done + 1) >> 1) & 1);
            if (!ok) break;
            scores(tile, (done + 1) & 1);
            if (tile == tiles - 1) umma_commit(&bars[kKEmpty + ((done + 1) & 1)]);
          } else {
            umma_commit(&bars[kOFull + tile]);
          }
        }
      }
      return ok;
    };
    for (int64_t item = blockIdx.x; go && next_item(item); item += gridDim.x) {
      if (it.steps == 0) continue;
      if (lane == 0) go = run_item();
      go = __shfl_sync(0xffffffffu, go, 0);
    }
    if (!go && lane == 0) {
      // Products may be in flight over shared and tensor memory: let them end (bounded) before anything is freed.
      umma_commit(&bars[kOFull]);
      (void)mbar_wait_bounded(&bars[kOFull], 0, kWaitLimitNs / 4);
    }
  }
  __syncwarp();
  tmem_fence_before();
  __syncthreads();
  if (warp == 16) {
    tmem_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
  }
  pdl_launch_dependents();
}

}  // namespace mas
