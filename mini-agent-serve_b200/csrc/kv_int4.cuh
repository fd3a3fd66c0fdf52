// kv_int4.cuh -- the paged KV cache held in 4 bits: its row format, the quantising append and the
// dequantising read (sm_100a).
//
// A row is one token's k or v of one kv head, D values x. It is stored as D codes of 4 bits and one bf16
// pair (scale s, minimum m):
//   m = the largest bf16 <= min(x);   s = the smallest bf16 >= max(2^-126, (max(x) - m) / 15)
//   c_i = floor(f32(x_i - m) / s + 1/2)   in 0..15;      value_i = c_i * s + m
// so every x_i lies in [m, m + 15 s] and its value within s / 2 of it. The pair is bf16 because it must
// reach as far as the activations do; rounding m down and s up, not to the nearest, keeps both ends of the row
// inside the codes' range, at a cost of at most 2^-7 of the step. A row that holds a NaN or an infinity
// has no such form: its pair is stored as NaN and all of it reads as NaN.
//
// Codes: two a byte, element 2i in the low half, k and v apart, [pages, page_size, heads, D / 2] (NHD) or
// [pages, heads, page_size, D / 2] (HND). Pairs: bf16 [pages, heads, page_size, 4], (k s, k m, v s, v m), head-major
// under either layout, so that a head's reader finds the pairs of consecutive tokens side by side
// (in token-major order it would use 8 bytes of each 32-byte sector).
//
// The arithmetic decides every code exactly. With h = s / 2 and d = x / 2 - m / 2 (halves, so that
// max(x) - m cannot overflow), c0 = floor(d * (1 / h)) may be one off only where d / h is nearly an integer,
// and there both candidates round to the same code; r = fma(-(c0 + 1/2), h, d) has the sign of
// d - (c0 + 1/2) h because that product has 13 significant bits and the fma rounds once. c = c0 + (r >= 0).
// s is decided the same way: 15 s / 2 has 12 bits, so comparing it with the difference rounded up is exact.
#pragma once

#include <type_traits>

#include "common.cuh"

namespace mas {

struct KVInt4Args {
  uint8_t* k_codes;
  uint8_t* v_codes;
  __nv_bfloat16* pairs;
  int64_t num_pages, page_size;
  int64_t stride_page, stride_entry, stride_head;  // bytes; k and v codes share them
  int64_t pair_stride_page;                        // elements
  int32_t heads;
};

struct KVInt4RowArgs {
  KVInt4Args kv;
  const int32_t* kv_indices;
  int64_t num_indices;
  const int32_t* kv_indptr;
  int64_t batch_size;
  int32_t page_shift;            // log2(page_size), or -1
  const int32_t* batch_indices;  // [T]; -1: a padding row
  const void* pos;               // [T]
  int64_t T;
  void* k;  // append: the rows to store (only read); read: where they go
  void* v;
  int64_t ksn, ksh, vsn, vsh;  // elements
  int32_t* status;
};

constexpr float kKVScaleMin = 1.17549435e-38f;  // 2^-126: 2 / s stays finite

// The least bf16 that is >= max(2^-126, 2 * dh / 15); dh >= 0 and finite, rounded up from half the difference.
__device__ __forceinline__ float kv_scale_up(float dh) {
  float s = __uint_as_float(__float_as_uint(dh * (2.0f / 15.0f)) & 0xffff0000u);
  // The truncated product is at most two bf16 steps short.
  if (s * 7.5f < dh) s = __uint_as_float(__float_as_uint(s) + 0x10000u);
  if (s * 7.5f < dh) s = __uint_as_float(__float_as_uint(s) + 0x10000u);
  return fmaxf(s, kKVScaleMin);
}

// The largest bf16 that is <= x (finite).
__device__ __forceinline__ float kv_min_down(float x) {
  const uint32_t u = __float_as_uint(x);
  return __uint_as_float((u & 0xffff0000u) + ((u & 0x8000ffffu) > 0x80000000u ? 0x10000u : 0u));
}

struct KVSlot {
  int64_t page;
  int32_t entry;  // -1: out of range, -2: a padding row
};

template <typename PosT>
__device__ __forceinline__ KVSlot kv_int4_slot(const KVInt4RowArgs& a, int64_t t) {
  const int32_t b = a.batch_indices[t];
  const int64_t pos = (int64_t)static_cast<const PosT*>(a.pos)[t];
  if (b == -1) return {0, -2};
  if (b < 0 || b >= a.batch_size || pos < 0 || pos > INT32_MAX) return {0, -1};
  const int64_t first = a.kv_indptr[b];
  const uint32_t p = (uint32_t)pos, size = (uint32_t)a.kv.page_size;
  const uint32_t block = a.page_shift >= 0 ? p >> a.page_shift : p / size;
  if (first < 0 || first + block >= a.num_indices) return {0, -1};
  const int64_t page = a.kv_indices[first + block];
  if (page < 0 || page >= a.kv.num_pages) return {0, -1};
  return {page, (int32_t)(p - block * size)};
}

constexpr int kKVInt4Threads = 256;
constexpr int kKVInt4Unroll = 4;  // row pairs a warp holds at once

// Packed 16-bit minima and maxima that pass a NaN on.
template <typename T>
__device__ __forceinline__ uint32_t min2_nan(uint32_t a, uint32_t b) {
  uint32_t r;
  if (std::is_same<T, __half>::value) asm("min.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  else asm("min.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
template <typename T>
__device__ __forceinline__ uint32_t max2_nan(uint32_t a, uint32_t b) {
  uint32_t r;
  if (std::is_same<T, __half>::value) asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  else asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ float2 add2_rz_f32(float2 a, float2 b) {
  float2 c;
  asm("{\n\t.reg .b64 ra, rb, rc;\n\t"
      "mov.b64 ra, {%2, %3};\n\t"
      "mov.b64 rb, {%4, %5};\n\t"
      "add.rz.f32x2 rc, ra, rb;\n\t"
      "mov.b64 {%0, %1}, rc;\n\t}"
      : "=f"(c.x), "=f"(c.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return c;
}
__device__ __forceinline__ float2 add2_f32(float2 a, float2 b) {
  float2 c;
  asm("{\n\t.reg .b64 ra, rb, rc;\n\t"
      "mov.b64 ra, {%2, %3};\n\t"
      "mov.b64 rb, {%4, %5};\n\t"
      "add.rn.f32x2 rc, ra, rb;\n\t"
      "mov.b64 {%0, %1}, rc;\n\t}"
      : "=f"(c.x), "=f"(c.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return c;
}
__device__ __forceinline__ float2 both(float x) { return make_float2(x, x); }

// 8 consecutive elements of a row as four packed words.
template <bool ALIGNED>
__device__ __forceinline__ Vec16 kv_load8(const uint16_t* p) {
  if (ALIGNED) return ld_ro(p);
  Vec16 v;
  v.a = p[0] | ((uint32_t)p[1] << 16);
  v.b = p[2] | ((uint32_t)p[3] << 16);
  v.c = p[4] | ((uint32_t)p[5] << 16);
  v.d = p[6] | ((uint32_t)p[7] << 16);
  return v;
}
template <bool ALIGNED>
__device__ __forceinline__ void kv_store8(uint16_t* p, const Vec16& v) {
  if (ALIGNED) {
    st_plain(p, v);
    return;
  }
  const uint32_t w[4] = {v.a, v.b, v.c, v.d};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    p[2 * i] = (uint16_t)w[i];
    p[2 * i + 1] = (uint16_t)(w[i] >> 16);
  }
}

// One pass of a warp stores 32 / (D / 8) rows (the k and the v row of one head at D = 128, of two at 64),
// 8 elements a lane, so a row's minimum and maximum are a few shuffles away and its codes leave as one
// 4-byte word a lane. A warp takes up to kKVInt4Unroll passes of one token, all their loads first
// (grid: x over tokens, y over its groups of heads, so that no index is divided).
// What bounds it is issue, not bytes: 168 warp instructions a (token, head) of 128, 63 % of the issue slots and 61 % of the
// ALU's; 38 K tokens of 8 heads take 67 us (floor 30 us at 6.5 TB/s), 73 with an index division a row.
template <typename T, typename PosT, int D, bool ALIGNED>
__global__ void __launch_bounds__(kKVInt4Threads) append_kv_int4_kernel(const KVInt4RowArgs a) {
  constexpr int kLanes = D / 8;               // lanes a row
  constexpr int kHeads = 32 / kLanes / 2;     // heads a pass
  constexpr int kGroup = kHeads * kKVInt4Unroll;  // heads a warp
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int sub = lane / kLanes, col = lane % kLanes;
  const bool is_v = sub & 1;
  const int head0 = blockIdx.y * kGroup + (sub >> 1);
  const int64_t nwarps = ((int64_t)gridDim.x * kKVInt4Threads) >> 5;
  for (int64_t t = ((int64_t)blockIdx.x * kKVInt4Threads + threadIdx.x) >> 5; t < a.T; t += nwarps) {
    const uint16_t* row = static_cast<const uint16_t*>(is_v ? a.v : a.k) + t * (is_v ? a.vsn : a.ksn) + col * 8;
    Vec16 x[kKVInt4Unroll];
#pragma unroll
    for (int i = 0; i < kKVInt4Unroll; ++i) {
      const int h = head0 + i * kHeads;
      if (h < a.kv.heads) x[i] = kv_load8<ALIGNED>(row + (int64_t)h * (is_v ? a.vsh : a.ksh));
      else x[i] = Vec16{0, 0, 0, 0};
    }
    const KVSlot slot = kv_int4_slot<PosT>(a, t);
    if (slot.entry < 0) {
      if (slot.entry == -1 && lane == 0) flag_status(a.status, MAS_STATUS_KV_SLOT_OUT_OF_RANGE);
      continue;
    }
    uint8_t* codes = (is_v ? a.kv.v_codes : a.kv.k_codes) + slot.page * a.kv.stride_page +
                     slot.entry * a.kv.stride_entry + col * 4;
    __nv_bfloat16* pairs = a.kv.pairs + slot.page * a.kv.pair_stride_page + (int64_t)slot.entry * 4 + (is_v ? 2 : 0);
#pragma unroll
    for (int i = 0; i < kKVInt4Unroll; ++i) {
      const int h = head0 + i * kHeads;
      const uint32_t xs[4] = {x[i].a, x[i].b, x[i].c, x[i].d};
      uint32_t lo2 = min2_nan<T>(min2_nan<T>(xs[0], xs[1]), min2_nan<T>(xs[2], xs[3]));
      uint32_t hi2 = max2_nan<T>(max2_nan<T>(xs[0], xs[1]), max2_nan<T>(xs[2], xs[3]));
      // The minimum and the negated maximum travel as one pair: a single minimum reduces both.
      lo2 = min2_nan<T>(lo2, __byte_perm(lo2, lo2, 0x1032));
      hi2 = max2_nan<T>(hi2, __byte_perm(hi2, hi2, 0x1032));
      uint32_t ends = __byte_perm(lo2, hi2 ^ 0x80008000u, 0x5410);
#pragma unroll
      for (int o = kLanes / 2; o > 0; o >>= 1) ends = min2_nan<T>(ends, __shfl_xor_sync(0xffffffffu, ends, o));
      const float2 lh = Elem<T>::to_f2(ends);
      const float lo = lh.x, hi = -lh.y;
      const bool finite = fabsf(lo) <= 3.4e38f && fabsf(hi) <= 3.4e38f;
      const float m = kv_min_down(lo);
      const float nmh = -0.5f * m;
      const float s = kv_scale_up(__fmaf_ru(hi, 0.5f, nmh));
      const float sh = 0.5f * s, inv = __frcp_rn(sh);
      // word accumulates bits(big) + 1 - (r < 0), whose low digit is the code; the constant digits leave at the end.
      uint32_t word = 0;
#pragma unroll
      for (int j = 3; j >= 0; --j) {
        const float2 d = fma2_f32(Elem<T>::to_f2(xs[j]), both(0.5f), both(nmh));
        const float2 big = add2_rz_f32(mul2_f32(d, both(inv)), both(8388608.0f));  // 2^23 + c0
        const float2 r = fma2_f32(add2_f32(big, both(-8388607.5f)), both(-sh), d);
        word = word * 16u + __float_as_uint(big.y) - (__float_as_uint(r.y) >> 31);
        word = word * 16u + __float_as_uint(big.x) - (__float_as_uint(r.x) >> 31);
      }
      word -= (0x4b000000u - 1u) * 0x11111111u;
      if (h < a.kv.heads) {
        *reinterpret_cast<uint32_t*>(codes + (int64_t)h * a.kv.stride_head) = finite ? word : 0u;
        if (col == 0) {
          const uint32_t pair = (__float_as_uint(s) >> 16) | (__float_as_uint(m) & 0xffff0000u);
          *reinterpret_cast<uint32_t*>(pairs + (int64_t)h * a.kv.page_size * 4) = finite ? pair : 0x7fc07fc0u;
        }
      }
    }
  }
  pdl_launch_dependents();
}

// T's largest value: c * s + m of a row that ends near it may lie a step past it, and reads as that value.
template <typename T>
__device__ __forceinline__ float kv_top() {
  return std::is_same<T, __half>::value ? 65504.0f : 3.38953139e38f;
}

// The read-back: the same lanes, 4 bytes of codes in and 16 bytes of values out each. 38 K tokens of 8 heads of 128: 44 us
// (floor 30), by issue again (59 %, ALU 64 %).
template <typename T, typename PosT, int D, bool ALIGNED>
__global__ void __launch_bounds__(kKVInt4Threads) read_kv_int4_kernel(const KVInt4RowArgs a) {
  constexpr int kLanes = D / 8;
  constexpr int kHeads = 32 / kLanes / 2;
  constexpr int kGroup = kHeads * kKVInt4Unroll;
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int sub = lane / kLanes, col = lane % kLanes;
  const bool is_v = sub & 1;
  const int head0 = blockIdx.y * kGroup + (sub >> 1);
  const int64_t nwarps = ((int64_t)gridDim.x * kKVInt4Threads) >> 5;
  for (int64_t t = ((int64_t)blockIdx.x * kKVInt4Threads + threadIdx.x) >> 5; t < a.T; t += nwarps) {
    const KVSlot slot = kv_int4_slot<PosT>(a, t);
    if (slot.entry == -1 && lane == 0) flag_status(a.status, MAS_STATUS_KV_SLOT_OUT_OF_RANGE);
    const uint8_t* codes = (is_v ? a.kv.v_codes : a.kv.k_codes) + slot.page * a.kv.stride_page +
                           slot.entry * a.kv.stride_entry + col * 4;
    const __nv_bfloat16* pairs = a.kv.pairs + slot.page * a.kv.pair_stride_page + (int64_t)slot.entry * 4 + (is_v ? 2 : 0);
    uint32_t word[kKVInt4Unroll], pair[kKVInt4Unroll];
#pragma unroll
    for (int i = 0; i < kKVInt4Unroll; ++i) {
      const int h = head0 + i * kHeads;
      const bool here = slot.entry >= 0 && h < a.kv.heads;
      word[i] = here ? *reinterpret_cast<const uint32_t*>(codes + (int64_t)h * a.kv.stride_head) : 0u;
      pair[i] = here ? *reinterpret_cast<const uint32_t*>(pairs + (int64_t)h * a.kv.page_size * 4) : 0u;
    }
    uint16_t* row = static_cast<uint16_t*>(is_v ? a.v : a.k) + t * (is_v ? a.vsn : a.ksn) + col * 8;
#pragma unroll
    for (int i = 0; i < kKVInt4Unroll; ++i) {
      const int h = head0 + i * kHeads;
      if (h >= a.kv.heads) continue;
      const float s = __uint_as_float(pair[i] << 16), m = __uint_as_float(pair[i] & 0xffff0000u);
      float f[8];
#pragma unroll
      for (int j = 0; j < 8; j += 2) {
        // 16 + c, the code in the top of the mantissa
        const uint32_t c0 = (j < 5 ? word[i] << (19 - 4 * j) : word[i] >> (4 * j - 19)) & 0x780000u;
        const uint32_t c1 = (j < 4 ? word[i] << (15 - 4 * j) : word[i] >> (4 * j - 15)) & 0x780000u;
        const float2 c = add2_f32(make_float2(__uint_as_float(c0 | 0x41800000u), __uint_as_float(c1 | 0x41800000u)), both(-16.0f));
        const float2 v = fma2_f32(c, both(s), both(m));
        f[j] = v.x;
        f[j + 1] = v.y;
      }
      if (fmaf(15.0f, s, m) > kv_top<T>() || m < -kv_top<T>()) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          f[j] = f[j] > kv_top<T>() ? kv_top<T>() : f[j];
          f[j] = f[j] < -kv_top<T>() ? -kv_top<T>() : f[j];
        }
      }
      kv_store8<ALIGNED>(row + (int64_t)h * (is_v ? a.vsh : a.ksh), pack8<T>(f));
    }
  }
  pdl_launch_dependents();
}

}  // namespace mas
