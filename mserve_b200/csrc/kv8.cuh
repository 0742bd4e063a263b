// Shared by the 8-bit paged cache's kernels (mskv_kv8_*): page addressing, conversions, checks.
#pragma once

#include <cuda_fp8.h>

#include <limits.h>

#include "common.cuh"

namespace mskv {

// Device copy of mskv_kv8_pages.
struct Kv8Dev {
  uint8_t* k;
  uint8_t* v;
  int8_t* exps;
  uint8_t* bounds;
  const int32_t* page_table;
  int64_t sp, sh, pt_stride, num_pages;
  int32_t max_pages, page_size, heads, batch;
};

inline Kv8Dev to_dev(const mskv_kv8_pages& p) {
  Kv8Dev d;
  d.k = static_cast<uint8_t*>(p.k);
  d.v = static_cast<uint8_t*>(p.v);
  d.exps = static_cast<int8_t*>(p.exps);
  d.bounds = static_cast<uint8_t*>(p.bounds);
  d.page_table = p.page_table;
  d.sp = p.stride_page; d.sh = p.stride_h; d.pt_stride = p.pt_stride_b; d.num_pages = p.num_pages;
  d.max_pages = p.max_pages; d.page_size = p.page_size; d.heads = p.kv_heads; d.batch = p.batch;
  return d;
}

// Host-side checks of the addressing; `what` names the entry point.
inline int check_kv8(const mskv_kv8_pages& p, const char* what) {
  if (!p.k || !p.v || !p.exps || !p.page_table) return fail(MSKV_ERR_ARG, "%s: NULL k, v, exps or page_table", what);
  if (p.dtype != MSKV_DT_FP8_E4M3 && p.dtype != MSKV_DT_FP8_E5M2)
    return fail(MSKV_ERR_DTYPE, "%s: the cache must be fp8 e4m3 or e5m2", what);
  if (p.batch <= 0 || p.kv_heads <= 0 || p.num_pages <= 0 || p.max_pages <= 0)
    return fail(MSKV_ERR_ARG, "%s: batch, kv_heads, num_pages and max_pages must be > 0", what);
  if ((int64_t)p.batch * p.kv_heads > INT_MAX / 64) return fail(MSKV_ERR_RANGE, "%s: batch*kv_heads too large", what);
  if (p.page_size <= 0 || p.page_size % 16 || p.page_size > 128)
    return fail(MSKV_ERR_RANGE, "%s: page_size must be a multiple of 16, at most 128", what);
  if (p.head_dim != 64 && p.head_dim != 128 && p.head_dim != 256)
    return fail(MSKV_ERR_RANGE, "%s: head_dim must be 64, 128 or 256", what);
  if (((uintptr_t)p.k | (uintptr_t)p.v | (uintptr_t)p.bounds | (uintptr_t)p.stride_page | (uintptr_t)p.stride_h) & 15)
    return fail(MSKV_ERR_ARG, "%s: k, v, bounds, stride_page and stride_h must be 16-byte aligned", what);
  if ((uintptr_t)p.exps & 1) return fail(MSKV_ERR_ARG, "%s: exps must be 2-byte aligned", what);
  if ((uintptr_t)p.page_table & 3) return fail(MSKV_ERR_ARG, "%s: page_table must be 4-byte aligned", what);
  return MSKV_OK;
}

// The call's arrays of 32-bit words (lengths, counts, lists, scores, the status word), NULL or aligned.
template <typename... T>
inline int check_words(const char* what, const T*... words) {
  if ((0 | ... | (uintptr_t)words) & 3) return fail(MSKV_ERR_ARG, "%s: arrays of 32-bit words must be 4-byte aligned", what);
  return MSKV_OK;
}

// Multiprocessors of the current device, asked for once per device (two plans a call).
inline int sms_of_device() {
  static std::atomic<int> known[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return num_sms();
  int n = known[dev].load(std::memory_order_relaxed);
  if (n == 0) known[dev].store(n = num_sms(), std::memory_order_relaxed);
  return n;
}

// Division by an invariant (Granlund and Montgomery): a multiplication, an average and a shift.
struct Divisor {
  uint32_t factor, shift;
  explicit Divisor(uint32_t d = 1) : factor(1), shift(0) {
    uint32_t l = 0;
    while (l < 32 && ((uint64_t)1 << l) < d) ++l;
    factor = (uint32_t)((((uint64_t)1 << 32) * (((uint64_t)1 << l) - d)) / d + 1);
    shift = l;
  }
  __device__ __forceinline__ uint32_t quotient(uint32_t n) const {
    const uint32_t t = __umulhi(factor, n);
    return shift ? (t + ((n - t) >> 1)) >> (shift - 1) : n;
  }
};

// 2^e for e in [-126, 127].
__device__ __forceinline__ float pow2i(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// The four codes of a word as two half2 (exact): lo = codes 0, 1; hi = codes 2, 3.  An e5m2 code is
// the upper byte of an fp16, so its conversion is a byte permutation.
template <bool E5M2>
__device__ __forceinline__ void codes_to_half(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if constexpr (E5M2) {
    lo = __byte_perm(w, 0u, 0x1404);
    hi = __byte_perm(w, 0u, 0x3424);
  } else {
    asm("{ .reg .b16 l, h; mov.b32 {l, h}, %2; cvt.rn.f16x2.e4m3x2 %0, l; cvt.rn.f16x2.e4m3x2 %1, h; }"
        : "=r"(lo), "=r"(hi) : "r"(w));
  }
}

// Two values to codes: round to nearest even, saturating to the largest finite code; NaN stays NaN.
template <bool E5M2>
__device__ __forceinline__ uint32_t to_codes(float a, float b) {
  return __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, E5M2 ? __NV_E5M2 : __NV_E4M3);
}

// Streaming 16-byte read-only load (no L1 allocation).
__device__ __forceinline__ uint4 ld_stream16(const void* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}

// D (fp32) += A (16x16 fp16, row) * B (16x8 fp16, col).
__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// One element of a 16-bit query as fp32.
template <bool BF16>
__device__ __forceinline__ float q_elem(const char* p) {
  const uint16_t u = *reinterpret_cast<const uint16_t*>(p);
  if constexpr (BF16) return __uint_as_float((uint32_t)u << 16);
  else return __half2float(__ushort_as_half(u));
}

}  // namespace mskv
