// Append to the 8-bit paged cache (mskv_kv8_append).
//
// A page of one KV head is quantised as a whole: x[t,d] are the values it holds after the append
// (tokens before tok0 as code * 2^e_old, new ones as given), a = max finite |x|, e the smallest
// exponent with a <= F * 2^e (F = 448 = 1.75 * 2^8 for e4m3, 57344 = 1.75 * 2^15 for e5m2), and
// code = rn(x * 2^-e).  The multiplication by a power of two is exact, so a code has one
// rounding; a page whose exponent a later token raises keeps its codes but for f8 subnormals.
//
// A unit is a (page, KV head): page_size/16 warps for K and as many for V, each with 16 rows of its half, 8
// neighbouring elements of a row per lane and step; a CTA of 8 warps has as many units as fit (one unit
// of 2 warps a CTA: 16400 CTAs for 2 x 16384 tokens of 8 heads start no faster than 77 us).
//  * A page that only receives 16-bit rows (a prompt's) holds them as loaded, packed: every row is read
//    once; the maximum and the bounds are packed too (the bounds of the inputs, as rounding keeps their order).
//  * Other pages (a decode token joins old rows; fp32 rows) take their rows as fp32, a batch of steps at a time,
//    a second time from the caches where one batch does not hold them.  Old rows are stored again only
//    when the exponent changed.
// Measured: 2 x 16384 bf16 tokens, 8 heads, 128 dims (206 MB) 37.4 us = 0.84 of the copy rate; 4 x up to 64 fp16 tokens,
// 8 heads 4.2 us; one token of 8 sequences, 4 heads 2.8 us (launch, length, page id, rows).
#include <algorithm>
#include <type_traits>

#include "kv8.cuh"

namespace mskv {

struct AppendDev {
  Kv8Dev pg;
  const char* x[2];                 // K, V rows
  int64_t sb[2], sh[2], st[2];
  const int32_t* tok0;
  const int32_t* counts;
  uint32_t* status;
  int32_t num_tokens;
  int32_t parts_log2;               // 16-row parts of a page; -1 where they are no power of two
  uint32_t touched, units, all_units;   // touched: pages of a sequence that num_tokens rows can reach; units of a CTA
  Divisor by_touched, by_heads;
};

enum NewType { kNewBf16 = 0, kNewF16 = 1, kNewF32 = 2 };

// Eight 16-bit elements as four words.
template <bool VEC>
__device__ __forceinline__ void load8_packed(const char* p, uint32_t (&w)[4]) {
  if constexpr (VEC) {
    const uint4 a = __ldg(reinterpret_cast<const uint4*>(p));
    w[0] = a.x; w[1] = a.y; w[2] = a.z; w[3] = a.w;
  } else {
    const uint16_t* s = reinterpret_cast<const uint16_t*>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = (uint32_t)s[2 * i] | ((uint32_t)s[2 * i + 1] << 16);
  }
}

template <int NT>
__device__ __forceinline__ void unpack8(const uint32_t (&w)[4], float (&x)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (NT == kNewBf16) {
      x[2 * i] = __uint_as_float(w[i] << 16);
      x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    } else {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      x[2 * i] = f.x;
      x[2 * i + 1] = f.y;
    }
  }
}

// Eight elements of row r of a page as loaded: an old row's codes (two words), a new row's elements (four or
// eight words), nothing.
template <int NT, bool VEC>
__device__ __forceinline__ void load_row(int r, int first_new, int rows, const uint8_t* codes, int d, int d0, const char* src,
                                         uint32_t (&w)[NT == kNewF32 ? 8 : 4]) {
  if (r < first_new) {
    const uint2 c = *reinterpret_cast<const uint2*>(codes + r * d + d0);
    w[0] = c.x;
    w[1] = c.y;
  } else if (r < rows) {
    if constexpr (NT != kNewF32) {
      load8_packed<VEC>(src, w);
    } else if constexpr (VEC) {
      const uint4 a = __ldg(reinterpret_cast<const uint4*>(src)), b = __ldg(reinterpret_cast<const uint4*>(src) + 1);
      w[0] = a.x; w[1] = a.y; w[2] = a.z; w[3] = a.w; w[4] = b.x; w[5] = b.y; w[6] = b.z; w[7] = b.w;
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i] = reinterpret_cast<const uint32_t*>(src)[i];
    }
  }
}

// Their values: of an old row code * scale.
template <bool E5M2, int NT>
__device__ __forceinline__ void row_values(bool old, const uint32_t (&w)[NT == kNewF32 ? 8 : 4], float scale, float (&x)[8]) {
  if (old) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      uint32_t lo, hi;
      codes_to_half<E5M2>(w[i], lo, hi);
      const float2 u = __half22float2(*reinterpret_cast<const __half2*>(&lo));
      const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&hi));
      x[4 * i] = u.x * scale; x[4 * i + 1] = u.y * scale; x[4 * i + 2] = v.x * scale; x[4 * i + 3] = v.y * scale;
    }
  } else if constexpr (NT == kNewF32) {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = __uint_as_float(w[i]);
  } else {
    unpack8<NT>(w, x);
  }
}

template <bool E5M2>
__device__ __forceinline__ void store_codes(uint8_t* p, const float (&x)[8], float inv) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    // a packed product of two
    float a, b;
    asm("{ .reg .b64 v, k; mov.b64 v, {%2, %3}; mov.b64 k, {%4, %4}; mul.rn.f32x2 v, v, k; mov.b64 {%0, %1}, v; }"
        : "=f"(a), "=f"(b) : "f"(x[2 * i]), "f"(x[2 * i + 1]), "f"(inv));
    w[i] = to_codes<E5M2>(a, b);
  }
  *reinterpret_cast<uint2*>(p) = make_uint2(w[0] | (w[1] << 16), w[2] | (w[3] << 16));
}

template <typename H2>
__device__ __forceinline__ H2 as_pair(uint32_t w) { return *reinterpret_cast<const H2*>(&w); }

__device__ __forceinline__ float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// The warps of one half (K or V) of a unit meet at a barrier of their own, as halves need not meet equally often.
__device__ __forceinline__ void half_barrier(int bar, int parts) {
  asm volatile("bar.sync %0, %1;" ::"r"(bar), "r"(parts * 32) : "memory");
}

// Maximum over the warps of a half; slots: a word for each.
__device__ __forceinline__ uint32_t half_max(uint32_t x, uint32_t* slots, int bar, int parts, int part, int lane) {
  x = __reduce_max_sync(0xffffffffu, x);
  if (parts > 1) {
    if (lane == 0) slots[part] = x;
    half_barrier(bar, parts);
    for (int i = 0; i < parts; ++i) x = max(x, slots[i]);
  }
  return x;
}

// Smallest e with a <= F * 2^e for the finite fp32 of bits `a`, F = 1.75 * 2^8 or 1.75 * 2^15.
template <bool E5M2>
__device__ __forceinline__ int exponent_for(uint32_t a) {
  if (!a) return MSKV_KV8_EXP_MIN;
  const int e = (int)(a >> 23) - 127 - (E5M2 ? 15 : 8) + ((a & 0x7fffffu) > 0x600000u);
  return min(max(e, MSKV_KV8_EXP_MIN), MSKV_KV8_EXP_MAX);
}

// A page (one half, one warp's 16 rows of it) that only receives new 16-bit rows.  A lane takes 16 elements of a row and
// step, eight from each half of the row, packed in pairs.
template <int D, bool E5M2, int NT, bool VEC>
__device__ __forceinline__ void new_page(const char* rows0, int64_t stride, uint8_t* codes, int8_t* ex, uint8_t* bounds, int rows,
                                         int kv, int parts, int part, int bar, uint32_t* slots, uint32_t* slots2,
                                         float* s_lo, float* s_hi, int lane) {
  using H2 = std::conditional_t<NT == kNewBf16, __nv_bfloat162, __half2>;
  constexpr uint32_t kInf = NT == kNewBf16 ? 0x7f80u : 0x7c00u;
  constexpr int kLanes = D / 16, kRows = 32 / kLanes, kSteps = 16 / kRows;
  const int r0 = part * 16 + lane / kLanes, c = (lane % kLanes) * 8;
  const char* src = rows0 + r0 * stride + c * 2;
  uint32_t x[kSteps][8];
#pragma unroll
  for (int s = 0; s < kSteps; ++s)
    if (r0 + s * kRows < rows) {
      load8_packed<VEC>(src + s * kRows * stride, *reinterpret_cast<uint32_t(*)[4]>(&x[s][0]));
      load8_packed<VEC>(src + s * kRows * stride + D, *reinterpret_cast<uint32_t(*)[4]>(&x[s][4]));
    }
  // the lane's columns: their bounds, and of those the largest magnitude (NaN and infinities stay visible)
  H2 lo[8], hi[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    lo[i] = as_pair<H2>(kInf * 0x10001u);
    hi[i] = as_pair<H2>(kInf * 0x10001u | 0x80008000u);
  }
#pragma unroll
  for (int s = 0; s < kSteps; ++s)
    if (r0 + s * kRows < rows)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        lo[i] = __hmin2_nan(lo[i], as_pair<H2>(x[s][i]));
        hi[i] = __hmax2_nan(hi[i], as_pair<H2>(x[s][i]));
      }
  uint32_t top = 0;
  if (r0 < rows) {
    H2 most = as_pair<H2>(0u);
#pragma unroll
    for (int i = 0; i < 8; ++i) most = __hmax2_nan(most, __hmax2_nan(__habs2(lo[i]), __habs2(hi[i])));
    const uint32_t both = *reinterpret_cast<const uint32_t*>(&most) & 0x7fff7fffu;   // NaN: all ones
    top = max(both >> 16, both & 0xffffu);
  }
  top = half_max(top, slots, bar, parts, part, lane);
  if (top >= kInf) {                        // infinities or NaN: the maximum of the others
    uint32_t both = 0;
#pragma unroll
    for (int s = 0; s < kSteps; ++s)
      if (r0 + s * kRows < rows)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const uint32_t m = x[s][i] & 0x7fff7fffu;
          both = __vmaxu2(both, m & __vcmpltu2(m, kInf * 0x10001u));
        }
    top = half_max(max(both >> 16, both & 0xffffu), slots2, bar, parts, part, lane);
  }
  const int e = exponent_for<E5M2>(NT == kNewBf16 ? top << 16 : __float_as_uint(__half2float(__ushort_as_half((uint16_t)top))));
  const float inv = pow2i(-e);
#pragma unroll
  for (int s = 0; s < kSteps; ++s)
    if (r0 + s * kRows < rows) {
      uint8_t* dst = codes + (r0 + s * kRows) * D + c;
      float f[8];
      unpack8<NT>(*reinterpret_cast<const uint32_t(*)[4]>(&x[s][0]), f);
      store_codes<E5M2>(dst, f, inv);
      unpack8<NT>(*reinterpret_cast<const uint32_t(*)[4]>(&x[s][4]), f);
      store_codes<E5M2>(dst + D / 2, f, inv);
    }
  if (part == 0 && lane == 0) *ex = (int8_t)e;
  if (kv || !bounds) return;
#pragma unroll
  for (int o = kLanes; o < 32; o <<= 1)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      lo[i] = __hmin2_nan(lo[i], __shfl_xor_sync(0xffffffffu, lo[i], o));
      hi[i] = __hmax2_nan(hi[i], __shfl_xor_sync(0xffffffffu, hi[i], o));
    }
  if (lane >= kLanes && parts == 1) return;
  float l[16], m[16];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    l[2 * i] = __low2float(lo[i]); l[2 * i + 1] = __high2float(lo[i]);
    m[2 * i] = __low2float(hi[i]); m[2 * i + 1] = __high2float(hi[i]);
  }
  if (parts > 1) {
    if (lane < kLanes)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int d = part * D + (i >> 3) * (D / 2) + c + (i & 7);
        s_lo[d] = l[i];
        s_hi[d] = m[i];
      }
    half_barrier(bar, parts);
    if (part || lane >= kLanes) return;
    for (int q = 1; q < parts; ++q)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int d = q * D + (i >> 3) * (D / 2) + c + (i & 7);
        l[i] = min_nan(l[i], s_lo[d]);
        m[i] = max_nan(m[i], s_hi[d]);
      }
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    store_codes<E5M2>(bounds + i * (D / 2) + c, *reinterpret_cast<const float(*)[8]>(&l[8 * i]), inv);
    store_codes<E5M2>(bounds + D + i * (D / 2) + c, *reinterpret_cast<const float(*)[8]>(&m[8 * i]), inv);
  }
}

// kFew: few units (see the launch).  Every page's rows then go through fp32 and are loaded together (eight steps;
// fp32 rows four), whatever registers that takes; otherwise a page of new rows is kept packed and others take
// four steps at a time, so that 64 registers do and 32 warps fit an SM.
template <int D, bool E5M2, int NT, bool VEC, bool kFew>
__global__ void __launch_bounds__(512, !kFew && D <= 128 && NT != kNewF32 ? 2 : 1) kv8_append_kernel(const AppendDev a) {
  constexpr int kLanes = D / 8;             // lanes of a row
  constexpr int kRows = 32 / kLanes;        // rows of a step
  constexpr int kSteps = 16 / kRows;
  constexpr int kElem = NT == kNewF32 ? 4 : 2;
  __shared__ uint32_t s_max[2][16];
  __shared__ float s_lo[8][D], s_hi[8][D];

  const int parts = a.pg.page_size >> 4;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int group = a.units == 1 ? 0 : a.parts_log2 >= 0 ? warp >> (a.parts_log2 + 1) : warp / (2 * parts);
  const int in_group = warp - group * 2 * parts;
  const int kv = in_group >= parts, part = in_group - kv * parts;
  const int bar = 1 + 2 * group + kv;       // a barrier for the warps of each half
  wait_for_previous_grid();
  allow_dependents();
  const uint32_t unit = blockIdx.x * a.units + group;
  if (unit >= a.all_units) return;
  const uint32_t bh = a.by_touched.quotient(unit), j = unit - bh * a.touched;
  const int b = (int)a.by_heads.quotient(bh), h = (int)(bh - b * a.pg.heads);

  // the page and its rows; every exit before the barriers is taken by the whole unit
  const int tok0 = a.tok0[b];
  const int n = a.counts ? min(max(a.counts[b], 0), a.num_tokens) : a.num_tokens;
  if (n == 0) return;
  if (tok0 < 0) {
    if (a.status && lane == 0) atomicOr(a.status, MSKV_STATUS_DST_OOB);
    return;
  }
  const int p = (a.parts_log2 >= 0 ? tok0 >> (a.parts_log2 + 4) : tok0 / a.pg.page_size) + (int)j;
  const int64_t t0 = (int64_t)p * a.pg.page_size;
  const int64_t end = (int64_t)tok0 + n;
  if (t0 >= end) return;
  if (p >= a.pg.max_pages) {
    if (a.status && lane == 0) atomicOr(a.status, MSKV_STATUS_DST_OOB);
    return;
  }
  const int64_t page = a.pg.page_table[(int64_t)b * a.pg.pt_stride + p];
  if (page < 0 || page >= a.pg.num_pages) {
    if (a.status && lane == 0) atomicOr(a.status, MSKV_STATUS_BAD_PAGE);
    return;
  }
  uint8_t* const codes = (kv ? a.pg.v : a.pg.k) + page * a.pg.sp + (int64_t)h * a.pg.sh;
  int8_t* const ex = a.pg.exps + (page * a.pg.heads + h) * 2 + kv;
  const int first_new = (int)max((int64_t)tok0 - t0, (int64_t)0);                  // rows [0, first_new) are old
  const int rows = (int)min(end - t0, (int64_t)a.pg.page_size);           // rows [0, rows) are held
  const int e_old = first_new ? *ex : 0;
  const int r0 = part * 16 + lane / kLanes, d0 = (lane % kLanes) * 8;
  const char* const src = a.x[kv] + (int64_t)b * a.sb[kv] + (int64_t)h * a.sh[kv] + (t0 + r0 - tok0) * a.st[kv] + d0 * kElem;
  const int64_t step = (int64_t)kRows * a.st[kv];

  float lo[8], hi[8];                       // of the K rows, for the lane's elements
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    lo[i] = INFINITY;
    hi[i] = -INFINITY;
  }
  if constexpr (NT != kNewF32 && !kFew) {
    if (first_new == 0) {
      const char* rows0 = a.x[kv] + (int64_t)b * a.sb[kv] + (int64_t)h * a.sh[kv] + (t0 - tok0) * a.st[kv];
      new_page<D, E5M2, NT, VEC>(rows0, a.st[kv], codes, ex, a.pg.bounds ? a.pg.bounds + (page * a.pg.heads + h) * 2 * D : nullptr,
                                 rows, kv, parts, part, bar, s_max[0] + warp - part, s_max[1] + warp - part, s_lo[group * parts],
                                 s_hi[group * parts], lane);
      return;
    }
  }
  {
    const float f_old = pow2i(e_old);
    // a batch of steps: their loads, then their values
    constexpr int kMost = kFew && NT != kNewF32 ? 8 : 4, kBatch = kSteps < kMost ? kSteps : kMost;
    uint32_t w[kBatch][kElem * 2];
    const auto load_batch = [&](int s0) {
#pragma unroll
      for (int k = 0; k < kBatch; ++k) load_row<NT, VEC>(r0 + (s0 + k) * kRows, first_new, rows, codes, D, d0, src + (s0 + k) * step, w[k]);
    };
    uint32_t top = 0;                       // fp32 magnitudes order as their bits, non-finite ones count as 0
#pragma unroll 1
    for (int s0 = 0; s0 < kSteps; s0 += kBatch) {
      load_batch(s0);
#pragma unroll
      for (int k = 0; k < kBatch; ++k) {
        const int r = r0 + (s0 + k) * kRows;
        if (r >= rows) continue;
        float x[8];
        row_values<E5M2, NT>(r < first_new, w[k], f_old, x);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const uint32_t u = __float_as_uint(x[i]) & 0x7fffffffu;
          top = max(top, u < 0x7f800000u ? u : 0u);
          lo[i] = min_nan(lo[i], x[i]);
          hi[i] = max_nan(hi[i], x[i]);
        }
      }
    }
    top = half_max(top, s_max[0] + warp - part, bar, parts, part, lane);
    const int e = exponent_for<E5M2>(top);
    const float inv = pow2i(-e);
    const int r_from = first_new && e == e_old ? first_new : 0;
#pragma unroll 1
    for (int s0 = 0; s0 < kSteps; s0 += kBatch) {
      if constexpr (kSteps > kBatch) load_batch(s0);      // again, from the caches
#pragma unroll
      for (int k = 0; k < kBatch; ++k) {
        const int r = r0 + (s0 + k) * kRows;
        if (r >= rows || r < r_from) continue;
        float x[8];
        row_values<E5M2, NT>(r < first_new, w[k], f_old, x);
        store_codes<E5M2>(codes + r * D + d0, x, inv);
      }
    }
    if (part == 0 && lane == 0) *ex = (int8_t)e;
    if (!a.pg.bounds) return;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      lo[i] *= inv;
      hi[i] *= inv;
    }
  }

  // bounds over the rows of the warp, then of the warps
  if (kv) return;
#pragma unroll
  for (int o = kLanes; o < 32; o <<= 1)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      lo[i] = min_nan(lo[i], __shfl_xor_sync(0xffffffffu, lo[i], o));
      hi[i] = max_nan(hi[i], __shfl_xor_sync(0xffffffffu, hi[i], o));
    }
  if (parts > 1) {
    const int first = group * parts;
    if (lane < kLanes)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        s_lo[first + part][d0 + i] = lo[i];
        s_hi[first + part][d0 + i] = hi[i];
      }
    half_barrier(bar, parts);
    if (part == 0 && lane < kLanes)
      for (int q = 1; q < parts; ++q)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          lo[i] = min_nan(lo[i], s_lo[first + q][d0 + i]);
          hi[i] = max_nan(hi[i], s_hi[first + q][d0 + i]);
        }
  }
  if (part == 0 && lane < kLanes) {
    uint8_t* const bd = a.pg.bounds + (page * a.pg.heads + h) * 2 * D + d0;
    store_codes<E5M2>(bd, lo, 1.f);
    store_codes<E5M2>(bd + D, hi, 1.f);
  }
}

template <int D, bool E5M2, int NT>
static int launch_append(const AppendDev& a, bool vec, bool few, int64_t ctas, cudaStream_t st) {
  const int threads = a.units * a.pg.page_size / 16 * 64;
  cudaError_t launched = cudaSuccess;
  const auto go = [&](auto kernel) { launched = launch_dependent(kernel, dim3((unsigned)ctas), dim3(threads), 0, st, a); };
  if (vec) few ? go(kv8_append_kernel<D, E5M2, NT, true, true>) : go(kv8_append_kernel<D, E5M2, NT, true, false>);
  else few ? go(kv8_append_kernel<D, E5M2, NT, false, true>) : go(kv8_append_kernel<D, E5M2, NT, false, false>);
  if (launched != cudaSuccess) return cuda_status(launched, "mskv_kv8_append launch");
  return after_launch("mskv_kv8_append");
}

template <int D, bool E5M2>
static int append_type(const AppendDev& a, int dtype, bool vec, bool few, int64_t ctas, cudaStream_t st) {
  switch (dtype) {
    case MSKV_DT_BF16: return launch_append<D, E5M2, kNewBf16>(a, vec, few, ctas, st);
    case MSKV_DT_F16: return launch_append<D, E5M2, kNewF16>(a, vec, few, ctas, st);
    default: return launch_append<D, E5M2, kNewF32>(a, vec, few, ctas, st);
  }
}

template <int D>
static int append_cache(const AppendDev& a, bool e5m2, int dtype, bool vec, bool few, int64_t ctas, cudaStream_t st) {
  return e5m2 ? append_type<D, true>(a, dtype, vec, few, ctas, st) : append_type<D, false>(a, dtype, vec, few, ctas, st);
}

}  // namespace mskv

using namespace mskv;

extern "C" int mskv_kv8_append(const mskv_kv8_append_desc* d, void* stream) {
  if (!d) return fail(MSKV_ERR_ARG, "mskv_kv8_append: NULL descriptor");
  if (const int rc = check_kv8(d->pages, "mskv_kv8_append")) return rc;
  if (d->dtype != MSKV_DT_BF16 && d->dtype != MSKV_DT_F16 && d->dtype != MSKV_DT_F32)
    return fail(MSKV_ERR_DTYPE, "mskv_kv8_append: new rows must be bf16, f16 or f32");
  if (d->num_tokens < 0) return fail(MSKV_ERR_ARG, "mskv_kv8_append: negative num_tokens");
  if (d->num_tokens == 0) return MSKV_OK;
  if (!d->k_new || !d->v_new || !d->tok0) return fail(MSKV_ERR_ARG, "mskv_kv8_append: NULL k_new, v_new or tok0");
  if (const int rc = check_words("mskv_kv8_append", d->tok0, d->counts, d->status)) return rc;
  const int elem = d->dtype == MSKV_DT_F32 ? 4 : 2;
  const uintptr_t k_bits = (uintptr_t)d->k_new | (uintptr_t)d->k_stride_b | (uintptr_t)d->k_stride_h | (uintptr_t)d->k_stride_t;
  const uintptr_t v_bits = (uintptr_t)d->v_new | (uintptr_t)d->v_stride_b | (uintptr_t)d->v_stride_h | (uintptr_t)d->v_stride_t;
  if ((k_bits | v_bits) & (elem - 1)) return fail(MSKV_ERR_ARG, "mskv_kv8_append: rows must be aligned to their elements");
  AppendDev a{};
  a.pg = to_dev(d->pages);
  a.x[0] = static_cast<const char*>(d->k_new);
  a.x[1] = static_cast<const char*>(d->v_new);
  a.sb[0] = d->k_stride_b; a.sh[0] = d->k_stride_h; a.st[0] = d->k_stride_t;
  a.sb[1] = d->v_stride_b; a.sh[1] = d->v_stride_h; a.st[1] = d->v_stride_t;
  a.tok0 = d->tok0;
  a.counts = d->counts;
  a.status = d->status;
  a.num_tokens = d->num_tokens;
  a.touched = (uint32_t)(((int64_t)d->num_tokens + a.pg.page_size - 2) / a.pg.page_size + 1);
  const int64_t all = (int64_t)a.touched * a.pg.batch * a.pg.heads;
  if (all > INT_MAX) return fail(MSKV_ERR_RANGE, "mskv_kv8_append: too many rows for one call");
  a.all_units = (uint32_t)all;
  a.by_touched = Divisor(a.touched);
  a.by_heads = Divisor((uint32_t)a.pg.heads);
  const int parts = a.pg.page_size / 16;
  a.parts_log2 = parts & (parts - 1) ? -1 : parts >= 8 ? 3 : parts >> 1;
  // Few units: one a CTA and all of a page's rows loaded together; more: up to 8 warps a CTA, in fewer registers.  128 dims,
  // bf16, pages of 16: 32 units 3.4 us against 4.8, 576 units 4.1 against 5.8, 1088 units 7.2 against 6.4, 2176
  // units 14.5 against 8.7.
  const bool few = all <= 4 * (int64_t)sms_of_device();
  a.units = few ? 1 : (uint32_t)std::max(1, 64 / a.pg.page_size);
  const int64_t ctas = (all + a.units - 1) / a.units;
  const bool vec = ((k_bits | v_bits) & 15) == 0;   // 16-byte loads; other layouts element by element
  const bool e5m2 = d->pages.dtype == MSKV_DT_FP8_E5M2;
  const cudaStream_t st = as_stream(stream);
  switch (d->pages.head_dim) {
    case 64: return append_cache<64>(a, e5m2, d->dtype, vec, few, ctas, st);
    case 128: return append_cache<128>(a, e5m2, d->dtype, vec, few, ctas, st);
    default: return append_cache<256>(a, e5m2, d->dtype, vec, few, ctas, st);
  }
}
