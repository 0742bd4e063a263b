// Append to the 8-bit paged cache (mskv_kv8_append).
//
// A page of one KV head is quantised as a whole: x[t,d] are the values it holds after the append
// (tokens before tok0 as code * 2^e_old, new ones as given), a = max finite |x|, e the smallest
// exponent with a <= F * 2^e (F = 448 = 1.75 * 2^8 for e4m3, 57344 = 1.75 * 2^15 for e5m2), and
// code = rn(x * 2^-e).  The multiplication by a power of two is exact, so a code has one
// rounding; a page whose exponent a later token raises keeps its codes but for f8 subnormals.
//
// One CTA per (page, KV head): page_size/16 warps for K and as many for V, each holding 16
// rows of its half in registers (8 elements of a row per lane and step), so every new row is
// read once, and the maximum (an integer maximum over the bits of |x|) and the K bounds are
// taken from registers.  Old rows are stored again only when the exponent changed.
#include "kv8.cuh"

namespace mskv {

struct AppendDev {
  Kv8Dev pg;
  const char* x[2];                 // K, V rows
  int64_t sb[2], sh[2], st[2];
  const int32_t* tok0;
  const int32_t* counts;
  uint32_t* status;
  int32_t num_tokens, touched;      // touched: pages of a sequence that num_tokens rows can reach
};

enum NewType { kNewBf16 = 0, kNewF16 = 1, kNewF32 = 2 };

template <int NT, bool VEC>
__device__ __forceinline__ void load8(const char* p, float (&x)[8]) {
  if constexpr (NT == kNewF32) {
    if constexpr (VEC) {
      const uint4 a = ld_stream16(p), b = ld_stream16(p + 16);
      const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = __uint_as_float(w[i]);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = reinterpret_cast<const float*>(p)[i];
    }
  } else {
    uint32_t w[4];
    if constexpr (VEC) {
      const uint4 a = ld_stream16(p);
      w[0] = a.x; w[1] = a.y; w[2] = a.z; w[3] = a.w;
    } else {
      const uint16_t* s = reinterpret_cast<const uint16_t*>(p);
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = (uint32_t)s[2 * i] | ((uint32_t)s[2 * i + 1] << 16);
    }
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
}

template <int D, bool E5M2, int NT, bool VEC>
__global__ void __launch_bounds__(512) kv8_append_kernel(const AppendDev a) {
  constexpr int kLanes = D / 8;             // lanes of a row
  constexpr int kRows = 32 / kLanes;        // rows of a step
  constexpr int kSteps = 16 / kRows;
  constexpr int kElem = NT == kNewF32 ? 4 : 2;
  __shared__ uint32_t s_max[2][8];
  __shared__ __half2 s_lo[8][D / 2], s_hi[8][D / 2];

  const int parts = a.pg.page_size / 16;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int kv = warp / parts, part = warp % parts;
  const int j = blockIdx.x % a.touched;
  const int bh = blockIdx.x / a.touched;
  const int b = bh / a.pg.heads, h = bh % a.pg.heads;

  // the page and its rows; every exit before the barriers is taken by the whole CTA
  const int64_t tok0 = a.tok0[b];
  const int n = a.counts ? min(max(a.counts[b], 0), a.num_tokens) : a.num_tokens;
  if (n == 0) return;
  if (tok0 < 0) {
    if (a.status && threadIdx.x == 0) atomicOr(a.status, MSKV_STATUS_DST_OOB);
    return;
  }
  const int64_t p = tok0 / a.pg.page_size + j;
  const int64_t t0 = p * a.pg.page_size;
  const int64_t end = tok0 + n;
  if (t0 >= end) return;
  if (p >= a.pg.max_pages) {
    if (a.status && threadIdx.x == 0) atomicOr(a.status, MSKV_STATUS_DST_OOB);
    return;
  }
  const int64_t page = a.pg.page_table[(int64_t)b * a.pg.pt_stride + p];
  if (page < 0 || page >= a.pg.num_pages) {
    if (a.status && threadIdx.x == 0) atomicOr(a.status, MSKV_STATUS_BAD_PAGE);
    return;
  }
  uint8_t* const codes = (kv ? a.pg.v : a.pg.k) + page * a.pg.sp + (int64_t)h * a.pg.sh;
  int8_t* const ex = a.pg.exps + (page * a.pg.heads + h) * 2 + kv;
  const int first_new = (int)max(tok0 - t0, (int64_t)0);                  // rows [0, first_new) are old
  const int rows = (int)min(end - t0, (int64_t)a.pg.page_size);           // rows [0, rows) are held
  const int e_old = first_new ? *ex : 0;
  const int r0 = part * 16 + lane / kLanes, d0 = (lane % kLanes) * 8;

  float x[kSteps][8];
#pragma unroll
  for (int s = 0; s < kSteps; ++s) {
    const int r = r0 + s * kRows;
    if (r >= first_new && r < rows) {
      const char* src = a.x[kv] + (int64_t)b * a.sb[kv] + (int64_t)h * a.sh[kv] + (t0 + r - tok0) * a.st[kv] + d0 * kElem;
      load8<NT, VEC>(src, x[s]);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[s][i] = 0.f;
    }
  }
  if (part * 16 < first_new) {
    const float f = pow2i(e_old);
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      const int r = r0 + s * kRows;
      if (r < first_new) {
        const uint2 c = *reinterpret_cast<const uint2*>(codes + (int64_t)r * D + d0);
        const uint32_t w[2] = {c.x, c.y};
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          uint32_t lo, hi;
          codes_to_half<E5M2>(w[i], lo, hi);
          const float2 u = __half22float2(*reinterpret_cast<const __half2*>(&lo));
          const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&hi));
          x[s][4 * i] = u.x * f; x[s][4 * i + 1] = u.y * f; x[s][4 * i + 2] = v.x * f; x[s][4 * i + 3] = v.y * f;
        }
      }
    }
  }

  // the largest finite magnitude: fp32 magnitudes order as their bits, non-finite ones count as 0
  uint32_t top = 0;
#pragma unroll
  for (int s = 0; s < kSteps; ++s)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t u = __float_as_uint(x[s][i]) & 0x7fffffffu;
      top = max(top, u < 0x7f800000u ? u : 0u);
    }
  top = __reduce_max_sync(0xffffffffu, top);
  if (parts > 1) {
    if (lane == 0) s_max[kv][part] = top;
    __syncthreads();
    for (int i = 0; i < parts; ++i) top = max(top, s_max[kv][i]);
  }
  int e = MSKV_KV8_EXP_MIN;
  if (top) {
    e = (int)(top >> 23) - 127 - (E5M2 ? 15 : 8) + ((top & 0x7fffffu) > 0x600000u);
    e = min(max(e, MSKV_KV8_EXP_MIN), MSKV_KV8_EXP_MAX);
  }

  const float inv = pow2i(-e);
  const bool keep_old = first_new && e == e_old;
  __half2 lo[4], hi[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    lo[i] = __half2half2(__ushort_as_half(0x7c00));
    hi[i] = __half2half2(__ushort_as_half(0xfc00));
  }
#pragma unroll
  for (int s = 0; s < kSteps; ++s) {
    const int r = r0 + s * kRows;
    if (r < rows) {
      uint2 c;
      c.x = to_codes<E5M2>(x[s][0] * inv, x[s][1] * inv) | (to_codes<E5M2>(x[s][2] * inv, x[s][3] * inv) << 16);
      c.y = to_codes<E5M2>(x[s][4] * inv, x[s][5] * inv) | (to_codes<E5M2>(x[s][6] * inv, x[s][7] * inv) << 16);
      if (r >= first_new || !keep_old) *reinterpret_cast<uint2*>(codes + (int64_t)r * D + d0) = c;
      if (kv == 0) {
        uint32_t f[4];
        codes_to_half<E5M2>(c.x, f[0], f[1]);
        codes_to_half<E5M2>(c.y, f[2], f[3]);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const __half2 v = *reinterpret_cast<const __half2*>(&f[i]);
          lo[i] = __hmin2_nan(lo[i], v);
          hi[i] = __hmax2_nan(hi[i], v);
        }
      }
    }
  }
  if (part == 0 && lane == 0) *ex = (int8_t)e;

  if (!a.pg.bounds) return;                 // the same for every thread of the launch
  if (kv == 0) {
#pragma unroll
    for (int o = kLanes; o < 32; o <<= 1)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        lo[i] = __hmin2_nan(lo[i], __shfl_xor_sync(0xffffffffu, lo[i], o));
        hi[i] = __hmax2_nan(hi[i], __shfl_xor_sync(0xffffffffu, hi[i], o));
      }
  }
  if (parts > 1) {
    if (kv == 0 && lane < kLanes)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        s_lo[part][d0 / 2 + i] = lo[i];
        s_hi[part][d0 / 2 + i] = hi[i];
      }
    __syncthreads();
    if (kv == 0 && part == 0 && lane < kLanes)
      for (int q = 1; q < parts; ++q)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          lo[i] = __hmin2_nan(lo[i], s_lo[q][d0 / 2 + i]);
          hi[i] = __hmax2_nan(hi[i], s_hi[q][d0 / 2 + i]);
        }
  }
  if (kv == 0 && part == 0 && lane < kLanes) {
    // the bounds are codes of the page, so these conversions are exact
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float2 u0 = __half22float2(lo[2 * i]), u1 = __half22float2(lo[2 * i + 1]);
      const float2 v0 = __half22float2(hi[2 * i]), v1 = __half22float2(hi[2 * i + 1]);
      w[i] = to_codes<E5M2>(u0.x, u0.y) | (to_codes<E5M2>(u1.x, u1.y) << 16);
      w[2 + i] = to_codes<E5M2>(v0.x, v0.y) | (to_codes<E5M2>(v1.x, v1.y) << 16);
    }
    uint8_t* const bd = a.pg.bounds + (page * a.pg.heads + h) * 2 * D + d0;
    *reinterpret_cast<uint2*>(bd) = make_uint2(w[0], w[1]);
    *reinterpret_cast<uint2*>(bd + D) = make_uint2(w[2], w[3]);
  }
}

template <int D, bool E5M2, int NT>
static int launch_append(const AppendDev& a, bool vec, int64_t ctas, cudaStream_t st) {
  const int threads = a.pg.page_size / 16 * 64;
  if (vec) kv8_append_kernel<D, E5M2, NT, true><<<(unsigned)ctas, threads, 0, st>>>(a);
  else kv8_append_kernel<D, E5M2, NT, false><<<(unsigned)ctas, threads, 0, st>>>(a);
  return after_launch("mskv_kv8_append");
}

template <int D, bool E5M2>
static int append_type(const AppendDev& a, int dtype, bool vec, int64_t ctas, cudaStream_t st) {
  switch (dtype) {
    case MSKV_DT_BF16: return launch_append<D, E5M2, kNewBf16>(a, vec, ctas, st);
    case MSKV_DT_F16: return launch_append<D, E5M2, kNewF16>(a, vec, ctas, st);
    default: return launch_append<D, E5M2, kNewF32>(a, vec, ctas, st);
  }
}

template <int D>
static int append_cache(const AppendDev& a, bool e5m2, int dtype, bool vec, int64_t ctas, cudaStream_t st) {
  return e5m2 ? append_type<D, true>(a, dtype, vec, ctas, st) : append_type<D, false>(a, dtype, vec, ctas, st);
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
  a.touched = (int)(((int64_t)d->num_tokens + a.pg.page_size - 2) / a.pg.page_size + 1);
  const int64_t ctas = (int64_t)a.touched * a.pg.batch * a.pg.heads;
  if (ctas > INT_MAX) return fail(MSKV_ERR_RANGE, "mskv_kv8_append: too many rows for one call");
  const bool vec = ((k_bits | v_bits) & 15) == 0;   // 16-byte loads; other layouts element by element
  const bool e5m2 = d->pages.dtype == MSKV_DT_FP8_E5M2;
  const cudaStream_t st = as_stream(stream);
  switch (d->pages.head_dim) {
    case 64: return append_cache<64>(a, e5m2, d->dtype, vec, ctas, st);
    case 128: return append_cache<128>(a, e5m2, d->dtype, vec, ctas, st);
    default: return append_cache<256>(a, e5m2, d->dtype, vec, ctas, st);
  }
}
