// Attention over the 8-bit paged cache, whole or over listed pages (mskv_kv8_attention).
//
//   s[r,t] = scale * q[r] . k8[t] * 2^eK(page of t),   o[r] = sum_t softmax(s[r])_t v8[t] * 2^eV(page of t)
//
// for the R = (q_heads/kv_heads) * q_len query rows of a KV head, from one pass over its codes.
//
// Mathematics.  Work unit: a tile of 16 tokens, which lies in one page, so both scales are one
// number.  With base-2 logarithms and t' = s * log2(e) + eV, the second product's weights
// P = 2^(t' - m) carry V's scale (m: running reference of t' over the tiles), the codes v8 enter it
// unscaled, and the softmax denominator is sum P * 2^-eV.  Exponents within [-60, 60] keep
// the term of the largest s above 2^-121 and so in fp32's normal range.  m moves only when a t'
// exceeds it by more than 8 (then P <= 2^8 until the next move): most tiles need one vote
// instead of a maximum over the warp.
// q is scaled per row to a largest magnitude in [1, 2) and enters as fp16 (a bf16 or fp16 value
// keeps all its bits down to 2^-14 of the row's largest; below, it is off by at most 2^-25 of that).
// K and V codes are exact in fp16.  P is rounded to fp16 (relative 2^-11); for fp16 outputs
// its remainder enters as a second fp16 term, as one term alone would be as far off as the output's
// own rounding.  All sums are fp32.
//
// Bound by the codes' bytes (2D a token and KV head).  mma.sync m16n8k16 with the tokens on M:
// S^T = K Q^T, O^T = V^T P^T, so the 8 columns hold the query rows (16 rows: two column tiles).
// A warp owns a tile: 16-byte loads straight from global memory into the fragments' registers -- the
// contraction's order is free, so a lane's 16 contiguous codes of a K row are four k-steps', and
// those of four V rows are eight row tiles' (byte permutations pair the tokens) -- no shared memory and
// no barrier on the way; K of the next tile is in flight during the softmax, V during the next product.
// A tcgen05 MMA would need 64 or 128 rows of f16 operands staged in shared memory after a
// conversion there; the legacy pipe is a fifth busy at the memory's speed.
//
// Split: all tiles of all (sequence, KV head, row tile) segments form one line, cut into equal parts
// for the CTAs however ragged the lengths are (a scan over the lengths in every CTA).  The 8 warps of a
// CTA take a segment's tiles in turn and merge in shared memory; a segment cut by a CTA border goes
// through the workspace and a second kernel.  Segments of few tiles go to one CTA each
// and need neither.
#include <math.h>

#include <algorithm>

#include "kv8.cuh"

namespace mskv {

struct Kv8AttnDev {
  Kv8Dev pg;
  const char* q;
  int64_t q_sb, q_sh, q_sq;
  char* out;
  int64_t o_sb, o_sh, o_sq;
  const int32_t* lens;
  const int32_t* blocks;
  int64_t blk_sb, blk_sh;
  const int32_t* counts;
  int4* info;                      // [segments]: first and last CTA of a cut segment, slot in the first
  float* part_ml;                  // [2 * CTAs][rows][2]
  float* part_o;                   // [2 * CTAs][rows][D]
  uint32_t* status;
  float scale_log2;
  int32_t group, q_len, rows, row_tiles, segments, max_tokens, width, whole;   // whole: a CTA per segment
  int32_t vec_q, pow2_page;
};

constexpr int kKaWarps = 8;
constexpr int kKaThreads = kKaWarps * 32;
constexpr float kNoMax = -1e30f;

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

__device__ __forceinline__ int kv8_len(const Kv8AttnDev& a, int b) { return min(max(a.lens[b], 0), a.max_tokens); }

// Tiles of (b, h).
__device__ __forceinline__ int kv8_tiles(const Kv8AttnDev& a, int b, int h) {
  if (!a.blocks) return (kv8_len(a, b) + 15) >> 4;
  const int n = a.counts ? min(max(a.counts[(int64_t)b * a.pg.heads + h], 0), a.width) : a.width;
  return n * (a.pg.page_size >> 4);
}

// Bytes that are no finite code, as 0xff; others 0.
template <bool E5M2>
__device__ __forceinline__ uint32_t nonfinite_bytes(uint32_t w) {
  return E5M2 ? __vcmpgtu4(w & 0x7f7f7f7fu, 0x7b7b7b7bu) : __vcmpeq4(w & 0x7f7f7f7fu, 0x7f7f7f7fu);
}

template <int D, int NT, bool E5M2, bool BF16>
struct Kv8Attn {
  static constexpr int kRows = NT * 8;
  static constexpr int kKVec = D / 64;            // 16-byte loads of a lane per K row
  static constexpr int kVWords = D / 32;          // words of a lane per V row
  static constexpr int kOT = D / 16;              // row tiles of O^T
  static constexpr int kOStride = D + 4;          // floats between rows of the merge buffer
  static constexpr bool kTwoTerms = !BF16;        // P as two fp16 terms

  struct Smem {
    float m[kKaWarps][kRows], l[kKaWarps][kRows];
    float o[kKaWarps][kRows][kOStride];
  };

  uint32_t qf[NT][kKVec * 4][2];
  float f[NT][2];                                 // scale * log2(e) * 2^(row exponent) of the lane's two columns
  float m[NT][2], l[NT][2];
  float o[NT][kOT][4];
  int lim[NT][2];                                 // tokens that the two columns see

  // Query rows of the segment as B fragments; column n = lane/4 of column tile nt is row
  // 8*(row tile*NT + nt) + n = position * group + head.
  __device__ __forceinline__ void load_q(const Kv8AttnDev& a, int b, int h, int rt, int len, int lane) {
    const int g = lane >> 2, c = lane & 3;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int r = (rt * NT + nt) * 8 + g;
      float x[kKVec][16];
      if (r < a.rows) {
        const int pos = r / a.group, head = h * a.group + r % a.group;
        const char* src = a.q + (int64_t)b * a.q_sb + (int64_t)head * a.q_sh + (int64_t)pos * a.q_sq + 32 * c;
#pragma unroll
        for (int v = 0; v < kKVec; ++v) {
          uint32_t w[8];
          if (a.vec_q) {
            const uint4 p0 = *reinterpret_cast<const uint4*>(src + 128 * v);
            const uint4 p1 = *reinterpret_cast<const uint4*>(src + 128 * v + 16);
            w[0] = p0.x; w[1] = p0.y; w[2] = p0.z; w[3] = p0.w; w[4] = p1.x; w[5] = p1.y; w[6] = p1.z; w[7] = p1.w;
          } else {
            const uint16_t* s = reinterpret_cast<const uint16_t*>(src + 128 * v);
#pragma unroll
            for (int i = 0; i < 8; ++i) w[i] = (uint32_t)s[2 * i] | ((uint32_t)s[2 * i + 1] << 16);
          }
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            if constexpr (BF16) {
              x[v][2 * i] = __uint_as_float(w[i] << 16);
              x[v][2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
            } else {
              const float2 y = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
              x[v][2 * i] = y.x;
              x[v][2 * i + 1] = y.y;
            }
          }
        }
      } else {
#pragma unroll
        for (int v = 0; v < kKVec; ++v)
#pragma unroll
          for (int i = 0; i < 16; ++i) x[v][i] = 0.f;
      }
      uint32_t top = 0;
#pragma unroll
      for (int v = 0; v < kKVec; ++v)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const uint32_t u = __float_as_uint(x[v][i]) & 0x7fffffffu;
          top = max(top, u < 0x7f800000u ? u : 0u);
        }
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const int e = top ? min(max((int)(top >> 23) - 127, -120), 120) : 0;
      const float inv = pow2i(-e);
#pragma unroll
      for (int v = 0; v < kKVec; ++v)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          qf[nt][v * 4 + i][0] = pack_half2(x[v][4 * i] * inv, x[v][4 * i + 1] * inv);
          qf[nt][v * 4 + i][1] = pack_half2(x[v][4 * i + 2] * inv, x[v][4 * i + 3] * inv);
        }
      const float row_f = a.scale_log2 * pow2i(e);
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        f[nt][k] = __shfl_sync(0xffffffffu, row_f, (2 * c + k) * 4);
        const int rc = (rt * NT + nt) * 8 + 2 * c + k;
        lim[nt][k] = len - a.q_len + 1 + (rc < a.rows ? rc / a.group : a.q_len - 1);
        m[nt][k] = kNoMax;
        l[nt][k] = 0.f;
      }
#pragma unroll
      for (int i = 0; i < kOT; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k) o[nt][i][k] = 0.f;
    }
  }

  struct Tile {                                   // warp-uniform
    int page, tok, exps;                          // page < 0: nothing to read; exps: eK, eV
  };

  // Tile `i` of (b, h) as one lane sees it.
  static __device__ __forceinline__ Tile find(const Kv8AttnDev& a, int b, int h, int len, int i) {
    const int parts = a.pg.page_size >> 4;
    int pi = i / parts;
    const int part = i - pi * parts;
    Tile t;
    t.page = -1;
    t.tok = 0;
    t.exps = 0;
    if (a.blocks) {
      pi = a.blocks[(int64_t)b * a.blk_sb + (int64_t)h * a.blk_sh + pi];
      if (pi < 0 || pi >= a.pg.max_pages) {
        if (a.status) atomicOr(a.status, MSKV_STATUS_INDEX_OOB);
        return t;
      }
    }
    const int64_t tok = (int64_t)pi * a.pg.page_size + part * 16;
    if (tok >= len) return t;                     // a listed page's rows behind the sequence
    const int page = a.pg.page_table[(int64_t)b * a.pg.pt_stride + pi];
    if (page < 0 || page >= a.pg.num_pages) {
      if (a.status) atomicOr(a.status, MSKV_STATUS_BAD_PAGE);
      return t;
    }
    t.page = page;
    t.tok = (int)tok;
    t.exps = *reinterpret_cast<const uint16_t*>(a.pg.exps + ((int64_t)page * a.pg.heads + h) * 2);
    return t;
  }

  // Page and position of the tile that `lane` looked up (its exponents: pick_exps, once the scores are there).
  static __device__ __forceinline__ Tile pick(const Tile& mine, int lane) {
    Tile t;
    t.page = __shfl_sync(0xffffffffu, mine.page, lane);
    t.tok = __shfl_sync(0xffffffffu, mine.tok, lane);
    t.exps = 0;
    return t;
  }

  // Row of the page that the tile begins with.
  static __device__ __forceinline__ int first_row(const Kv8AttnDev& a, const Tile& t) {
    return a.pow2_page ? t.tok & (a.pg.page_size - 1) : t.tok % a.pg.page_size;
  }

  uint4 kr[2][kKVec];                             // K rows lane/4 and lane/4 + 8
  uint32_t vr[4][kVWords];                        // V rows 2c, 2c+1, 2c+8, 2c+9

  // A tile whose 16 tokens all exist is loaded without tests; missing rows are zero.
  __device__ __forceinline__ void load_k(const Kv8AttnDev& a, const Tile& t, int h, int len, int lane) {
    if (t.page < 0) return;
    const int g = lane >> 2, c = lane & 3;
    const uint8_t* src = a.pg.k + (int64_t)t.page * a.pg.sp + (int64_t)h * a.pg.sh + (first_row(a, t) + g) * D + 16 * c;
    if (t.tok + 16 <= len) {
#pragma unroll
      for (int r = 0; r < 2; ++r)
#pragma unroll
        for (int v = 0; v < kKVec; ++v) kr[r][v] = ld_stream16(src + 8 * r * D + 64 * v);
    } else {
#pragma unroll
      for (int r = 0; r < 2; ++r)
#pragma unroll
        for (int v = 0; v < kKVec; ++v) {
          kr[r][v] = make_uint4(0u, 0u, 0u, 0u);
          if (t.tok + g + 8 * r < len) kr[r][v] = ld_stream16(src + 8 * r * D + 64 * v);
        }
    }
  }

  __device__ __forceinline__ void load_v_row(int r, const uint8_t* src) {
    if constexpr (D == 64) {
      const uint2 x = ld_stream8(src);
      vr[r][0] = x.x; vr[r][1] = x.y;
    } else {
#pragma unroll
      for (int u = 0; u < D / 128; ++u) {
        const uint4 x = ld_stream16(src + 128 * u);
        vr[r][4 * u] = x.x; vr[r][4 * u + 1] = x.y; vr[r][4 * u + 2] = x.z; vr[r][4 * u + 3] = x.w;
      }
    }
  }

  __device__ __forceinline__ void load_v(const Kv8AttnDev& a, const Tile& t, int h, int len, int lane) {
    if (t.page < 0) return;
    const int g = lane >> 2, c = lane & 3;
    const uint8_t* src = a.pg.v + (int64_t)t.page * a.pg.sp + (int64_t)h * a.pg.sh + (first_row(a, t) + 2 * c) * D
                         + g * (D == 64 ? 8 : 16);
    if (t.tok + 16 <= len) {
#pragma unroll
      for (int r = 0; r < 4; ++r) load_v_row(r, src + ((r >> 1) * 8 + (r & 1)) * D);
    } else {
#pragma unroll
      for (int r = 0; r < 4; ++r) {
#pragma unroll
        for (int i = 0; i < kVWords; ++i) vr[r][i] = 0u;
        if (t.tok + 2 * c + (r >> 1) * 8 + (r & 1) < len) load_v_row(r, src + ((r >> 1) * 8 + (r & 1)) * D);
      }
    }
  }

  // acc[row tile 2i and 2i + 1] += V words * B; f(i) gives the four words.
  template <typename W>
  static __device__ __forceinline__ void v_product(float (&acc0)[4], float (&acc1)[4], const W& w, uint32_t b0, uint32_t b1) {
    uint32_t x0, x1, y0, y1;
    codes_to_half<E5M2>(__byte_perm(w[0], w[1], 0x5140), x0, x1);
    codes_to_half<E5M2>(__byte_perm(w[2], w[3], 0x5140), y0, y1);
    mma_f16(acc0, x0, x1, y0, y1, b0, b1);
    codes_to_half<E5M2>(__byte_perm(w[0], w[1], 0x7362), x0, x1);
    codes_to_half<E5M2>(__byte_perm(w[2], w[3], 0x7362), y0, y1);
    mma_f16(acc1, x0, x1, y0, y1, b0, b1);
  }

  // Scores of the tile in kr; kr is free afterwards.
  __device__ __forceinline__ void scores(float (&s)[NT][4]) {
    float odd[NT][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int k = 0; k < 4; ++k) s[nt][k] = odd[nt][k] = 0.f;
#pragma unroll
    for (int v = 0; v < kKVec; ++v) {
      const uint32_t x[4] = {kr[0][v].x, kr[0][v].y, kr[0][v].z, kr[0][v].w};
      const uint32_t y[4] = {kr[1][v].x, kr[1][v].y, kr[1][v].z, kr[1][v].w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint32_t a0, a1, a2, a3;
        codes_to_half<E5M2>(x[i], a0, a2);
        codes_to_half<E5M2>(y[i], a1, a3);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
          mma_f16((i & 1) ? odd[nt] : s[nt], a0, a1, a2, a3, qf[nt][v * 4 + i][0], qf[nt][v * 4 + i][1]);
      }
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int k = 0; k < 4; ++k) s[nt][k] += odd[nt][k];
  }

  // Softmax weights of the tile from its raw scores: B fragments of P (and of its remainder).
  __device__ __forceinline__ void weights(const Tile& t, float (&s)[NT][4], uint32_t (&p)[NT][2], uint32_t (&rest)[NT][2],
                                          bool edge, int lane) {
    const float tk = pow2i((int8_t)(t.exps & 0xff)), ev = (float)(int8_t)((t.exps >> 8) & 0xff);
    const float iv = pow2i(-(int8_t)((t.exps >> 8) & 0xff));
    const int g = lane >> 2;
    bool over = false;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const float fk[2] = {f[nt][0] * tk, f[nt][1] * tk};
#pragma unroll
      for (int k = 0; k < 4; ++k) s[nt][k] = fmaf(s[nt][k], fk[k & 1], ev);
      if (edge) {
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (t.tok + g + (k >> 1) * 8 >= lim[nt][k & 1]) s[nt][k] = -INFINITY;
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) over |= s[nt][k] > m[nt][k & 1] + 8.f;
    }
    if (__any_sync(0xffffffffu, over)) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          float x = fmaxf(s[nt][k], s[nt][k + 2]);
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
          x = fmaxf(x, m[nt][k]);
          const float down = exp2_fast(m[nt][k] - x);
          m[nt][k] = x;
          l[nt][k] *= down;
#pragma unroll
          for (int i = 0; i < kOT; ++i) {
            o[nt][i][k] *= down;
            o[nt][i][k + 2] *= down;
          }
        }
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        s[nt][k] = exp2_fast(s[nt][k] - m[nt][k & 1]);
        l[nt][k & 1] = fmaf(s[nt][k], iv, l[nt][k & 1]);
      }
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const uint32_t w = pack_half2(s[nt][2 * k], s[nt][2 * k + 1]);
        p[nt][k] = transpose8x8(w);
        if constexpr (kTwoTerms) {
          const float2 y = __half22float2(*reinterpret_cast<const __half2*>(&w));
          rest[nt][k] = transpose8x8(pack_half2(s[nt][2 * k] - y.x, s[nt][2 * k + 1] - y.y));
        }
      }
    }
  }

  // O^T += V^T P^T of the tile in vr; vr is free afterwards.
  __device__ __forceinline__ void product(const Tile& t, const uint32_t (&p)[NT][2], const uint32_t (&rest)[NT][2],
                                          bool edge, int lane) {
    if (edge) not_finite(t, lane);
#pragma unroll
    for (int i = 0; i < kVWords; ++i) {
      const uint32_t w[4] = {vr[0][i], vr[1][i], vr[2][i], vr[3][i]};
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        v_product(o[nt][2 * i], o[nt][2 * i + 1], w, p[nt][0], p[nt][1]);
        if constexpr (kTwoTerms) v_product(o[nt][2 * i], o[nt][2 * i + 1], w, rest[nt][0], rest[nt][1]);
      }
    }
  }

  // A tile that some of the rows see only in part: a NaN (or infinite) code of a token must reach the rows
  // that see it and no other, but 0 * NaN is NaN.  Such codes are counted per row in a product of
  // their own (1 for each, times 1 for each row that sees the token), turn the row's sums to NaN
  // and are cleared.
  __device__ __forceinline__ void not_finite(const Tile& t, int lane) {
    bool any = false;
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int i = 0; i < kVWords; ++i) any |= nonfinite_bytes<E5M2>(vr[r][i]) != 0u;
    if (!__any_sync(0xffffffffu, any)) return;
    const int g = lane >> 2;
    constexpr uint32_t kOnes = E5M2 ? 0x3c3c3c3cu : 0x38383838u;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      uint32_t sees[2];
#pragma unroll
      for (int k = 0; k < 2; ++k)
        sees[k] = transpose8x8(pack_half2(t.tok + g + 8 * k < lim[nt][0] ? 1.f : 0.f, t.tok + g + 8 * k < lim[nt][1] ? 1.f : 0.f));
#pragma unroll
      for (int i = 0; i < kVWords; ++i) {
        float n0[4] = {}, n1[4] = {};
        uint32_t w[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) w[r] = nonfinite_bytes<E5M2>(vr[r][i]) & kOnes;
        v_product(n0, n1, w, sees[0], sees[1]);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          if (n0[k] != 0.f) o[nt][2 * i][k] = NAN;
          if (n1[k] != 0.f) o[nt][2 * i + 1][k] = NAN;
        }
      }
    }
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int i = 0; i < kVWords; ++i) vr[r][i] &= ~nonfinite_bytes<E5M2>(vr[r][i]);
  }

  // This warp's share (every kKaWarps-th) of tiles [first, last) of (b, h).
  __device__ __forceinline__ void stream(const Kv8AttnDev& a, int b, int h, int len, int first, int last, int warp, int lane) {
    const int seen_by_all = len - a.q_len + 1;    // tokens below: every row sees them
    const int mine = first + warp;
    if (mine >= last) return;
    const int n = (last - mine + kKaWarps - 1) / kKaWarps;
    // lane j describes this warp's tile 32*k + j; the next 32 are looked up halfway through
    Tile now{-1, 0, 0}, next{-1, 0, 0};
    if (lane < n) now = find(a, b, h, len, mine + lane * kKaWarps);
    Tile t = pick(now, 0);
    load_k(a, t, h, len, lane);
    load_v(a, t, h, len, lane);
    for (int i = 0; i < n; ++i) {
      if ((i & 31) == 16) {
        const int at = (i & ~31) + 32 + lane;
        next.page = -1;
        if (at < n) next = find(a, b, h, len, mine + at * kKaWarps);
      }
      const int exps_of = now.exps;
      if ((i & 31) == 31) now = next;
      Tile ahead = pick(now, (i + 1) & 31);
      if (i + 1 >= n) ahead.page = -1;
      const bool edge = t.tok + 16 > seen_by_all;
      float s[NT][4];
      uint32_t p[NT][2], rest[NT][2];
      if (t.page >= 0) scores(s);
      load_k(a, ahead, h, len, lane);
      if (t.page >= 0) {
        t.exps = __shfl_sync(0xffffffffu, exps_of, i & 31);
        weights(t, s, p, rest, edge, lane);
        product(t, p, rest, edge, lane);
      }
      load_v(a, ahead, h, len, lane);
      t = ahead;
    }
  }

  // Merges the warps and writes the segment's rows: to `out`, or (slot >= 0) to the workspace.
  __device__ __forceinline__ void finish(const Kv8AttnDev& a, Smem& sm, int b, int h, int rt, int slot, int warp, int lane) {
    const int g = lane >> 2, c = lane & 3;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        float x = l[nt][k];
        x += __shfl_xor_sync(0xffffffffu, x, 4);
        x += __shfl_xor_sync(0xffffffffu, x, 8);
        x += __shfl_xor_sync(0xffffffffu, x, 16);
        if (g == 0) {
          sm.m[warp][nt * 8 + 2 * c + k] = m[nt][k];
          sm.l[warp][nt * 8 + 2 * c + k] = x;
        }
      }
    __syncthreads();
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int r = nt * 8 + 2 * c + k;
        float top = sm.m[0][r];
#pragma unroll
        for (int w = 1; w < kKaWarps; ++w) top = fmaxf(top, sm.m[w][r]);
        const float down = exp2_fast(m[nt][k] - top);
        // the lane's dims: 128u + (D/8 of them from g on) -- word i of a V row, byte by byte
        constexpr int kPer = D < 128 ? kVWords : 4;
#pragma unroll
        for (int i = 0; i < kVWords; ++i) {
          const int d = (i / kPer) * 128 + g * kPer * 4 + (i % kPer) * 4;
          *reinterpret_cast<float4*>(&sm.o[warp][r][d]) =
              make_float4(o[nt][2 * i][k] * down, o[nt][2 * i][k + 2] * down, o[nt][2 * i + 1][k] * down, o[nt][2 * i + 1][k + 2] * down);
        }
      }
    __syncthreads();
    for (int i = threadIdx.x; i < kRows * D / 4; i += kKaThreads) {
      const int r = i / (D / 4), d = (i % (D / 4)) * 4;
      float top = sm.m[0][r], sum = 0.f;
#pragma unroll
      for (int w = 1; w < kKaWarps; ++w) top = fmaxf(top, sm.m[w][r]);
      float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < kKaWarps; ++w) {
        const float4 y = *reinterpret_cast<const float4*>(&sm.o[w][r][d]);
        x.x += y.x; x.y += y.y; x.z += y.z; x.w += y.w;
        sum += sm.l[w][r] * exp2_fast(sm.m[w][r] - top);
      }
      if (slot >= 0) {
        *reinterpret_cast<float4*>(a.part_o + ((int64_t)slot * kRows + r) * D + d) = x;
        if (d == 0) *reinterpret_cast<float2*>(a.part_ml + ((int64_t)slot * kRows + r) * 2) = make_float2(top, sum);
      } else if (rt * kRows + r < a.rows) {
        write_out(a, b, h, rt * kRows + r, d, x, sum);
      }
    }
    __syncthreads();                              // the next segment reuses the buffers
  }

  // out[row][d .. d+3] = x / sum, 0 for a row that saw nothing.
  static __device__ __forceinline__ void write_out(const Kv8AttnDev& a, int b, int h, int r, int d, float4 x, float sum) {
    const int pos = r / a.group, head = h * a.group + r % a.group;
    char* dst = a.out + (int64_t)b * a.o_sb + (int64_t)head * a.o_sh + (int64_t)pos * a.o_sq + d * 2;
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    const float y[4] = {x.x * inv, x.y * inv, x.z * inv, x.w * inv};
    uint16_t u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) u[i] = BF16 ? __bfloat16_as_ushort(__float2bfloat16_rn(y[i])) : __half_as_ushort(__float2half_rn(y[i]));
    if (((uintptr_t)dst & 7) == 0) {
      *reinterpret_cast<uint2*>(dst) = make_uint2(u[0] | ((uint32_t)u[1] << 16), u[2] | ((uint32_t)u[3] << 16));
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) reinterpret_cast<uint16_t*>(dst)[i] = u[i];
    }
  }
};

// The line of tiles (below 2^31) in parts of nearly equal length: the first `longer` parts have size + 1
// tiles, the others size; every part has a tile, and kKaWarps of them while there are that many.
struct Line {
  uint32_t parts, size, longer;
  uint32_t unit, before;           // the unit ((b) or, with lists, (b, h)) that holds this CTA's first tile, and the tiles before it

  __device__ __forceinline__ uint32_t begin(uint32_t c) const { return c * size + min(c, longer); }
  __device__ __forceinline__ uint32_t part_of(uint32_t x) const {
    const uint32_t edge = longer * (size + 1);
    return x < edge ? x / (size + 1) : longer + (x - edge) / size;
  }
};

__device__ __forceinline__ Line line_start(const Kv8AttnDev& a, uint32_t* scratch) {
  // A unit's tiles are those of its segments: all heads and row tiles of b, or all row tiles of (b, h).
  const int units = a.blocks ? a.pg.batch * a.pg.heads : a.pg.batch;
  const uint32_t per = a.blocks ? a.row_tiles : a.row_tiles * a.pg.heads;
  const int each = (units + kKaThreads - 1) / kKaThreads;
  const int u0 = min((int)threadIdx.x * each, units), u1 = min(u0 + each, units);
  uint32_t sum = 0;
  for (int u = u0; u < u1; ++u)
    sum += per * (a.blocks ? kv8_tiles(a, u / a.pg.heads, u % a.pg.heads) : kv8_tiles(a, u, 0));
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint32_t upto = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t x = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += x;
  }
  if (lane == 31) scratch[warp] = upto;
  __syncthreads();
  uint32_t total = 0, base = 0;
#pragma unroll
  for (int w = 0; w < kKaWarps; ++w) {
    if (w < warp) base += scratch[w];
    total += scratch[w];
  }
  Line line{};
  line.parts = min(gridDim.x, (total + kKaWarps - 1) / kKaWarps);
  if (line.parts == 0) return line;
  line.size = total / line.parts;
  line.longer = total - line.size * line.parts;
  const uint32_t begin = line.begin(blockIdx.x);
  uint32_t before = base + upto - sum;
  if (begin >= before && begin - before < sum) {
    for (int u = u0; u < u1; ++u) {
      const uint32_t n = per * (a.blocks ? kv8_tiles(a, u / a.pg.heads, u % a.pg.heads) : kv8_tiles(a, u, 0));
      if (begin - before < n) {
        scratch[kKaWarps] = u;
        scratch[kKaWarps + 1] = before;
        break;
      }
      before += n;
    }
  }
  __syncthreads();
  line.unit = scratch[kKaWarps];
  line.before = scratch[kKaWarps + 1];
  return line;
}

template <int D, int NT, bool E5M2, bool BF16>
__global__ void __launch_bounds__(kKaThreads, D <= 128 && NT == 1 ? 2 : 1) kv8_attn_kernel(const Kv8AttnDev a) {
  using K = Kv8Attn<D, NT, E5M2, BF16>;
  extern __shared__ __align__(16) char smem_raw[];
  typename K::Smem& sm = *reinterpret_cast<typename K::Smem*>(smem_raw);
  __shared__ uint32_t s_line[kKaWarps + 2];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  K k;
  if (a.whole) {
    const int rt = blockIdx.x % a.row_tiles, bh = blockIdx.x / a.row_tiles;
    const int b = bh / a.pg.heads, h = bh % a.pg.heads;
    const int len = kv8_len(a, b);
    k.load_q(a, b, h, rt, len, lane);
    k.stream(a, b, h, len, 0, kv8_tiles(a, b, h), warp, lane);
    k.finish(a, sm, b, h, rt, -1, warp, lane);
    return;
  }
  const Line line = line_start(a, s_line);
  if (blockIdx.x < line.parts) {
    const uint32_t begin = line.begin(blockIdx.x), end = line.begin(blockIdx.x + 1);
    // segment of `begin`
    int b, h, rt;
    uint32_t n = a.blocks ? kv8_tiles(a, line.unit / a.pg.heads, line.unit % a.pg.heads) : kv8_tiles(a, line.unit, 0);
    const uint32_t seg = (begin - line.before) / n;
    uint32_t start = line.before + seg * n;           // the segment's first tile on the line
    rt = (int)(seg % a.row_tiles);
    if (a.blocks) {
      b = line.unit / a.pg.heads;
      h = line.unit % a.pg.heads;
    } else {
      b = line.unit;
      h = (int)(seg / a.row_tiles);
    }
    uint32_t at = begin;
    for (;;) {
      const uint32_t first = at - start, last = min(n, end - start);
      const bool cut = first > 0 || last < n;
      const int len = kv8_len(a, b);
      k.load_q(a, b, h, rt, len, lane);
      k.stream(a, b, h, len, first, last, warp, lane);
      k.finish(a, sm, b, h, rt, cut ? 2 * (int)blockIdx.x + (at == begin ? 0 : 1) : -1, warp, lane);
      if (first == 0 && threadIdx.x == 0)
        a.info[((int64_t)b * a.pg.heads + h) * a.row_tiles + rt] =
            make_int4((int)blockIdx.x, (int)line.part_of(start + n - 1), at == begin ? 0 : 1, 0);
      at = start + last;
      if (at >= end) break;
      start += n;
      if (++rt == a.row_tiles) {                      // the next segment that has tiles
        rt = 0;
        do {
          if (++h == a.pg.heads) {
            h = 0;
            ++b;
          }
          n = kv8_tiles(a, b, h);
        } while (n == 0);
      }
    }
  }
  allow_dependents();
}

// Rows of segments that CTA borders cut, and of segments without tiles.  One CTA per (segment, row):
// its warps take the parts in turn, each lane D/32 dims.
constexpr int kKmWarps = 4;

template <int D, int NT, bool BF16>
__global__ void __launch_bounds__(kKmWarps * 32) kv8_merge_kernel(const Kv8AttnDev a) {
  constexpr int kRows = NT * 8;
  __shared__ float s_m[kKmWarps], s_l[kKmWarps];
  __shared__ __align__(16) float s_o[kKmWarps][D];
  const int seg = blockIdx.x / kRows, r = blockIdx.x % kRows;
  const int rt = seg % a.row_tiles, bh = seg / a.row_tiles;
  const int b = bh / a.pg.heads, h = bh % a.pg.heads;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (rt * kRows + r >= a.rows) return;
  const bool empty = kv8_tiles(a, b, h) == 0;
  wait_for_previous_grid();
  float top = kNoMax, sum = 0.f;
  float x[D / 32];
#pragma unroll
  for (int i = 0; i < D / 32; ++i) x[i] = 0.f;
  if (!empty) {
    const int4 info = a.info[seg];
    if (info.x == info.y) return;                     // written by its CTA
    for (int c = info.x + warp; c <= info.y; c += kKmWarps) {
      const int64_t row = (int64_t)(2 * c + (c == info.x ? info.z : 0)) * kRows + r;
      const float2 ml = *reinterpret_cast<const float2*>(a.part_ml + row * 2);
      const float m = fmaxf(top, ml.x);
      const float was = exp2_fast(top - m), is = exp2_fast(ml.x - m);
      sum = sum * was + ml.y * is;
#pragma unroll
      for (int i = 0; i < D / 32; ++i) x[i] = x[i] * was + a.part_o[row * D + lane + 32 * i] * is;
      top = m;
    }
  }
  if (lane == 0) {
    s_m[warp] = top;
    s_l[warp] = sum;
  }
#pragma unroll
  for (int i = 0; i < D / 32; ++i) s_o[warp][lane + 32 * i] = x[i];
  __syncthreads();
  if (threadIdx.x < D / 4) {
    const int d = threadIdx.x * 4;
    top = kNoMax;
#pragma unroll
    for (int w = 0; w < kKmWarps; ++w) top = fmaxf(top, s_m[w]);
    sum = 0.f;
    float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kKmWarps; ++w) {
      const float is = exp2_fast(s_m[w] - top);
      const float4 z = *reinterpret_cast<const float4*>(&s_o[w][d]);
      y.x += z.x * is; y.y += z.y * is; y.z += z.z * is; y.w += z.w * is;
      sum += s_l[w] * is;
    }
    Kv8Attn<D, NT, false, BF16>::write_out(a, b, h, rt * kRows + r, d, y, sum);
  }
}

// ---- host --------------------------------------------------------------------------------------
struct Kv8Plan {
  int nt, row_tiles, whole;
  int64_t segments, ctas;          // ctas: of the first kernel
  uint64_t info_bytes, ml_bytes, o_bytes;
};

static Kv8Plan make_plan(const mskv_kv8_attn_desc& d) {
  Kv8Plan p{};
  const int rows = d.q_heads / d.pages.kv_heads * d.q_len;
  p.nt = rows <= 8 || d.pages.head_dim == 256 ? 1 : 2;   // 256 dims: two column tiles do not fit the registers
  p.row_tiles = (rows + p.nt * 8 - 1) / (p.nt * 8);
  p.segments = (int64_t)d.pages.batch * d.pages.kv_heads * p.row_tiles;
  const int64_t most = d.blocks ? (int64_t)d.num_blocks * (d.pages.page_size / 16) : ((int64_t)d.max_tokens + 15) / 16;
  p.whole = most <= 16;
  if (p.whole) {
    p.ctas = p.segments;
    return p;
  }
  const int per_sm = d.pages.head_dim <= 128 && p.nt == 1 ? 2 : 1;
  p.ctas = std::min<int64_t>((int64_t)num_sms() * per_sm, (p.segments * most + kKaWarps - 1) / kKaWarps);
  const uint64_t slots = 2 * (uint64_t)p.ctas * p.nt * 8;
  p.info_bytes = ((uint64_t)p.segments * sizeof(int4) + 255) / 256 * 256;
  p.ml_bytes = (slots * 2 * sizeof(float) + 255) / 256 * 256;
  p.o_bytes = slots * d.pages.head_dim * sizeof(float);
  return p;
}

template <int D, int NT, bool E5M2, bool BF16>
static int launch_attn(const Kv8AttnDev& a, const Kv8Plan& p, cudaStream_t st) {
  constexpr int smem = (int)sizeof(typename Kv8Attn<D, NT, E5M2, BF16>::Smem);
  const auto kernel = kv8_attn_kernel<D, NT, E5M2, BF16>;
  if (const int rc = ensure_smem_limit(reinterpret_cast<const void*>(kernel), smem, "mskv_kv8_attention")) return rc;
  kernel<<<(unsigned)p.ctas, kKaThreads, smem, st>>>(a);
  if (const int rc = after_launch("mskv_kv8_attention")) return rc;
  if (p.whole) return MSKV_OK;
  const cudaError_t e = launch_dependent(kv8_merge_kernel<D, NT, BF16>, dim3((unsigned)(p.segments * NT * 8)),
                                         dim3(kKmWarps * 32), 0, st, a);
  if (e != cudaSuccess) return cuda_status(e, "mskv_kv8_attention merge launch");
  return after_launch("mskv_kv8_attention merge");
}

template <int D, int NT>
static int attn_types(const Kv8AttnDev& a, const Kv8Plan& p, bool e5m2, bool bf16, cudaStream_t st) {
  if (e5m2) return bf16 ? launch_attn<D, NT, true, true>(a, p, st) : launch_attn<D, NT, true, false>(a, p, st);
  return bf16 ? launch_attn<D, NT, false, true>(a, p, st) : launch_attn<D, NT, false, false>(a, p, st);
}

template <int D>
static int attn_rows(const Kv8AttnDev& a, const Kv8Plan& p, bool e5m2, bool bf16, cudaStream_t st) {
  if constexpr (D == 256) return attn_types<D, 1>(a, p, e5m2, bf16, st);
  else return p.nt == 1 ? attn_types<D, 1>(a, p, e5m2, bf16, st) : attn_types<D, 2>(a, p, e5m2, bf16, st);
}

static int check_attn(const mskv_kv8_attn_desc* d) {
  const char* what = "mskv_kv8_attention";
  if (!d) return fail(MSKV_ERR_ARG, "%s: NULL descriptor", what);
  if (const int rc = check_kv8(d->pages, what)) return rc;
  if (d->dtype != MSKV_DT_BF16 && d->dtype != MSKV_DT_F16) return fail(MSKV_ERR_DTYPE, "%s: q and out must be bf16 or f16", what);
  if (d->q_heads <= 0 || d->q_heads % d->pages.kv_heads)
    return fail(MSKV_ERR_ARG, "%s: q_heads must be a multiple of kv_heads", what);
  if (d->q_len <= 0 || d->q_len > MSKV_KV8_MAX_QLEN)
    return fail(MSKV_ERR_RANGE, "%s: q_len must lie in [1, %d]", what, MSKV_KV8_MAX_QLEN);
  if (d->max_tokens < 0 || (int64_t)d->max_tokens > (int64_t)d->pages.max_pages * d->pages.page_size)
    return fail(MSKV_ERR_ARG, "%s: max_tokens must lie in [0, max_pages*page_size]", what);
  if (d->max_tokens > INT_MAX - 64) return fail(MSKV_ERR_RANGE, "%s: max_tokens too large", what);
  if (d->blocks && (d->num_blocks < 0 || d->num_blocks > (1 << 24)))
    return fail(MSKV_ERR_RANGE, "%s: num_blocks must lie in [0, 2^24]", what);
  const int64_t row_tiles = ((int64_t)d->q_heads / d->pages.kv_heads * d->q_len + 7) / 8;
  if (row_tiles * d->pages.batch * d->pages.kv_heads > INT_MAX / 16)
    return fail(MSKV_ERR_RANGE, "%s: too many query rows for one call", what);
  const int64_t most = d->blocks ? (int64_t)d->num_blocks * (d->pages.page_size / 16) : ((int64_t)d->max_tokens + 15) / 16;
  if (row_tiles * d->pages.batch * d->pages.kv_heads * most > INT_MAX / 2)
    return fail(MSKV_ERR_RANGE, "%s: too many tokens for one call", what);
  if (!(fabsf(d->scale) <= 3e38f)) return fail(MSKV_ERR_ARG, "%s: scale must be finite", what);
  return MSKV_OK;
}

}  // namespace mskv

using namespace mskv;

extern "C" uint64_t mskv_kv8_attention_workspace_bytes(const mskv_kv8_attn_desc* d) {
  if (check_attn(d)) return 0;
  const Kv8Plan p = make_plan(*d);
  return p.info_bytes + p.ml_bytes + p.o_bytes;
}

extern "C" int mskv_kv8_attention(const mskv_kv8_attn_desc* d, void* stream) {
  if (const int rc = check_attn(d)) return rc;
  if (!d->q || !d->out || !d->lens) return fail(MSKV_ERR_ARG, "mskv_kv8_attention: NULL q, out or lens");
  const uintptr_t q_bits = (uintptr_t)d->q | (uintptr_t)d->q_stride_b | (uintptr_t)d->q_stride_h | (uintptr_t)d->q_stride_q;
  const uintptr_t o_bits = (uintptr_t)d->out | (uintptr_t)d->out_stride_b | (uintptr_t)d->out_stride_h | (uintptr_t)d->out_stride_q;
  if ((q_bits | o_bits) & 1) return fail(MSKV_ERR_ARG, "mskv_kv8_attention: q and out must be aligned to their elements");
  const Kv8Plan p = make_plan(*d);
  const uint64_t need = p.info_bytes + p.ml_bytes + p.o_bytes;
  if (need && (!d->workspace || d->workspace_bytes < need || ((uintptr_t)d->workspace & 15)))
    return fail(MSKV_ERR_ARG, "mskv_kv8_attention: needs %llu bytes of 16-byte aligned workspace", (unsigned long long)need);
  Kv8AttnDev a{};
  a.pg = to_dev(d->pages);
  a.q = static_cast<const char*>(d->q);
  a.q_sb = d->q_stride_b; a.q_sh = d->q_stride_h; a.q_sq = d->q_stride_q;
  a.out = static_cast<char*>(d->out);
  a.o_sb = d->out_stride_b; a.o_sh = d->out_stride_h; a.o_sq = d->out_stride_q;
  a.lens = d->lens;
  a.blocks = d->blocks;
  a.blk_sb = d->blk_stride_b; a.blk_sh = d->blk_stride_h;
  a.counts = d->counts;
  char* ws = static_cast<char*>(d->workspace);
  a.info = reinterpret_cast<int4*>(ws);
  a.part_ml = reinterpret_cast<float*>(ws + p.info_bytes);
  a.part_o = reinterpret_cast<float*>(ws + p.info_bytes + p.ml_bytes);
  a.status = d->status;
  a.scale_log2 = d->scale * 1.44269504088896340736f;
  a.group = d->q_heads / d->pages.kv_heads;
  a.q_len = d->q_len;
  a.rows = a.group * a.q_len;
  a.row_tiles = p.row_tiles;
  a.segments = (int32_t)p.segments;
  a.max_tokens = d->max_tokens;
  a.width = d->num_blocks;
  a.whole = p.whole;
  a.vec_q = (q_bits & 15) == 0;
  a.pow2_page = (a.pg.page_size & (a.pg.page_size - 1)) == 0;
  const bool e5m2 = d->pages.dtype == MSKV_DT_FP8_E5M2, bf16 = d->dtype == MSKV_DT_BF16;
  const cudaStream_t st = as_stream(stream);
  switch (d->pages.head_dim) {
    case 64: return attn_rows<64>(a, p, e5m2, bf16, st);
    case 128: return attn_rows<128>(a, p, e5m2, bf16, st);
    default: return attn_rows<256>(a, p, e5m2, bf16, st);
  }
}
