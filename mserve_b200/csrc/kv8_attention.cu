// Attention over the 8-bit paged cache, whole or over listed pages (mskv_kv8_attention).
//
//   s[r,t] = scale * q[r] . k8[t] * 2^eK(page of t),   o[r] = sum_t softmax(s[r])_t v8[t] * 2^eV(page of t)
//
// for the R = (q_heads/kv_heads) * q_len query rows of a KV head, from one pass over its codes.
//
// Mathematics.  Work unit: a tile of 16 tokens, which lies in one page, so both scales are one
// number.  With base-2 logarithms and t' = s * log2(e) + eV, the second product's weights
// P = 2^(t' - m) carry V's scale (m: running reference of t' over the tiles), the codes v8 enter it
// unscaled, and the softmax denominator is sum P * 2^-eV in fp32.  Exponents within [-60, 60] keep
// its term of the largest s above 2^-121 and so in fp32's normal range.  m moves only when a t'
// exceeds it by more than 15 (then P <= 2^15 until the next move): most tiles need one vote
// instead of a maximum over the warp.
// q is scaled per row to a largest magnitude in [1, 2) and enters as fp16 (a bf16 or fp16 value
// keeps all its bits down to 2^-14 of the row's largest; below, it is off by at most 2^-25 of that).
// K and V codes are exact in fp16.  P is rounded to fp16 (relative 2^-11); for fp16 outputs
// its remainder enters as a second fp16 term, as one term alone would be as far off as the output's
// own rounding.  For bf16 outputs, whose rounding is eight times as coarse, one term adds 0.5% to the error
// against 64 bits (1.681e-3 of the 2-norm against 1.673e-3, 8 x 16384 tokens; up to 9% of the values round
// to another bf16), and the second would cost 4% (16 x 32768 tokens 173 us -> 180) to 11% (two column tiles, 36.7 -> 40.6).
// All sums are fp32.  m starts 7 below the largest t' and so uses fp16's range above 1: the steps of 2^-24 at its lower
// end put a weight off by at most 2^-32 of the largest P of its warp, relative to P by more than the roundings above only
// where P is below 2^-21 of that -- a score 15 lower, or a page whose V exponent is 21 below another's (one
// outlier of V raises its page's).  From 2^-32 on a weight counts in the denominator only.
//
// Bound by the codes' bytes (2D a token and KV head).  mma.sync m16n8k16 with the tokens on M:
// S^T = K Q^T, O^T = V^T P^T, so the 8 columns hold the query rows (16 rows: two column tiles, and
// the codes converted once for both).
// A warp owns a tile and a ring of tiles in flight: one lane starts a TMA box of 16 rows of K and one of V,
// completing on the stage's mbarrier, three to six tiles ahead; nothing in the loop waits for another warp.
// The contraction's order is free, so the 16 contiguous codes that a lane reads of a K row are four
// k-steps', and those of four V rows are eight row tiles' (byte permutations pair the tokens); TMA's
// swizzle keeps these 16-byte reads free of bank conflicts.
// A tcgen05 MMA would need 64 or 128 rows of f16 operands staged in shared memory after a conversion there;
// the legacy pipe is a fifth busy at the memory's speed.
//
// Split: a segment is a (sequence, KV head, row tile).  Where the segments fill the GPU evenly, or are short, a
// thread-block cluster (of one CTA, where they are many) takes each and merges through distributed shared memory.
// Otherwise all tiles of all segments form one line, cut into parts for the CTAs however ragged the lengths are (a scan over the
// lengths in every CTA); a segment of several parts goes through the workspace and a second kernel.
//
// Measured (device time, three sets of inputs in turn): 40/8 heads, 128 dims, 16 sequences of 32768 tokens
// (1.07 GB) 173 us = 0.95 of the copy rate in a burst, 189 = 0.87 in calls that go on for tenths of a second, at the power
// limit's clocks; 16/4 heads of 256 dims, the same bytes 172 us, 64/8 heads of 64 dims, half of them, 114 us = 0.72; 28/4
// heads, 8 of 16384 (134 MB) 28.3 us = 0.73, of which 3 us pass before the first codes are there and 2 after the
// last; 136 listed pages of each (18 MB) 8.8 us.
// Loads straight into registers instead of the ring (one tile ahead, as many as the registers hold): 181,
// 32.5 and 11.7 us, and 10% more than that at the clocks of a GPU at its power limit; the same chunks through
// cp.async into a ring: 257 us for the first.
#include <cooperative_groups.h>
#include <math.h>

#include <algorithm>
#include <atomic>

#include "kv8.cuh"
#include "ring.cuh"
#include "tensor_map.cuh"

namespace cg = cooperative_groups;

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
  int32_t group, q_len, rows, row_tiles, segments, max_tokens, width;
  int32_t cluster, cluster_log2;   // CTAs that share a segment (1, 2, 4, 8); 0: the line
  int32_t parts_log2;              // tiles of a page; -1 where they are no power of two
  int32_t vec_q, pow2_page, aligned;
  int32_t expire;                  // every first wait for codes counts as expired (mskv_kv8_expire_waits)
  Divisor by_heads;
};

// Warps of a CTA, its ring's stages and CTAs of an SM, by what the registers (64 dims: 80 a thread, 128 with a second
// column tile; 128 dims: 128, 168 with it; 256 dims: 255) and 227 KB of shared memory hold.
__host__ __device__ constexpr int ka_warps(int d, int nt) { return d == 128 && nt == 2 ? 12 : 8; }
__host__ __device__ constexpr int ka_stages(int d, int nt) { return d == 64 ? (nt == 1 ? 4 : 6) : d == 128 && nt == 2 ? 4 : 3; }
__host__ __device__ constexpr int ka_ctas(int d, int nt) { return d == 256 || (d == 128 && nt == 2) ? 1 : d == 64 && nt == 1 ? 3 : 2; }
constexpr int kKaMaxCluster = 8;
constexpr float kNoMax = -3e38f;   // below every finite score's exponent
constexpr float kBelow = 7.f, kAbove = 15.f;   // m is set 7 below the largest exponent, and again for one over 15 above m

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

// The line of tiles (below 2^31) of all segments, cut into parts, one for each CTA.
// With at most half as many segments as CTAs (a.aligned) parts do not cross segments.  A segment of n
// tiles has ceil(n / size) parts of nearly equal length; size = ceil(total / (CTAs - segments))
// makes them at most as many as the CTAs.  A CTA that goes on to a second segment starts its pipeline and
// merges again, about 4 us.
// Otherwise all parts are of nearly equal length, the first `longer` of size + 1 tiles, the others of size.
// Every part has a tile.
struct Line {
  uint32_t size, longer;

  __device__ __forceinline__ uint32_t even_begin(uint32_t c) const { return c * size + min(c, longer); }
  // Last part of the segment of tiles [start, start + n) whose first part is c.
  __device__ __forceinline__ uint32_t last_part(bool aligned, uint32_t c, uint32_t start, uint32_t n) const {
    if (aligned) return c + (n + size - 1) / size - 1;
    const uint32_t x = start + n - 1, edge = longer * (size + 1);
    return x < edge ? x / (size + 1) : longer + (x - edge) / size;
  }
};

// A CTA's place: the segment, its tiles and its first one's place on the line, the CTA's tiles [at, end)
// from this segment on, its first of all.
struct Place {
  int b, h, rt, len;
  uint32_t n, start, at, end, begin;
  Line line;
};

template <int D, int NT, bool E5M2, bool BF16>
struct Kv8Attn {
  static constexpr int kWarps = ka_warps(D, NT), kThreads = kWarps * 32;
  static constexpr int kRows = NT * 8;
  static constexpr int kKVec = D / 64;            // 16-byte loads of a lane per K row
  static constexpr int kVWords = D / 32;          // words of a lane per V row
  static constexpr int kOT = D / 16;              // row tiles of O^T
  static constexpr int kOStride = D + 4;          // floats between rows of the merge buffer
  static constexpr bool kTwoTerms = !BF16;        // P as two fp16 terms

  static constexpr int kBox = 16 * (D < 128 ? D : 128);    // bytes of a box: 16 rows, at most 128 dims
  static constexpr int kTileBytes = 2 * 16 * D;            // K boxes, then V boxes
  static constexpr int kStages = ka_stages(D, NT);         // tiles of a warp in flight

  struct Smem {
    union {
      uint8_t ring[kWarps][kStages][kTileBytes];  // 1024-byte aligned stages (the swizzle's period)
      float o[kWarps][kRows][kOStride];           // the warps' sums, when the ring is empty
    };
    float sent[kRows][D];                         // of the cluster's CTAs: [CTA][rows of this one]
    float2 sent_ml[kRows];
    uint64_t arrived[kWarps][kStages];            // mbarriers
    float m[kWarps][kRows], l[kWarps][kRows];
    __half q[kRows][D + 8];
    float f[kRows];
    int lim[kRows];                               // tokens that a row sees
    uint32_t expired;                             // a wait of one of the warps ran out
  };

  // With two column tiles the query's fragments stay in shared memory (the registers hold O and the codes).
  static constexpr bool kKeepQ = NT == 1;
  uint32_t qf[kKeepQ ? kKVec * 4 : 1][2];
  float f[NT][2];                                 // scale * log2(e) * 2^(row exponent) of the lane's two columns
  float m[NT][2], l[NT][2];
  float o[NT][kOT][4];

  // Query position of row r of a KV head.
  static __device__ __forceinline__ int position(const Kv8AttnDev& a, int r) { return a.q_len == 1 ? 0 : r / a.group; }

  // Query rows of the segment to shared memory, in two steps, so that the codes' first loads come between: a
  // warp takes rows warp and warp + kWarps (two column tiles), a lane D/32 neighbouring elements of each.
  // Row 8*(row tile*NT + nt) + n is position * group + head.
  static constexpr int kQEach = (kRows + kWarps - 1) / kWarps, kQPer = D / 32;
  struct QRows {
    uint32_t w[kQEach][kQPer / 2];
  };
  static __device__ __forceinline__ QRows load_q(const Kv8AttnDev& a, int b, int h, int rt, int warp, int lane) {
    QRows q;
#pragma unroll
    for (int k = 0; k < kQEach; ++k) {
      const int n = warp + k * kWarps, r = rt * kRows + n;
#pragma unroll
      for (int i = 0; i < kQPer / 2; ++i) q.w[k][i] = 0u;
      if (n < kRows && r < a.rows) {
        const int pos = position(a, r), head = h * a.group + r - pos * a.group;
        const char* src = a.q + (int64_t)b * a.q_sb + (int64_t)head * a.q_sh + (int64_t)pos * a.q_sq + lane * (kQPer * 2);
        if (!a.vec_q) {
          const uint16_t* u = reinterpret_cast<const uint16_t*>(src);
#pragma unroll
          for (int i = 0; i < kQPer / 2; ++i) q.w[k][i] = (uint32_t)u[2 * i] | ((uint32_t)u[2 * i + 1] << 16);
        } else if constexpr (kQPer == 2) {
          q.w[k][0] = *reinterpret_cast<const uint32_t*>(src);
        } else if constexpr (kQPer == 4) {
          const uint2 y = *reinterpret_cast<const uint2*>(src);
          q.w[k][0] = y.x; q.w[k][1] = y.y;
        } else {
          const uint4 y = *reinterpret_cast<const uint4*>(src);
          q.w[k][0] = y.x; q.w[k][1] = y.y; q.w[k][2] = y.z; q.w[k][3] = y.w;
        }
      }
    }
    return q;
  }

  // Scaled to a largest magnitude in [1, 2), as fp16.
  static __device__ __forceinline__ void stage_q(const Kv8AttnDev& a, Smem& sm, const QRows& q, int rt, int len, int warp, int lane) {
#pragma unroll
    for (int k = 0; k < kQEach; ++k) {
      const int n = warp + k * kWarps, r = rt * kRows + n;
      if (n >= kRows) break;
      float x[kQPer];
      uint32_t top = 0;
#pragma unroll
      for (int i = 0; i < kQPer; ++i) {
        const uint16_t u = (uint16_t)(i & 1 ? q.w[k][i / 2] >> 16 : q.w[k][i / 2]);
        x[i] = BF16 ? __uint_as_float((uint32_t)u << 16) : __half2float(__ushort_as_half(u));
        const uint32_t mag = __float_as_uint(x[i]) & 0x7fffffffu;
        top = max(top, mag < 0x7f800000u ? mag : 0u);
      }
      top = __reduce_max_sync(0xffffffffu, top);
      const int e = top ? min(max((int)(top >> 23) - 127, -120), 120) : 0;
      const float inv = pow2i(-e);
#pragma unroll
      for (int i = 0; i < kQPer; i += 2)
        *reinterpret_cast<uint32_t*>(&sm.q[n][lane * kQPer + i]) = pack_half2(x[i] * inv, x[i + 1] * inv);
      if (lane == 0) {
        sm.f[n] = a.scale_log2 * pow2i(e);
        sm.lim[n] = len - a.q_len + 1 + (r < a.rows ? position(a, r) : a.q_len - 1);
      }
    }
  }

  // The staged rows as B fragments: column n = lane/4 of column tile nt is row 8*nt + n, the lane's k-steps
  // of a 64-element stretch are its 16 contiguous elements.  Resets the running sums.
  static __device__ __forceinline__ void q_fragments(const Smem& sm, int nt, int v, int lane, uint32_t (&x)[4][2]) {
    const uint4* src = reinterpret_cast<const uint4*>(&sm.q[nt * 8 + (lane >> 2)][64 * v + 16 * (lane & 3)]);
    const uint4 lo = src[0], hi = src[1];
    x[0][0] = lo.x; x[0][1] = lo.y; x[1][0] = lo.z; x[1][1] = lo.w;
    x[2][0] = hi.x; x[2][1] = hi.y; x[3][0] = hi.z; x[3][1] = hi.w;
  }

  __device__ __forceinline__ void start(const Smem& sm, int lane) {
    const int c = lane & 3;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      if constexpr (kKeepQ) {
#pragma unroll
        for (int v = 0; v < kKVec; ++v) {
          uint32_t x[4][2];
          q_fragments(sm, 0, v, lane, x);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            qf[v * 4 + i][0] = x[i][0];
            qf[v * 4 + i][1] = x[i][1];
          }
        }
      }
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        f[nt][k] = sm.f[nt * 8 + 2 * c + k];
        m[nt][k] = kNoMax;
        l[nt][k] = 0.f;
      }
#pragma unroll
      for (int i = 0; i < kOT; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k) o[nt][i][k] = 0.f;
    }
  }

  struct Tile {                                   // one lane's lookup
    int page, tok, exps;                          // page < 0: nothing to read; exps: eK, eV, bit 16: there are tokens
  };

  // Tile `i` of (b, h) as one lane sees it.
  static __device__ __forceinline__ Tile find(const Kv8AttnDev& a, int b, int h, int len, int i) {
    const int parts = a.pg.page_size >> 4;
    int pi = a.parts_log2 >= 0 ? i >> a.parts_log2 : i / parts;
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
    t.exps = *reinterpret_cast<const uint16_t*>(a.pg.exps + ((int64_t)page * a.pg.heads + h) * 2) | 0x10000;
    return t;
  }

  // A tile's codes are 16-row boxes in shared memory, their 16-byte chunks permuted by the row (TMA's 128-byte
  // swizzle, 64-byte at 64 dims).  Fragment row g of K is row g ^ 4*(g & 1) of the tile, so that the eight lanes
  // of a phase of a 16-byte load read different banks; the tokens of V, the same contraction index, follow.
  static __device__ __forceinline__ int tile_row(int g) { return g ^ ((g & 1) << 2); }
  static __device__ __forceinline__ uint32_t chunk_at(int row, int chunk) {
    return D < 128 ? row * 64 + ((chunk ^ (row >> 1)) & 3) * 16 : row * 128 + (chunk ^ (row & 7)) * 16;
  }
  static __device__ __forceinline__ uint4 read16(uint32_t at) {
    uint4 x;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(x.x), "=r"(x.y), "=r"(x.z), "=r"(x.w) : "r"(at) : "memory");
    return x;
  }

  // 64 dims of K rows lane/4 and lane/4 + 8: four k-steps.
  static __device__ __forceinline__ void read_k(uint32_t tile, int v, int lane, uint4 (&x)[2]) {
    const int row = tile_row(lane >> 2), c = lane & 3;
    const uint32_t at = tile + (v >> 1) * kBox + chunk_at(row, c + 4 * (v & 1));
    x[0] = read16(at);
    x[1] = read16(at + 8 * (D < 128 ? 64 : 128));
  }

  // V rows of tokens 2c, 2c+1, 2c+8, 2c+9 (as fragment rows), the lane's dims.
  uint32_t vr[4][kVWords];
  __device__ __forceinline__ void read_v(uint32_t tile, int lane) {
    const int g = lane >> 2, c = lane & 3;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int row = tile_row(2 * c + (r & 1));
      const uint32_t at = tile + 16 * D + (r >> 1) * 8 * (D < 128 ? 64 : 128);
      if constexpr (D == 64) {
        asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];"
                     : "=r"(vr[r][0]), "=r"(vr[r][1]) : "r"(at + chunk_at(row, g >> 1) + (g & 1) * 8) : "memory");
      } else {
#pragma unroll
        for (int u = 0; u < D / 128; ++u) {
          const uint4 x = read16(at + u * kBox + chunk_at(row, g));
          vr[r][4 * u] = x.x; vr[r][4 * u + 1] = x.y; vr[r][4 * u + 2] = x.z; vr[r][4 * u + 3] = x.w;
        }
      }
    }
  }

  // Starts the loads of a tile into a stage (one lane); a tile without tokens completes at once.
  static __device__ __forceinline__ void fetch(const Kv8AttnDev& a, const CUtensorMap* k_map, const CUtensorMap* v_map, int page,
                                               int tok, int h, uint32_t stage, uint32_t bar) {
    if (page < 0) {
      asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
      return;
    }
    const int row = a.pow2_page ? tok & (a.pg.page_size - 1) : tok % a.pg.page_size;
    mbar_expect_tx(bar, kTileBytes);
#pragma unroll
    for (int u = 0; u < (D < 128 ? 1 : D / 128); ++u) {
      load_box(stage + u * kBox, k_map, 128 * u, row, h, page, bar);
      load_box(stage + 16 * D + u * kBox, v_map, 128 * u, row, h, page, bar);
    }
  }
  static __device__ __forceinline__ void load_box(uint32_t dst, const CUtensorMap* map, int d, int row, int h, int page,
                                                  uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
                 ::"r"(dst), "l"(map), "r"(d), "r"(row), "r"(h), "r"(page), "r"(bar) : "memory");
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

  // Raw scores of a tile.
  __device__ __forceinline__ void scores(const Smem& sm, uint32_t tile, float (&s)[NT][4], int lane) {
    float odd[NT][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int k = 0; k < 4; ++k) s[nt][k] = odd[nt][k] = 0.f;
#pragma unroll
    for (int v = 0; v < kKVec; ++v) {
      uint4 kr[2];
      read_k(tile, v, lane, kr);
      const uint32_t x[4] = {kr[0].x, kr[0].y, kr[0].z, kr[0].w};
      const uint32_t y[4] = {kr[1].x, kr[1].y, kr[1].z, kr[1].w};
      uint32_t q[NT][4][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        if constexpr (kKeepQ) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            q[nt][i][0] = qf[v * 4 + i][0];
            q[nt][i][1] = qf[v * 4 + i][1];
          }
        } else {
          q_fragments(sm, nt, v, lane, q[nt]);
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint32_t a0, a1, a2, a3;
        codes_to_half<E5M2>(x[i], a0, a2);
        codes_to_half<E5M2>(y[i], a1, a3);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) mma_f16((i & 1) ? odd[nt] : s[nt], a0, a1, a2, a3, q[nt][i][0], q[nt][i][1]);
      }
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int k = 0; k < 4; ++k) s[nt][k] += odd[nt][k];
  }

  // Softmax weights of the tile from its raw scores: B fragments of P (and of its remainder).
  __device__ __forceinline__ void weights(const Smem& sm, int tok, int exps, float (&s)[NT][4], uint32_t (&p)[NT][2], uint32_t (&rest)[NT][2],
                                          bool edge, int lane) {
    const float tk = pow2i((int8_t)(exps & 0xff)), ev = (float)(int8_t)((exps >> 8) & 0xff);
    const float iv = pow2i(-(int8_t)((exps >> 8) & 0xff));
    const int row = tile_row(lane >> 2);
    bool over = false;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const float fk[2] = {f[nt][0] * tk, f[nt][1] * tk};
#pragma unroll
      for (int k = 0; k < 4; ++k) s[nt][k] = fmaf(s[nt][k], fk[k & 1], ev);
      if (edge) {
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (tok + row + (k >> 1) * 8 >= sm.lim[nt * 8 + 2 * (lane & 3) + (k & 1)]) s[nt][k] = -INFINITY;
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) over |= s[nt][k] > m[nt][k & 1] + kAbove;
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
          x = fmaxf(x - kBelow, m[nt][k]);
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

  // O^T += V^T P^T of the tile in vr.
  __device__ __forceinline__ void product(const Smem& sm, int tok, int len, const uint32_t (&p)[NT][2],
                                          const uint32_t (&rest)[NT][2], bool edge, int lane) {
    if (edge) {
      // rows behind the sequence hold anything
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (tok + tile_row(2 * (lane & 3) + (r & 1)) + 8 * (r >> 1) >= len)
#pragma unroll
          for (int i = 0; i < kVWords; ++i) vr[r][i] = 0u;
      not_finite(sm, tok, lane);
    }
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
  __device__ __forceinline__ void not_finite(const Smem& sm, int tok, int lane) {
    bool any = false;
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int i = 0; i < kVWords; ++i) any |= nonfinite_bytes<E5M2>(vr[r][i]) != 0u;
    if (!__any_sync(0xffffffffu, any)) return;
    const int row = tile_row(lane >> 2);
    constexpr uint32_t kOnes = E5M2 ? 0x3c3c3c3cu : 0x38383838u;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      uint32_t sees[2];
#pragma unroll
      for (int k = 0; k < 2; ++k)
        sees[k] = transpose8x8(pack_half2(tok + row + 8 * k < sm.lim[nt * 8 + 2 * (lane & 3)] ? 1.f : 0.f,
                                          tok + row + 8 * k < sm.lim[nt * 8 + 2 * (lane & 3) + 1] ? 1.f : 0.f));
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

  // The bounded wait for the tile at `place` ran out, `left` before the warp's last: the rows are incomplete, so say so, wait
  // (again with a limit) for the copies still in flight and take no more tiles, of this segment or another: the
  // CTA contributes nothing from here on.  Kept out of the tile loop's code.
  static __device__ __noinline__ void give_up(uint32_t* status, Smem& sm, RingPlace<kStages> place, uint32_t bars, int left, int lane) {
    if (lane == 0) {
      if (status) atomicOr(status, MSKV_STATUS_TIMEOUT);
      sm.expired = 1;
    }
    place.drain(0, left, [&](int stage, uint32_t phase) { return bulk_wait(bars + 8 * stage, phase); });
  }

  // The CTA's tiles of the segment: the warp's share (every kWarps-th).  The first tile's codes are on their way
  // while the query is staged.
  __device__ __forceinline__ void piece(const Kv8AttnDev& a, const CUtensorMap* k_map, const CUtensorMap* v_map, Smem& sm, const Place& at,
                                        uint32_t& turn, int warp, int lane) {
    const int b = at.b, h = at.h, rt = at.rt;
    const int first = (int)(at.at - at.start), last = (int)min(at.n, at.end - at.start);
    const int len = at.len;
    const int seen_by_all = len - a.q_len + 1;    // tokens below: every row sees them
    const int mine = first + warp;
    int n = mine < last ? (last - mine + kWarps - 1) / kWarps : 0;
    // lane j describes this warp's tile 32*k + j; the next 32 are looked up halfway through
    Tile now{-1, 0, 0}, next{-1, 0, 0};
    if (lane < n) now = find(a, b, h, len, mine + lane * kWarps);
    const QRows q = load_q(a, b, h, rt, warp, lane);
    const uint32_t ring = smem_addr(&sm.ring[warp][0][0]), bars = smem_addr(&sm.arrived[warp][0]);
    RingPlace<kStages> place(turn);               // of tile i; tile number turn + i of the warp
#pragma unroll 1
    for (int i = 0; i < kStages; ++i) {
      const int page = __shfl_sync(0xffffffffu, now.page, i), tok = __shfl_sync(0xffffffffu, now.tok, i);
      const int to = place.stage_ahead(i);
      if (lane == 0 && i < n) fetch(a, k_map, v_map, page, tok, h, ring + to * kTileBytes, bars + 8 * to);
    }
    stage_q(a, sm, q, rt, len, warp, lane);
    __syncthreads();
    start(sm, lane);
    if (a.expire && n > 0) {
      give_up(a.status, sm, place, bars, n, lane);
      n = 0;
    }
#pragma unroll 1
    for (int i = 0; i < n; ++i) {
      if ((i & 31) == 16) {
        const int j = (i & ~31) + 32 + lane;
        next = Tile{-1, 0, 0};
        if (j < n) next = find(a, at.b, h, len, (int)(at.at - at.start) + warp + j * kWarps);
      }
      const int tok = __shfl_sync(0xffffffffu, now.tok, i & 31), exps = __shfl_sync(0xffffffffu, now.exps, i & 31);
      const uint32_t bar = bars + 8 * place.stage, tile = ring + place.stage * kTileBytes;
      if (!__all_sync(0xffffffffu, bulk_wait(bar, place.phase))) {
        give_up(a.status, sm, place, bars, n - i, lane);
        break;
      }
      if (exps & 0x10000) {
        const bool edge = tok + 16 > seen_by_all;
        float s[NT][4];
        uint32_t p[NT][2], rest[NT][2];
        scores(sm, tile, s, lane);
        read_v(tile, lane);
        weights(sm, tok, exps, s, p, rest, edge, lane);
        product(sm, tok, len, p, rest, edge, lane);
      }
      // the tile kStages further takes the stage
      const bool other = (i & 31) + kStages > 31;
      const int page_ahead = __shfl_sync(0xffffffffu, other ? next.page : now.page, (i + kStages) & 31);
      const int tok_ahead = __shfl_sync(0xffffffffu, other ? next.tok : now.tok, (i + kStages) & 31);
      if (lane == 0 && i + kStages < n) fetch(a, k_map, v_map, page_ahead, tok_ahead, h, tile, bar);
      place.advance();
      if ((i & 31) == 31) now = next;
    }
    turn += n;
    collect(sm, warp, lane);
  }

  // The warps' (m, l, O) to shared memory, O relative to the CTA's m.  O takes the ring's place, so not after an
  // expired wait, when a copy may still be under way to it.
  __device__ __forceinline__ void collect(Smem& sm, int warp, int lane) {
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
    if (sm.expired) return;                       // the whole CTA
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int r = nt * 8 + 2 * c + k;
        float top = sm.m[0][r];
#pragma unroll
        for (int w = 1; w < kWarps; ++w) top = fmaxf(top, sm.m[w][r]);
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
  }

  // Sums of the CTA for dims d .. d+3 of row r, after collect; nothing after an expired wait.
  struct Part {
    float4 x;
    float top, sum;
  };
  static __device__ __forceinline__ Part cta_part(const Smem& sm, bool expired, int r, int d) {
    if (expired) return {make_float4(0.f, 0.f, 0.f, 0.f), kNoMax, 0.f};
    Part y{make_float4(0.f, 0.f, 0.f, 0.f), sm.m[0][r], 0.f};
#pragma unroll
    for (int w = 1; w < kWarps; ++w) y.top = fmaxf(y.top, sm.m[w][r]);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float4 z = *reinterpret_cast<const float4*>(&sm.o[w][r][d]);
      y.x.x += z.x; y.x.y += z.y; y.x.z += z.z; y.x.w += z.w;
      y.sum += sm.l[w][r] * exp2_fast(sm.m[w][r] - y.top);
    }
    return y;
  }

  // Writes the CTA's rows after a piece: to `out`, or (slot >= 0) to the workspace.
  static __device__ __forceinline__ void finish(const Kv8AttnDev& a, const Smem& sm, const Place& at, int slot) {
    const bool expired = sm.expired;
#pragma unroll 1
    for (int i = threadIdx.x; i < kRows * D / 4; i += kThreads) {
      const int r = i / (D / 4), d = (i % (D / 4)) * 4;
      const Part y = cta_part(sm, expired, r, d);
      if (slot >= 0) {
        *reinterpret_cast<float4*>(a.part_o + ((int64_t)slot * kRows + r) * D + d) = y.x;
        if (d == 0) *reinterpret_cast<float2*>(a.part_ml + ((int64_t)slot * kRows + r) * 2) = make_float2(y.top, y.sum);
      } else if (at.rt * kRows + r < a.rows) {
        write_out(a, at.b, at.h, at.rt * kRows + r, d, y.x, y.sum);
      }
    }
  }

  // The same for a cluster of `ctas` CTAs that share a segment: every CTA stores its sums of row r into the shared
  // memory of CTA r % ctas, which finishes the row after one barrier of the cluster (nothing reads another
  // CTA's memory after that, so each may end).
  static __device__ __forceinline__ void finish_cluster(const Kv8AttnDev& a, Smem& sm, const Place& at, int rank, int ctas, int log2) {
    const bool expired = sm.expired;
    cg::cluster_group cluster = cg::this_cluster();
    cluster.barrier_wait();                       // all CTAs of the cluster run (they arrived when they began)
#pragma unroll 1
    for (int i = threadIdx.x; i < kRows * D / 4; i += kThreads) {
      const int r = i / (D / 4), d = (i % (D / 4)) * 4, owner = r & (ctas - 1), slot = rank * (kRows >> log2) + (r >> log2);
      const Part y = cta_part(sm, expired, r, d);
      *cluster.map_shared_rank(reinterpret_cast<float4*>(&sm.sent[slot][d]), owner) = y.x;
      if (d == 0) *cluster.map_shared_rank(&sm.sent_ml[slot], owner) = make_float2(y.top, y.sum);
    }
    cluster.sync();
    const int each = kRows >> log2;               // rows of a CTA; a row is a stretch of D/4 threads
    const int stretch = threadIdx.x / (D / 4), d = (threadIdx.x % (D / 4)) * 4;
#pragma unroll 1
    for (int k = stretch; k < each; k += kThreads / (D / 4)) {
      const int r = k * ctas + rank;
      if (at.rt * kRows + r >= a.rows) break;
      float top = kNoMax, sum = 0.f;
#pragma unroll 1
      for (int c = 0; c < ctas; ++c) top = fmaxf(top, sm.sent_ml[c * each + k].x);
      float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 2
      for (int c = 0; c < ctas; ++c) {
        const float2 ml = sm.sent_ml[c * each + k];
        const float is = exp2_fast(ml.x - top);
        const float4 z = *reinterpret_cast<const float4*>(&sm.sent[c * each + k][d]);
        x.x += z.x * is; x.y += z.y * is; x.z += z.z * is; x.w += z.w * is;
        sum += ml.y * is;
      }
      write_out(a, at.b, at.h, at.rt * kRows + r, d, x, sum);
    }
  }

  // out[row][d .. d+3] = x / sum, 0 for a row that saw nothing.
  static __device__ __forceinline__ void write_out(const Kv8AttnDev& a, int b, int h, int r, int d, float4 x, float sum) {
    const int pos = position(a, r), head = h * a.group + r - pos * a.group;
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

__device__ __forceinline__ uint32_t unit_tiles(const Kv8AttnDev& a, int u) {
  return a.blocks ? kv8_tiles(a, u / a.pg.heads, u % a.pg.heads) : kv8_tiles(a, u, 0);
}

// The place of this CTA (by one warp, its lanes taking units 32 at a time); false: no part is left for it.
// A unit's tiles are those of its segments: all heads and row tiles of b, or with lists all row tiles of (b, h).
template <int kWarps>
__device__ __forceinline__ bool line_place(const Kv8AttnDev& a, Place& at, int lane) {
  const int units = a.blocks ? a.pg.batch * a.pg.heads : a.pg.batch;
  const uint32_t per = a.blocks ? a.row_tiles : a.row_tiles * a.pg.heads;
  const uint32_t n0 = lane < units ? unit_tiles(a, lane) : 0u;
  uint32_t total = n0;
#pragma unroll 4
  for (int u = lane + 32; u < units; u += 32) total += unit_tiles(a, u);
  total = __reduce_add_sync(0xffffffffu, total) * per;
  if (total == 0) return false;
  Line line{};
  uint32_t target;                 // this CTA's first part, or tile
  if (a.aligned) {
    line.size = max((total - 1) / (gridDim.x - a.segments) + 1, (uint32_t)kWarps);
    target = blockIdx.x;
  } else {
    const uint32_t parts = min(gridDim.x, (total + kWarps - 1) / kWarps);
    if (blockIdx.x >= parts) return false;
    line.size = total / parts;
    line.longer = total - line.size * parts;
    target = line.even_begin(blockIdx.x);
  }
  uint32_t before = 0;             // parts, or tiles, of the units before
#pragma unroll 1
  for (int u0 = 0; u0 < units; u0 += 32) {
    const int u = u0 + lane;
    const uint32_t n = u0 == 0 ? n0 : u < units ? unit_tiles(a, u) : 0u;
    const uint32_t count = per * (a.aligned ? (n + line.size - 1) / line.size : n);
    uint32_t upto = count;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t x = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += x;
    }
    const uint32_t hit = __ballot_sync(0xffffffffu, before + upto > target);
    if (hit) {
      if (lane == __ffs(hit) - 1) {
        const uint32_t rest = target - (before + upto - count);
        uint32_t seg;
        if (a.aligned) {
          // tiles are counted from the segment's first one: the part needs no others
          const uint32_t of_segment = (n + line.size - 1) / line.size;
          seg = rest / of_segment;
          const uint32_t part = rest - seg * of_segment, share = n / of_segment, longer = n - share * of_segment;
          at.start = 0;
          at.at = part * share + min(part, longer);
          at.end = at.at + share + (part < longer ? 1 : 0);
        } else {
          seg = rest / n;
          at.start = before + upto - count + seg * n;
          at.at = target;
          at.end = line.even_begin(blockIdx.x + 1);
        }
        at.begin = at.at;
        at.n = n;
        at.rt = (int)(seg % a.row_tiles);
        at.b = a.blocks ? u / a.pg.heads : u;
        at.h = a.blocks ? u % a.pg.heads : (int)(seg / a.row_tiles);
        at.len = kv8_len(a, at.b);
        at.line = line;
      }
      return true;
    }
    before += __shfl_sync(0xffffffffu, upto, 31);
  }
  return false;
}

template <int D, int NT, bool E5M2, bool BF16>
__global__ void __launch_bounds__(32 * ka_warps(D, NT), ka_ctas(D, NT))
kv8_attn_kernel(const Kv8AttnDev a, const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map) {
  using K = Kv8Attn<D, NT, E5M2, BF16>;
  extern __shared__ uint8_t smem_raw[];
  typename K::Smem& sm = *reinterpret_cast<typename K::Smem*>(smem_raw + (-smem_addr(smem_raw) & 1023u));
  __shared__ bool s_some;
  __shared__ Place at;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(&k_map) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&v_map) : "memory");
    sm.expired = 0;
  }
  if (a.cluster > 1) cg::this_cluster().barrier_arrive();
  if (lane == 0) {
    for (int i = 0; i < K::kStages; ++i) mbar_init(smem_addr(&sm.arrived[warp][i]), 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  wait_for_previous_grid();
  allow_dependents();              // what follows may be set up from here on; it waits for this grid's end
  // The CTA's place is kept in shared memory: it would cost the tile loop registers.
  if (a.cluster) {
    // the CTAs of a cluster share a segment, and need not know the others
    if (threadIdx.x == 0) {
      const uint32_t rank = blockIdx.x & (a.cluster - 1), seg = blockIdx.x >> a.cluster_log2;
      const int bh = a.row_tiles == 1 ? (int)seg : (int)(seg / a.row_tiles);
      at.rt = (int)(seg - bh * a.row_tiles);
      at.b = (int)a.by_heads.quotient(bh);
      at.h = bh - at.b * a.pg.heads;
      at.len = kv8_len(a, at.b);
      at.n = kv8_tiles(a, at.b, at.h);
      at.start = 0;
      const uint32_t share = at.n >> a.cluster_log2, longer = at.n & (a.cluster - 1);
      at.begin = at.at = rank * share + min(rank, longer);
      at.end = at.at + share + (rank < longer ? 1 : 0);
    }
  } else {
    if (warp == 0) {
      const bool some = line_place<K::kWarps>(a, at, lane);
      if (lane == 0) s_some = some;
    }
  }
  __syncthreads();
  if (!a.cluster && !s_some) return;
  K k;
  uint32_t turn = 0;               // tiles that this warp has taken
  for (;;) {
    if (!sm.expired) k.piece(a, &k_map, &v_map, sm, at, turn, warp, lane);   // stable here: set before a piece's last barrier
    if (a.cluster > 1) {
      K::finish_cluster(a, sm, at, (int)(blockIdx.x & (a.cluster - 1)), a.cluster, a.cluster_log2);
      return;
    }
    const uint32_t first = at.at - at.start, last = min(at.n, at.end - at.start);
    const bool cut = !a.cluster && (first > 0 || last < at.n);
    K::finish(a, sm, at, cut ? 2 * (int)blockIdx.x + (at.at == at.begin ? 0 : 1) : -1);
    if (a.cluster) return;
    const bool done = at.start + last >= at.end;
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");   // the warps' sums were ordinary stores to the ring's place
    __syncthreads();                                  // the buffers and the place have been read
    if (threadIdx.x == 0) {
      if (first == 0)
        a.info[((int64_t)at.b * a.pg.heads + at.h) * a.row_tiles + at.rt] =
            make_int4((int)blockIdx.x, (int)at.line.last_part(a.aligned, blockIdx.x, at.start, at.n), at.at == at.begin ? 0 : 1, 0);
      if (!done) {                                    // the next segment that has tiles
        at.at = at.start + last;
        at.start += at.n;
        if (++at.rt == a.row_tiles) {
          at.rt = 0;
          do {
            if (++at.h == a.pg.heads) {
              at.h = 0;
              ++at.b;
            }
            at.n = kv8_tiles(a, at.b, at.h);
          } while (at.n == 0);
          at.len = kv8_len(a, at.b);
        }
      }
    }
    if (done) return;
    __syncthreads();
  }
}

// Rows of segments of several parts, and of segments without tiles.  One CTA per (segment, row); its warps
// take the parts in turn, four at a time, each lane D/32 neighbouring dims.
constexpr int kKmWarps = 8;

template <int D, int NT, bool BF16>
__global__ void __launch_bounds__(kKmWarps * 32) kv8_merge_kernel(const Kv8AttnDev a) {
  constexpr int kRows = NT * 8, kPer = D / 32, kAtOnce = 4;
  __shared__ float s_m[kKmWarps], s_l[kKmWarps];
  __shared__ __align__(16) float s_o[kKmWarps][D];
  const int seg = blockIdx.x / kRows, r = blockIdx.x % kRows;
  const int rt = seg % a.row_tiles, bh = seg / a.row_tiles;
  const int b = (int)a.by_heads.quotient(bh), h = bh - b * a.pg.heads;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  wait_for_previous_grid();
  allow_dependents();
  // both on their way at once; nobody wrote the entry of a segment without tiles, and nothing follows it
  const int4 info = a.info[seg];
  const bool empty = kv8_tiles(a, b, h) == 0;
  if (rt * kRows + r >= a.rows) return;
  float top = kNoMax, sum = 0.f;
  float x[kPer] = {};
  if (!empty) {
    if (info.x == info.y) return;                     // written by its CTA
#pragma unroll 1
    for (int c0 = info.x + warp; c0 <= info.y; c0 += kKmWarps * kAtOnce) {
      float2 ml[kAtOnce];
      float y[kAtOnce][kPer];
#pragma unroll
      for (int j = 0; j < kAtOnce; ++j) {
        const int c = c0 + j * kKmWarps;
        ml[j] = make_float2(kNoMax, 0.f);
#pragma unroll
        for (int i = 0; i < kPer; ++i) y[j][i] = 0.f;
        if (c <= info.y) {
          const int64_t row = (int64_t)(2 * c + (c == info.x ? info.z : 0)) * kRows + r;
          ml[j] = *reinterpret_cast<const float2*>(a.part_ml + row * 2);
          const float* src = a.part_o + row * D + lane * kPer;
#pragma unroll
          for (int i = 0; i < kPer; i += 2) {
            const float2 z = *reinterpret_cast<const float2*>(src + i);
            y[j][i] = z.x;
            y[j][i + 1] = z.y;
          }
        }
      }
      float now = top;
#pragma unroll
      for (int j = 0; j < kAtOnce; ++j) now = fmaxf(now, ml[j].x);
      const float was = exp2_fast(top - now);
      sum *= was;
#pragma unroll
      for (int i = 0; i < kPer; ++i) x[i] *= was;
#pragma unroll
      for (int j = 0; j < kAtOnce; ++j) {
        const float is = exp2_fast(ml[j].x - now);
        sum += ml[j].y * is;
#pragma unroll
        for (int i = 0; i < kPer; ++i) x[i] += y[j][i] * is;
      }
      top = now;
    }
  }
  if (lane == 0) {
    s_m[warp] = top;
    s_l[warp] = sum;
  }
#pragma unroll
  for (int i = 0; i < kPer; ++i) s_o[warp][lane * kPer + i] = x[i];
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
  int nt, row_tiles, cluster, aligned;
  int64_t segments, ctas;          // ctas: of the first kernel
  uint64_t info_bytes, ml_bytes, o_bytes;
};

template <int D, int NT>
constexpr int ka_smem() {
  return (int)sizeof(typename Kv8Attn<D, NT, false, true>::Smem) + 1024;   // + the ring's alignment
}

// A launch of `ctas` CTAs in clusters; `attrs` must outlive the configuration.
template <int D, int NT>
static cudaLaunchConfig_t ka_config(cudaLaunchAttribute (&attrs)[2], int64_t ctas, int cluster, cudaStream_t st) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)ctas);
  cfg.blockDim = dim3(32 * ka_warps(D, NT));
  cfg.dynamicSmemBytes = ka_smem<D, NT>();
  cfg.stream = st;
  attrs[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attrs[0].val.programmaticStreamSerializationAllowed = 1;
  attrs[1].id = cudaLaunchAttributeClusterDimension;
  attrs[1].val.clusterDim.x = (unsigned)std::max(cluster, 1);
  attrs[1].val.clusterDim.y = attrs[1].val.clusterDim.z = 1;
  cfg.attrs = attrs;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  return cfg;
}

// Clusters of 2^log2 CTAs that run at once: fewer than the CTAs that do, as a cluster lies within one group of
// multiprocessors (33 of 8 instead of 37 at 128 dims).  Asked for once per device and shape.
template <int D, int NT>
static int64_t clusters_at_once(int log2, int64_t slots) {
  static std::atomic<int> known[64][4];
  int dev = 0;
  if (log2 == 0 || cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return slots >> log2;
  int n = known[dev][log2].load(std::memory_order_relaxed);
  if (n == 0) {
    const auto kernel = kv8_attn_kernel<D, NT, false, true>;
    cudaLaunchAttribute attrs[2];
    cudaLaunchConfig_t cfg = ka_config<D, NT>(attrs, slots >> log2 << log2, 1 << log2, nullptr);
    cfg.attrs = attrs + 1;
    cfg.numAttrs = 1;
    if (ensure_smem_limit(reinterpret_cast<const void*>(kernel), ka_smem<D, NT>(), "mskv_kv8_attention") ||
        cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess || n <= 0) {
      cudaGetLastError();
      return slots >> log2;
    }
    known[dev][log2].store(n, std::memory_order_relaxed);
  }
  return n;
}

static int64_t clusters_at_once(int d, int nt, int log2, int64_t slots) {
  if (d == 256) return clusters_at_once<256, 1>(log2, slots);
  if (d == 128) return nt == 1 ? clusters_at_once<128, 1>(log2, slots) : clusters_at_once<128, 2>(log2, slots);
  return nt == 1 ? clusters_at_once<64, 1>(log2, slots) : clusters_at_once<64, 2>(log2, slots);
}

static Kv8Plan make_plan(const mskv_kv8_attn_desc& d) {
  Kv8Plan p{};
  const int rows = d.q_heads / d.pages.kv_heads * d.q_len;
  p.nt = rows <= 8 || d.pages.head_dim == 256 ? 1 : 2;   // 256 dims: two column tiles do not fit the registers
  p.row_tiles = (rows + p.nt * 8 - 1) / (p.nt * 8);
  p.segments = (int64_t)d.pages.batch * d.pages.kv_heads * p.row_tiles;
  const int64_t most = d.blocks ? (int64_t)d.num_blocks * (d.pages.page_size / 16) : ((int64_t)d.max_tokens + 15) / 16;
  const int warps = ka_warps(d.pages.head_dim, p.nt);
  const int64_t slots = (int64_t)sms_of_device() * ka_ctas(d.pages.head_dim, p.nt);   // CTAs that run at once
  // A cluster of 1 to 8 CTAs for each segment, merged in its shared memory, spares the line's look-up and the second
  // kernel (4 us, and 4 more where parts would cross segments), but the segments wait for the longest: its tiles a
  // warp, at the time that one takes on an SM of its own.  It is chosen while that is less than what the codes take
  // at 6.3 TB/s, as far as the clusters fill the GPU, and those 4 us; of whole caches, whose lengths may differ, 0.85
  // of the codes' time and 25 us at most are counted (lists are of one length as a rule): past that the line's 4 us are
  // little beside what uneven lengths cost a cluster (16 of 32768 below, 107 us of codes a cluster).  A cluster has two tiles
  // a warp or fewer where all clusters run at once.  Measured, cluster / line: 28/4 heads, 8 sequences of 16384 tokens
  // 28.0 / 31.6 us (ragged down to an eighth 23.1 / 22.0), 16 of 4096 17.0 / 20.8, 64 of up to 4096 41.2 / 46.1, 4 of
  // 32768 41.0 / 31.7, 5 of up to 9000 14.2 / 11.6; 40/8 heads, 30 of up to 2900 30.3 / 36.4, 16 of 32768 175 / 173, ragged
  // 144 / 107; 8/1 heads of 256 dims, 2 positions, 46 of 846 13.5 / 19.5; 32/8 heads of 64 dims, 4 positions, 6 of up to
  // 9001 25.7 / 20.2; lists of 516 pages, 40/8 heads, 10 sequences 43.7 / 40.2, of 208, 32/8
  // heads of 64 dims, 8 sequences 14.1 / 15.4.
  const int d_of = d.pages.head_dim;
  const double tile_us = d_of == 64 ? 0.73 : d_of == 256 ? 1.14 : p.nt == 1 ? 0.84 : 1.25;
  const double codes_us = (double)p.segments * most * 32 * d_of / 6.3e6;
  int cluster = 1;
  for (int log2 = 1; (1 << log2) <= kKaMaxCluster && most > 2 * warps * cluster; ++log2) {
    if (p.segments > clusters_at_once(d_of, p.nt, log2, slots)) break;
    cluster = 1 << log2;
  }
  const double alone_us = tile_us * ((most + warps * cluster - 1) / (warps * cluster));
  const double fill = (double)p.segments * cluster / slots;
  const double line_us = fill * (d.blocks ? codes_us : std::min(0.85 * codes_us, 25.0)) + (p.segments * 2 > slots ? 8 : 4);
  // Of several waves of segments, each is a CTA's own while the longest takes no longer than the starts that a CTA of
  // the line has for all of its segments, 8 us each.  Own / line, ragged, 5 positions: 96/8 heads of 64 dims, 43 lists
  // of up to 504 tokens 40 / 127 us; 56/8 heads, 30 of up to 997 54 / 150; of 256 dims, 96/8 heads, 28 of up to 1100 130 / 259;
  // 64/8 heads, 4 positions, 64 of up to 8192 268 / 350.
  const bool many = p.segments > slots && alone_us <= 8.0 * fill;
  if (most <= 4 * warps * cluster || many || (fill <= 1 && alone_us <= line_us)) {
    p.cluster = cluster;
    p.ctas = p.segments * cluster;
    return p;
  }
  // Long lines in twice as many parts, so that CTAs which get less of the memory's bandwidth take fewer: 40/8
  // heads, 16 sequences of 32768 tokens (886 tiles a CTA in one wave) 174 us against 181; 28/4 heads, 8 of
  // 16384 (111 a CTA) 36.8 against 32.2, as the second wave starts its pipelines anew.
  p.ctas = std::min<int64_t>(p.segments * most > 512 * slots ? 2 * slots : slots, (p.segments * most + warps - 1) / warps);
  // Parts that do not cross segments leave some CTAs without work, a part that does costs a second start:
  // 33.0 us against 37.1 for the 8 sequences of 16384 tokens above.
  p.aligned = p.segments * 2 <= p.ctas;
  const uint64_t rows_held = 2 * (uint64_t)p.ctas * p.nt * 8;
  p.info_bytes = ((uint64_t)p.segments * sizeof(int4) + 255) / 256 * 256;
  p.ml_bytes = (rows_held * 2 * sizeof(float) + 255) / 256 * 256;
  p.o_bytes = rows_held * d.pages.head_dim * sizeof(float);
  return p;
}

static std::atomic<int32_t> g_expire{0};   // mskv_kv8_expire_waits

// K or V as a 4-D tensor [page][head][row][dim] of bytes, in boxes of 16 rows and at most 128 dims.
static bool encode_pages_map(CUtensorMap* m, uint8_t* base, const Kv8Dev& pg, int d) {
  const EncodeTiledFn encode = tensor_map_encoder();
  if (!encode) return false;
  const cuuint64_t dims[4] = {(cuuint64_t)d, (cuuint64_t)pg.page_size, (cuuint64_t)pg.heads, (cuuint64_t)pg.num_pages};
  // a single head or page has no stride of its own
  const cuuint64_t page_bytes = (cuuint64_t)pg.page_size * d;
  const cuuint64_t strides[3] = {(cuuint64_t)d, pg.heads > 1 ? (cuuint64_t)pg.sh : page_bytes,
                                 pg.num_pages > 1 ? (cuuint64_t)pg.sp : page_bytes};
  const cuuint32_t box[4] = {(cuuint32_t)std::min(d, 128), 16, 1, 1};
  const cuuint32_t estr[4] = {1, 1, 1, 1};
  return encode(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, base, dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                d < 128 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int D, int NT, bool E5M2, bool BF16>
static int launch_attn(const Kv8AttnDev& a, const Kv8Plan& p, cudaStream_t st) {
  static_assert(sizeof(typename Kv8Attn<D, NT, E5M2, BF16>::Smem) == sizeof(typename Kv8Attn<D, NT, false, true>::Smem));
  const auto kernel = kv8_attn_kernel<D, NT, E5M2, BF16>;
  if (const int rc = ensure_smem_limit(reinterpret_cast<const void*>(kernel), ka_smem<D, NT>(), "mskv_kv8_attention")) return rc;
  CUtensorMap maps[2];
  if (!encode_pages_map(&maps[0], a.pg.k, a.pg, D) || !encode_pages_map(&maps[1], a.pg.v, a.pg, D))
    return fail(MSKV_ERR_CUDA, "mskv_kv8_attention: the cache's layout cannot be encoded for TMA");
  cudaLaunchAttribute attrs[2];
  const cudaLaunchConfig_t cfg = ka_config<D, NT>(attrs, p.ctas, p.cluster, st);
  const cudaError_t launched = cudaLaunchKernelEx(&cfg, kernel, a, maps[0], maps[1]);
  if (launched != cudaSuccess) return cuda_status(launched, "mskv_kv8_attention launch");
  if (const int rc = after_launch("mskv_kv8_attention")) return rc;
  if (p.cluster) return MSKV_OK;
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
  constexpr int64_t kMaxStride = (int64_t)1 << 40;
  if ((d->pages.kv_heads > 1 && (d->pages.stride_h <= 0 || d->pages.stride_h >= kMaxStride)) ||
      (d->pages.num_pages > 1 && (d->pages.stride_page <= 0 || d->pages.stride_page >= kMaxStride)) ||
      d->pages.num_pages > INT_MAX)
    return fail(MSKV_ERR_RANGE, "%s: stride_page and stride_h must lie in (0, 2^40), num_pages below 2^31", what);
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
  if (!(fabsf(d->scale) <= 2e38f)) return fail(MSKV_ERR_ARG, "%s: scale must be finite", what);   // times log2(e) too
  return MSKV_OK;
}

}  // namespace mskv

using namespace mskv;

extern "C" uint64_t mskv_kv8_attention_workspace_bytes(const mskv_kv8_attn_desc* d) {
  if (check_attn(d)) return 0;
  const Kv8Plan p = make_plan(*d);
  return p.info_bytes + p.ml_bytes + p.o_bytes;
}

extern "C" int32_t mskv_kv8_expire_waits(int32_t on) { return g_expire.exchange(on != 0, std::memory_order_relaxed); }

extern "C" int mskv_kv8_attention(const mskv_kv8_attn_desc* d, void* stream) {
  if (const int rc = check_attn(d)) return rc;
  if (!d->q || !d->out || !d->lens) return fail(MSKV_ERR_ARG, "mskv_kv8_attention: NULL q, out or lens");
  if (const int rc = check_words("mskv_kv8_attention", d->lens, d->blocks, d->counts, d->status)) return rc;
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
  a.by_heads = Divisor((uint32_t)a.pg.heads);
  a.cluster = p.cluster;
  const int parts = a.pg.page_size / 16;
  a.parts_log2 = parts & (parts - 1) ? -1 : parts >= 8 ? 3 : parts >> 1;
  for (a.cluster_log2 = 0; (2 << a.cluster_log2) <= p.cluster; ++a.cluster_log2) {}
  a.aligned = p.aligned;
  a.vec_q = (q_bits & 15) == 0;
  a.pow2_page = (a.pg.page_size & (a.pg.page_size - 1)) == 0;
  a.expire = g_expire.load(std::memory_order_relaxed);
  const bool e5m2 = d->pages.dtype == MSKV_DT_FP8_E5M2, bf16 = d->dtype == MSKV_DT_BF16;
  const cudaStream_t st = as_stream(stream);
  switch (d->pages.head_dim) {
    case 64: return attn_rows<64>(a, p, e5m2, bf16, st);
    case 128: return attn_rows<128>(a, p, e5m2, bf16, st);
    default: return attn_rows<256>(a, p, e5m2, bf16, st);
  }
}
