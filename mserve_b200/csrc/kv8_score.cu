// Block scores of the 8-bit paged cache (mskv_kv8_block_score).
//
// score(block) = 2^e * sum_d (max_d * P_d + min_d * N_d), P_d = sum_g max(q_gd, 0) and
// N_d = sum_g min(q_gd, 0) over the query heads of the KV head: the sum over the heads of each
// head's largest possible q.k in the block, collapsed to one product of length 2D.
//
// Bound by the bounds' bytes (2D a block and head).  A warp takes 16 blocks at a time, straight
// from global memory into the A fragments of mma.sync m16n8k16 (the contraction's order is free,
// so each lane's 16 contiguous codes are four k-steps' worth).  The weights are the B operand: the fp32
// P and N, scaled to magnitudes below 2, split in two fp16 terms in columns 0 and 1 (the second times
// 2^12), so the products are exact and the weights keep 23 bits; lane c = 0 of a row holds
// both columns' sums.  FMAs in fp32 would need an unpacking and an FMA per code and a
// shuffle reduction; the tensor core needs neither.  The next tile's page ids are looked up during a tile, its
// bounds loaded as soon as the tile's are in the products.
// Measured: 56/8 heads, 128 dims, 16 sequences of up to 65536 tokens in pages of 16 (77 MB) 16.0 us = 0.74 of the
// copy rate; 28/4 heads, 8 of 16384 (8.6 MB) 4.8 us, a chain of launch, page id, bounds and products.
#include <algorithm>

#include "kv8.cuh"

namespace mskv {

struct BlockScoreDev {
  Kv8Dev pg;
  const char* q;
  int64_t q_sb, q_sh;
  const int32_t* lens;
  float* scores;
  int64_t stride;
  uint32_t* status;
  int32_t group, max_blocks, chunks, tiles;   // chunks of a (b, h); tiles of 16 blocks a warp takes of one
  Divisor by_chunks, by_heads;
};

constexpr int kBsWarps = 8;

template <int D, bool E5M2, bool BF16>
__global__ void __launch_bounds__(kBsWarps * 32, D <= 128 ? 4 : 2) kv8_block_score_kernel(const BlockScoreDev a) {
  constexpr int kVec = D / 32;              // 16-byte loads of a lane per block (64 codes a step of 4 lanes)
  constexpr int kK = 2 * D / 16;            // k-steps
  __shared__ __align__(16) uint2 s_w[kK][32];   // the weights [min | max] as B fragments
  __shared__ uint32_t s_top[kBsWarps];

  wait_for_previous_grid();
  allow_dependents();
  const int bh = (int)a.by_chunks.quotient(blockIdx.x), chunk = (int)blockIdx.x - bh * a.chunks;
  const int b = (int)a.by_heads.quotient(bh), h = bh - b * a.pg.heads;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  const int first = chunk * a.tiles * kBsWarps * 16;
  const int j0 = first + warp * 16 + g;
  const int32_t* const table = a.pg.page_table + (int64_t)b * a.pg.pt_stride;
  // the first tile's table entries, before the length is known
  const int entry[2] = {j0 < a.max_blocks ? table[j0] : -1, j0 + 8 < a.max_blocks ? table[j0 + 8] : -1};
  const int64_t len = min((int64_t)max(a.lens[b], 0), (int64_t)a.max_blocks * a.pg.page_size);
  const int held = (int)(((uint32_t)len + a.pg.page_size - 1) / a.pg.page_size);
  if (first >= held) return;                // the whole CTA

  // Block j's page: -2 where there is no block, -1 where its page is unmapped.
  const auto page_of = [&](int j, int p) { return j >= held ? -2 : p >= 0 && p < a.pg.num_pages ? p : -1; };
  uint4 x[2][kVec];
  int e[2];
  const auto load = [&](const int (&page)[2]) {
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int64_t ph = (int64_t)page[r] * a.pg.heads + h;
      e[r] = 0;
#pragma unroll
      for (int v = 0; v < kVec; ++v) x[r][v] = make_uint4(0u, 0u, 0u, 0u);
      if (page[r] >= 0) {
        const uint8_t* src = a.pg.bounds + ph * 2 * D + 16 * c;
#pragma unroll
        for (int v = 0; v < kVec; ++v) x[r][v] = ld_stream16(src + 64 * v);
        e[r] = a.pg.exps[ph * 2];
      }
    }
  };
  // the first tile's bounds are on their way while the weights are made
  int page[2] = {page_of(j0, entry[0]), page_of(j0 + 8, entry[1])};
  load(page);

  // weights: sums over the heads, then both terms at a common power of two
  float up = 0.f, down = 0.f;
  const int d = threadIdx.x;
  if (d < D) {
    const char* q = a.q + (int64_t)b * a.q_sb + (int64_t)h * a.group * a.q_sh + d * 2;
#pragma unroll 8
    for (int i = 0; i < a.group; ++i) {
      const float y = q_elem<BF16>(q + (int64_t)i * a.q_sh);
      // a NaN reaches both sums
      up += y < 0.f ? 0.f : y;
      down += y > 0.f ? 0.f : y;
    }
  }
  const uint32_t mu = __float_as_uint(up) & 0x7fffffffu, md = __float_as_uint(down) & 0x7fffffffu;
  uint32_t top = max(mu < 0x7f800000u ? mu : 0u, md < 0x7f800000u ? md : 0u);
  top = __reduce_max_sync(0xffffffffu, top);
  if (lane == 0) s_top[warp] = top;
  for (int i = threadIdx.x; i < kK * 32; i += kBsWarps * 32)
    if ((i & 31) >= 8) s_w[i >> 5][i & 31] = make_uint2(0u, 0u);        // columns 2 to 7
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kBsWarps; ++i) top = max(top, s_top[i]);
  const int eq = min(max((int)(top >> 23) - 127, -120), 120);
  if (d < D) {
    const float f = pow2i(-eq);
    const float w[2] = {down * f, up * f};
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const __half first_term = __float2half_rn(w[i]);
      const float rest = (w[i] - __half2float(first_term)) * 4096.f;
      // element 64 v + 16 c' + 4 k + m of [min | max] is in k-step 4 v + k, lane 4 * column + c', half m
      const int at = i * D + d, v = at >> 6, c1 = (at >> 4) & 3, k = (at >> 2) & 3, m = at & 3;
      __half* const lane0 = reinterpret_cast<__half*>(&s_w[4 * v + k][c1]);
      lane0[m] = first_term;
      lane0[16 + m] = __float2half_rn(fabsf(w[i]) <= 65504.f ? rest : 0.f);   // column 1; 0 beside an infinity or NaN
    }
  }
  __syncthreads();
  const float q_scale = pow2i(eq);

#pragma unroll 1
  for (int t = 0; t < a.tiles; ++t) {
    const int j = j0 + t * kBsWarps * 16;
    if (j - g >= held) break;
    int ahead[2] = {-2, -2};
    if (t + 1 < a.tiles) {
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const int k = j + kBsWarps * 16 + 8 * r;
        ahead[r] = page_of(k, k < held ? table[k] : -1);
      }
    }
    float acc[2][4] = {};                   // two chains of k-steps
#pragma unroll
    for (int v = 0; v < kVec; ++v) {
      const uint32_t lo_rows[4] = {x[0][v].x, x[0][v].y, x[0][v].z, x[0][v].w};
      const uint32_t hi_rows[4] = {x[1][v].x, x[1][v].y, x[1][v].z, x[1][v].w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint32_t a0, a1, a2, a3;
        codes_to_half<E5M2>(lo_rows[i], a0, a2);
        codes_to_half<E5M2>(hi_rows[i], a1, a3);
        const uint2 w = s_w[v * 4 + i][lane];
        mma_f16(acc[i & 1], a0, a1, a2, a3, w.x, w.y);
      }
    }
    const int was[2] = {page[0], page[1]}, e_was[2] = {e[0], e[1]};
    page[0] = ahead[0];
    page[1] = ahead[1];
    load(page);
    if (c == 0) {
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        if (was[r] == -2) continue;
        float s = (acc[0][2 * r] + acc[1][2 * r]) + (acc[0][2 * r + 1] + acc[1][2 * r + 1]) * (1.f / 4096.f);
        s = s * pow2i(e_was[r]) * q_scale;
        if (was[r] < 0) {
          s = __int_as_float(0xff800000);
          if (a.status) atomicOr(a.status, MSKV_STATUS_BAD_PAGE);
        }
        a.scores[(int64_t)bh * a.stride + j + 8 * r] = s;
      }
    }
  }
}

template <int D, bool E5M2>
static int launch_block_score(const BlockScoreDev& a, bool bf16, int64_t ctas, cudaStream_t st) {
  const cudaError_t e = launch_dependent(bf16 ? kv8_block_score_kernel<D, E5M2, true> : kv8_block_score_kernel<D, E5M2, false>,
                                         dim3((unsigned)ctas), dim3(kBsWarps * 32), 0, st, a);
  if (e != cudaSuccess) return cuda_status(e, "mskv_kv8_block_score launch");
  return after_launch("mskv_kv8_block_score");
}

template <int D>
static int block_score_cache(const BlockScoreDev& a, bool e5m2, bool bf16, int64_t ctas, cudaStream_t st) {
  return e5m2 ? launch_block_score<D, true>(a, bf16, ctas, st) : launch_block_score<D, false>(a, bf16, ctas, st);
}

}  // namespace mskv

using namespace mskv;

extern "C" int mskv_kv8_block_score(const mskv_kv8_score_desc* d, void* stream) {
  if (!d) return fail(MSKV_ERR_ARG, "mskv_kv8_block_score: NULL descriptor");
  if (const int rc = check_kv8(d->pages, "mskv_kv8_block_score")) return rc;
  if (d->dtype != MSKV_DT_BF16 && d->dtype != MSKV_DT_F16)
    return fail(MSKV_ERR_DTYPE, "mskv_kv8_block_score: q must be bf16 or f16");
  if (!d->pages.bounds) return fail(MSKV_ERR_ARG, "mskv_kv8_block_score: the cache has no bounds");
  if (!d->q || !d->lens || !d->scores) return fail(MSKV_ERR_ARG, "mskv_kv8_block_score: NULL q, lens or scores");
  if (const int rc = check_words("mskv_kv8_block_score", d->lens, d->scores, d->status)) return rc;
  if (d->q_heads <= 0 || d->q_heads % d->pages.kv_heads)
    return fail(MSKV_ERR_ARG, "mskv_kv8_block_score: q_heads must be a multiple of kv_heads");
  if (d->max_blocks < 0 || d->max_blocks > d->pages.max_pages || d->max_blocks > d->scores_stride)
    return fail(MSKV_ERR_ARG, "mskv_kv8_block_score: max_blocks must lie in [0, min(max_pages, scores_stride)]");
  if (d->max_blocks > INT_MAX - (1 << 16)) return fail(MSKV_ERR_RANGE, "mskv_kv8_block_score: max_blocks too large");
  if (((uintptr_t)d->q | (uintptr_t)d->q_stride_b | (uintptr_t)d->q_stride_h) & 1)
    return fail(MSKV_ERR_ARG, "mskv_kv8_block_score: q must be aligned to its elements");
  if (d->max_blocks == 0) return MSKV_OK;
  BlockScoreDev a{};
  a.pg = to_dev(d->pages);
  a.q = static_cast<const char*>(d->q);
  a.q_sb = d->q_stride_b; a.q_sh = d->q_stride_h;
  a.lens = d->lens;
  a.scores = d->scores;
  a.stride = d->scores_stride;
  a.status = d->status;
  a.group = d->q_heads / d->pages.kv_heads;
  a.max_blocks = d->max_blocks;
  // Tiles a warp takes per CTA: one while that fits one wave of the GPU, up to four beyond, so that the weights' set-up is
  // shared.  One, two, four, eight: 8 sequences of 1024 pages, 4 heads 4.8, 5.8, 7.7, 11.3 us; 16 of 2048, 8 heads
  // 20.0, 16.6, 14.7, 15.5 us; 64 of 256, 4 heads 6.8, 7.2, 7.2, 7.3 us.
  const int64_t segs = (int64_t)a.pg.batch * a.pg.heads;
  const int64_t rows = ((int64_t)d->max_blocks + 16 * kBsWarps - 1) / (16 * kBsWarps);
  a.tiles = (int)std::min<int64_t>(4, std::max<int64_t>(1, segs * rows / (2 * sms_of_device())));
  a.chunks = (int)((rows + a.tiles - 1) / a.tiles);
  a.by_chunks = Divisor((uint32_t)a.chunks);
  a.by_heads = Divisor((uint32_t)a.pg.heads);
  const int64_t ctas = segs * a.chunks;
  if (ctas > INT_MAX) return fail(MSKV_ERR_RANGE, "mskv_kv8_block_score: too many blocks for one call");
  const bool e5m2 = d->pages.dtype == MSKV_DT_FP8_E5M2, bf16 = d->dtype == MSKV_DT_BF16;
  const cudaStream_t st = as_stream(stream);
  switch (d->pages.head_dim) {
    case 64: return block_score_cache<64>(a, e5m2, bf16, ctas, st);
    case 128: return block_score_cache<128>(a, e5m2, bf16, ctas, st);
    default: return block_score_cache<256>(a, e5m2, bf16, ctas, st);
  }
}
