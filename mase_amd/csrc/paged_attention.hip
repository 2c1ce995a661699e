// Attention of one new token per sequence over a paged key-value cache for gfx950: x = scaling (q . k) + mask,
// out = softmax(x) v, with the cache held in 16 bits or as MX codes (paged_kv.hpp).  The attention core of the reference's
// Llama block on a cache (models/llama/modeling_llama.py:362-480, nn/quantized/modules/llama/attention.py:182-187, 352-395)
// for one query.  Bound by HBM: every cached byte is read once.
//
// One wavefront takes 32 slots at a time through two matrix products with up to 16 query heads of one cached head on the
// other side, and no LDS: scores S^T = K Q^T (A = 16 key rows, B = the queries, both with 8 consecutive elements per lane),
// which leaves lane (i, g) = (lane % 16, lane / 16) with the scores of head i at slots 4 g .. 4 g + 3 of each 16-slot tile;
// their exponentials are then already the B operand of O^T += V^T P^T when its 8 contraction slots of group g are those 8.
// The V^T operand (lane = a place in the head dimension, 8 slots) comes from 16-byte pieces of V's rows as they lie: with
// row i of output tile n standing for element c i + n (c = D / 16), the c elements that a lane needs of one slot for all
// tiles are consecutive, and pairs of slots are joined in registers by byte permutes.  Output tile n, register r of lane
// (i, g) is then head i, element c (4 g + r) + n.
// MX codes are widened to 16 bits in registers as they are used (exact), two per conversion instruction for MXFP.
#include "paged_kv.hpp"

namespace mase {
namespace {

typedef __bf16 pa_bf16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 pa_f16x8_t __attribute__((ext_vector_type(8)));
typedef float pa_f32x4_t __attribute__((ext_vector_type(4)));

constexpr int kWaves = 4;
constexpr int kSlots = 32;                  // per wavefront and step
constexpr int kChunkStep = kWaves * kSlots;  // lengths of parts are multiples of it
constexpr int kHeadTile = 16;
constexpr float kLog2e = 1.4426950408889634f;

struct DecodeParams {
  PagedKv c;
  const unsigned char* q;
  size_t q_sb, q_sh;  // bytes
  const int32_t* lengths;
  const unsigned char* mask;
  size_t mask_sb;  // elements
  int mask_f32;
  unsigned char* out;
  float* part_o;   // [batch * heads][splits][D]
  float* part_ml;  // [batch * heads][splits][2]
  float* scores;   // [batch * heads][score_stride], NULL without weights
  float* weights;
  size_t w_sb, w_sh;
  size_t score_stride;
  int heads, group, head_tiles, max_length, chunk, splits;
  float scaling;
};

template <bool F16>
__device__ __forceinline__ pa_f32x4_t mfma16(const uint32_t* a, const uint32_t* b, pa_f32x4_t c) {
  const uint4 av = make_uint4(a[0], a[1], a[2], a[3]), bv = make_uint4(b[0], b[1], b[2], b[3]);
  if constexpr (F16)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(pa_f16x8_t, av), __builtin_bit_cast(pa_f16x8_t, bv), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(pa_bf16x8_t, av), __builtin_bit_cast(pa_bf16x8_t, bv), c, 0, 0, 0);
}

// value of the lanes 16 apart and 32 apart combined
__device__ __forceinline__ float max_over_groups(float v) {
  v = fmaxf(v, __shfl_xor(v, 16, 64));
  return fmaxf(v, __shfl_xor(v, 32, 64));
}
__device__ __forceinline__ float sum_over_groups(float v) {
  v += __shfl_xor(v, 16, 64);
  return v + __shfl_xor(v, 32, 64);
}

// How a format's rows are read.  Keys: lane group g of a row takes kRun consecutive elements per load, kKeyLoads loads
// 4 kRun apart.  Values: a lane takes c = D / 16 consecutive elements of each of its 8 slots.
template <int D, int FMT>
struct Rows {
  static constexpr int kBits = FMT == MASE_KV_16BIT ? 16 : (FMT == MASE_KV_MXFP4 ? 4 : 8);
  static constexpr int kRun = (128 / kBits < D / 4) ? 128 / kBits : D / 4;
  static constexpr int kKeyLoads = D / (4 * kRun);
  static constexpr int kKeyBytes = kRun * kBits / 8;
  static constexpr int kC = D / 16;
  static constexpr int kValBytes = kC * kBits / 8;
  static constexpr int kKeyWords = kKeyBytes / 4;
  static constexpr int kValWords = kValBytes < 4 ? 1 : kValBytes / 4;
  static constexpr bool kPacked = FMT != MASE_KV_16BIT;
  static constexpr int kScaleWords = kPacked ? (D == 256 ? 2 : 1) : 1;
};

template <int D, int FMT, bool F16>
__global__ __launch_bounds__(256) void paged_decode_kernel(DecodeParams p) {
  using R = Rows<D, FMT>;
  constexpr float kGrow = F16 ? 4.0f : 8.0f;   // see the reference point of the exponentials below
  constexpr float kShift = F16 ? 11.0f : 0.0f;
  extern __shared__ __attribute__((aligned(16))) float lds[];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int i = lane & 15, g = lane >> 4;
  const int split = blockIdx.x, b = blockIdx.z;
  const int hk = (int)blockIdx.y / p.head_tiles, tile = (int)blockIdx.y % p.head_tiles;
  const int rows = min(kHeadTile, p.group - tile * kHeadTile);  // query heads here
  const int head0 = hk * p.group + tile * kHeadTile;
  const int length = kv_length(p.lengths[b], p.max_length, p.c.table_pages, p.c.page_shift);
  const int lo = split * p.chunk, hi = min(lo + p.chunk, length);
  if (split > 0 && lo >= length) return;  // an empty part; part 0 always reports
  const int32_t* table = p.c.table + (size_t)b * p.c.table_stride;
  const int page_mask = (1 << p.c.page_shift) - 1;

  uint32_t qf[D / 32][4];
#pragma unroll
  for (int u = 0; u < R::kKeyLoads; ++u)
#pragma unroll
    for (int s = 0; s < R::kRun / 8; ++s) {
      uint32_t* f = qf[u * (R::kRun / 8) + s];
      if (i < rows) kv_load<16>(p.q + (size_t)b * p.q_sb + (size_t)(head0 + i) * p.q_sh + (u * 4 * R::kRun + g * R::kRun + s * 8) * 2, f);
      else f[0] = f[1] = f[2] = f[3] = 0;
    }

  // page and first row of the 16-slot tiles of a step (uniform); a page number that must not be followed reads page 0 and
  // its slots count as absent
  auto tile_page = [&](int slot, int& row) __attribute__((always_inline)) {
    row = slot & page_mask;
    return slot < hi ? kv_page(table, p.c.table_pages, p.c.page_shift, p.c.num_pages, slot) : -1;
  };

  uint32_t kr[2][R::kKeyLoads][R::kKeyWords], ksc[2][R::kScaleWords];
  uint32_t vr[8][R::kValWords], vsc[2];
  auto load_keys = [&](const int* page, const int* row) __attribute__((always_inline)) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int pg = max(page[t], 0);
      const unsigned char* base = p.c.k + (size_t)pg * p.c.k_page + (size_t)hk * p.c.k_head + (size_t)row[t] * p.c.k_slot;
#pragma unroll
      for (int u = 0; u < R::kKeyLoads; ++u)
        kv_load<R::kKeyBytes>(base + (uint32_t)i * p.c.k_slot + (uint32_t)((u * 4 + g) * R::kKeyBytes), kr[t][u]);
      if constexpr (R::kPacked)
        kv_load<D / 32>((const unsigned char*)p.c.ks + ((((size_t)pg * p.c.heads + hk) << p.c.page_shift) + row[t]) * (D / 32) + i * (D / 32), ksc[t]);
    }
  };
  auto load_values = [&](const int* page, const int* row) __attribute__((always_inline)) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int pg = max(page[t], 0);
      const unsigned char* base = p.c.v + (size_t)pg * p.c.v_page + (size_t)hk * p.c.v_head + (size_t)row[t] * p.c.v_slot;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        kv_load<R::kValBytes>(base + (uint32_t)(4 * g + j) * p.c.v_slot + (uint32_t)(i * R::kValBytes), vr[4 * t + j]);
      if constexpr (R::kPacked)
        vsc[t] = *(const uint32_t*)(p.c.vs + (((((size_t)pg * p.c.heads + hk) * (D / 32)) + (i * R::kC) / 32) << p.c.page_shift) + row[t] + 4 * g);
    }
  };

  pa_f32x4_t o[R::kC];
#pragma unroll
  for (int n = 0; n < R::kC; ++n) o[n] = pa_f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
  float m = -__builtin_inff(), l = 0.0f;

  for (int t0 = lo + wave * kSlots; t0 < hi; t0 += kChunkStep) {
    int page[2], row[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) page[t] = tile_page(t0 + 16 * t, row[t]);
    load_keys(page, row);
    load_values(page, row);
    // scores of head i at slots t0 + 16 t + 4 g + r
    float x[2][4];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      pa_f32x4_t acc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int u = 0; u < R::kKeyLoads; ++u) {
        uint32_t wide[R::kRun / 2];
        float scale = 0.0f;
        if constexpr (R::kPacked) {
          const int blk = (u * 4 * R::kRun + g * R::kRun) / 32;
          const uint32_t word = R::kScaleWords == 1 ? ksc[t][0] : (blk < 4 ? ksc[t][0] : ksc[t][R::kScaleWords - 1]);
          scale = kv_scale<FMT>((word >> (8 * (blk & 3))) & 0xFFu);
        }
        kv_widen<FMT, F16, R::kRun>(kr[t][u], scale, wide);
#pragma unroll
        for (int s = 0; s < R::kRun / 8; ++s) acc = mfma16<F16>(wide + 4 * s, qf[u * (R::kRun / 8) + s], acc);
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) x[t][r] = acc[r] * p.scaling;
    }
    const bool whole = t0 + kSlots <= hi && page[0] >= 0 && page[1] >= 0;
    uint32_t gone = 0;  // bit 4 t + r: the slot is absent
    if (!whole || p.mask != nullptr) {
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int slot = t0 + 16 * t + 4 * g + r;
          bool absent = page[t] < 0 || slot >= hi;
          if (p.mask != nullptr && !absent) {
            const size_t at = (size_t)b * p.mask_sb + slot;
            const float add = p.mask_f32 ? ((const float*)p.mask)[at] : DTypeTraits<F16 ? MASE_DT_F16 : MASE_DT_BF16>::load1(p.mask, at);
            absent = add == -__builtin_inff();
            x[t][r] += add;
          }
          if (absent) {
            x[t][r] = -__builtin_inff();
            gone |= 1u << (4 * t + r);
          }
        }
    }
    if (p.scores != nullptr && i < rows) {
      float* sp = p.scores + ((size_t)b * p.heads + head0 + i) * p.score_stride + t0 + 4 * g;
#pragma unroll
      for (int t = 0; t < 2; ++t) *(float4*)(sp + 16 * t) = make_float4(x[t][0], x[t][1], x[t][2], x[t][3]);
    }
    // The reference point m of the exponentials moves only when some head has met a score more than kGrow (in the exponent's
    // unit) above it: probabilities then reach 2^kGrow, and most steps skip the rescaling and the exchange between lanes.
    float mx = x[0][0];
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) mx = fmaxf(mx, x[t][r]);
    if (__builtin_amdgcn_ballot_w64((mx - m) * kLog2e > kGrow) != 0) {
      const float mn = fmaxf(m, max_over_groups(mx));
      const float alpha = mn == -__builtin_inff() ? 1.0f : __builtin_amdgcn_exp2f((m - mn) * kLog2e);
      m = mn;
      l *= alpha;
#pragma unroll
      for (int n = 0; n < R::kC; ++n) o[n] *= alpha;
    }
    const float ms = m == -__builtin_inff() ? 0.0f : m;
    // fp16 probabilities are held 2^kShift up, where small ones keep their bits (fp16 loses them below 2^-14)
    uint32_t pf[4];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      float e[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        e[r] = __builtin_amdgcn_exp2f((x[t][r] - ms) * kLog2e + kShift);
        l += e[r];
      }
      pf[2 * t] = kv_pack2<F16>(e[0], e[1]);
      pf[2 * t + 1] = kv_pack2<F16>(e[2], e[3]);
    }
    // values: widened slot by slot, then pairs of slots joined
    uint32_t wv[8][R::kC / 2];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float scale = R::kPacked ? kv_scale<FMT>((vsc[j >> 2] >> (8 * (j & 3))) & 0xFFu) : 0.0f;
      kv_widen<FMT, F16, R::kC>(vr[j], scale, wv[j]);
    }
    if (gone != 0) {  // what an absent slot holds must not meet its probability of zero: it may be infinite or NaN
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if ((gone >> j) & 1u) {
#pragma unroll
          for (int n = 0; n < R::kC / 2; ++n) wv[j][n] = 0;
        }
    }
#pragma unroll
    for (int n = 0; n < R::kC; ++n) {
      uint32_t f[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) f[q] = __builtin_amdgcn_perm(wv[2 * q + 1][n >> 1], wv[2 * q][n >> 1], (n & 1) ? 0x07060302u : 0x05040100u);
      o[n] = mfma16<F16>(f, pf, o[n]);
    }
  }

  // join the wavefronts: [wave][head] maxima and sums, [wave][head][D] outputs
  l = sum_over_groups(l);
  float* sm = lds;
  float* sl = lds + kWaves * kHeadTile;
  float* so = lds + 2 * kWaves * kHeadTile;
  if (g == 0) {
    sm[wave * kHeadTile + i] = m;
    sl[wave * kHeadTile + i] = l;
  }
  if (i < rows) {
    float* dst = so + (size_t)(wave * rows + i) * D;
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int n = 0; n < R::kC; n += 4)
        *(float4*)(dst + R::kC * (4 * g + r) + n) = make_float4(o[n][r], o[n + 1][r], o[n + 2][r], o[n + 3][r]);
  }
  __syncthreads();
  const bool direct = p.splits == 1 && p.scores == nullptr;
  const float down = __builtin_amdgcn_exp2f(-kShift);
  for (int e = threadIdx.x; e < rows * D; e += 256) {
    const int r = e / D, d = e % D;
    float top = sm[r];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) top = fmaxf(top, sm[w * kHeadTile + r]);
    float acc = 0.0f, sum = 0.0f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const float mw = sm[w * kHeadTile + r];
      // a wavefront without a slot has m = -inf and zeros; one that met only NaN has them in its sums, which must show
      const float f = mw == top ? 1.0f : __builtin_amdgcn_exp2f((mw - top) * kLog2e);
      acc += f * so[(size_t)(w * rows + r) * D + d];
      sum += f * sl[w * kHeadTile + r];
    }
    const size_t bh = (size_t)b * p.heads + head0 + r;
    if (direct) {
      const float y = sum == 0.0f ? 0.0f : acc / sum;
      DTypeTraits<F16 ? MASE_DT_F16 : MASE_DT_BF16>::store1(p.out, bh * D + d, y);
    } else {
      p.part_o[(bh * p.splits + split) * D + d] = acc * down;
      if (d == 0) {
        p.part_ml[(bh * p.splits + split) * 2] = top;
        p.part_ml[(bh * p.splits + split) * 2 + 1] = sum * down;
      }
    }
  }
}

// Joins the parts.  grid (x, cached head, sequence): a work-group takes the query heads x, x + gridDim.x, ... of its cached
// head and, with weights, the slots of its share.
constexpr int kMaxGroup = 256;
constexpr int kWeightSlots = 1024;  // per work-group

template <int D, bool F16>
__global__ __launch_bounds__(256) void paged_decode_join_kernel(DecodeParams p) {
  __shared__ float top_s[kMaxGroup], inv_s[kMaxGroup];
  __shared__ __attribute__((aligned(16))) float red[256 * 4];
  const int hk = blockIdx.y, b = blockIdx.z, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int length = kv_length(p.lengths[b], p.max_length, p.c.table_pages, p.c.page_shift);
  const int parts = max(1, (length + p.chunk - 1) / p.chunk);
  const size_t bh0 = (size_t)b * p.heads + (size_t)hk * p.group;
  const int step = (int)gridDim.x;
  const bool all = p.scores != nullptr;
  // reference point and 1 / sum of each head that this work-group needs
  for (int h = wave; h < p.group; h += 4) {
    if (!all && h % step != (int)blockIdx.x) continue;
    const float* ml = p.part_ml + (bh0 + h) * p.splits * 2;
    float top = -__builtin_inff();
    for (int s = lane; s < parts; s += 64) top = fmaxf(top, ml[2 * s]);
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) top = fmaxf(top, __shfl_xor(top, d, 64));
    float sum = 0.0f;
    for (int s = lane; s < parts; s += 64) sum += ml[2 * s + 1] * (ml[2 * s] == top ? 1.0f : __builtin_amdgcn_exp2f((ml[2 * s] - top) * kLog2e));
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) sum += __shfl_xor(sum, d, 64);
    if (lane == 0) {
      top_s[h] = top;
      inv_s[h] = sum == 0.0f ? 0.0f : 1.0f / sum;
    }
  }
  __syncthreads();
  constexpr int kCols = D / 4, kRows = 256 / kCols;  // threads along the head dimension, parts side by side
  const int col = tid % kCols, rowi = tid / kCols;
  for (int h = blockIdx.x; h < p.group; h += step) {
    const float* ml = p.part_ml + (bh0 + h) * p.splits * 2;
    const float* po = p.part_o + (bh0 + h) * p.splits * D + col * 4;
    const float top = top_s[h];
    float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int s = rowi; s < parts; s += kRows) {
      const float f = ml[2 * s] == top ? 1.0f : __builtin_amdgcn_exp2f((ml[2 * s] - top) * kLog2e);
      const float4 v = *(const float4*)(po + (size_t)s * D);
      acc.x += f * v.x; acc.y += f * v.y; acc.z += f * v.z; acc.w += f * v.w;
    }
    ((float4*)red)[tid] = acc;
    __syncthreads();
    if (tid < kCols) {
      for (int r = 1; r < kRows; ++r) {
        const float4 v = ((const float4*)red)[r * kCols + tid];
        acc.x += v.x; acc.y += v.y; acc.z += v.z; acc.w += v.w;
      }
      const float inv = inv_s[h];
      uint2 y;
      y.x = kv_pack2<F16>(acc.x * inv, acc.y * inv);
      y.y = kv_pack2<F16>(acc.z * inv, acc.w * inv);
      *(uint2*)(p.out + ((bh0 + h) * D + tid * 4) * 2) = y;
    }
    __syncthreads();
  }
  if (!all) return;
  float* wrow = p.weights + (size_t)b * p.w_sb + (size_t)hk * p.w_sh;
  const int end = min(length, ((int)blockIdx.x + 1) * kWeightSlots);
  for (int s = (int)blockIdx.x * kWeightSlots + tid; s < end; s += 256) {
    float acc = 0.0f;
    for (int h = 0; h < p.group; ++h) {
      const float x = p.scores[(bh0 + h) * p.score_stride + s];
      const float e = x == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f((x - top_s[h]) * kLog2e);
      acc += e * inv_s[h];
    }
    wrow[s] += acc;
  }
}

struct DecodePlan {
  int chunk, splits, head_tiles;
  size_t score_stride, part_floats, ml_floats, score_floats;
};

// How the cache's length is split: parts of a whole number of work-group steps, about kPartsPerCu work-groups per CU when
// all sequences are as long as the longest may be.
constexpr int kPartsPerCu = 8;

DecodePlan decode_plan(size_t batch, size_t heads, size_t kv_heads, size_t head_dim, size_t max_length, bool weights) {
  DecodePlan d{};
  const size_t group = heads / kv_heads;
  d.head_tiles = (int)((group + kHeadTile - 1) / kHeadTile);
  int cus = device_cu_count();
  if (cus <= 0) cus = 256;
  const size_t rows = batch * kv_heads * d.head_tiles;
  const size_t steps = (max_length + kChunkStep - 1) / kChunkStep;
  size_t splits = (size_t)cus * kPartsPerCu / (rows ? rows : 1);
  if (splits < 1) splits = 1;
  if (splits > steps) splits = steps ? steps : 1;
  const size_t per = steps ? (steps + splits - 1) / splits : 1;
  d.chunk = (int)(per * kChunkStep);
  d.splits = (int)(steps ? (steps + per - 1) / per : 1);
  d.score_stride = steps * kChunkStep;
  const bool join = d.splits > 1 || weights;
  d.part_floats = join ? batch * heads * d.splits * head_dim : 0;
  d.ml_floats = join ? (batch * heads * d.splits * 2 + 3) / 4 * 4 : 0;
  d.score_floats = weights ? batch * heads * d.score_stride : 0;
  return d;
}

template <int D, int FMT, bool F16>
int launch_decode(const DecodeParams& p, size_t batch, hipStream_t st) {
  const int lds = (int)sizeof(float) * (2 * kWaves * kHeadTile + kWaves * min(p.group, kHeadTile) * D);
  static std::atomic<uint64_t> attr_done{0};
  const void* fn = (const void*)paged_decode_kernel<D, FMT, F16>;
  if (!set_dynamic_lds_once(attr_done, fn, (int)sizeof(float) * (2 * kWaves * kHeadTile + kWaves * kHeadTile * D))) return MASE_ERR_LAUNCH;
  const dim3 grid((unsigned)p.splits, (unsigned)(p.c.heads * p.head_tiles), (unsigned)batch);
  hipLaunchKernelGGL((paged_decode_kernel<D, FMT, F16>), grid, dim3(256), (size_t)lds, st, p);
  return MASE_OK;
}

template <int D>
int launch_decode_d(const DecodeParams& p, int format, bool f16, size_t batch, hipStream_t st) {
  int rc;
  switch (format * 2 + (f16 ? 1 : 0)) {
    case MASE_KV_16BIT * 2: rc = launch_decode<D, MASE_KV_16BIT, false>(p, batch, st); break;
    case MASE_KV_16BIT * 2 + 1: rc = launch_decode<D, MASE_KV_16BIT, true>(p, batch, st); break;
    case MASE_KV_MXINT8 * 2: rc = launch_decode<D, MASE_KV_MXINT8, false>(p, batch, st); break;
    case MASE_KV_MXINT8 * 2 + 1: rc = launch_decode<D, MASE_KV_MXINT8, true>(p, batch, st); break;
    case MASE_KV_MXFP8_E4M3 * 2: rc = launch_decode<D, MASE_KV_MXFP8_E4M3, false>(p, batch, st); break;
    case MASE_KV_MXFP8_E4M3 * 2 + 1: rc = launch_decode<D, MASE_KV_MXFP8_E4M3, true>(p, batch, st); break;
    case MASE_KV_MXFP8_E5M2 * 2: rc = launch_decode<D, MASE_KV_MXFP8_E5M2, false>(p, batch, st); break;
    case MASE_KV_MXFP8_E5M2 * 2 + 1: rc = launch_decode<D, MASE_KV_MXFP8_E5M2, true>(p, batch, st); break;
    case MASE_KV_MXFP4 * 2: rc = launch_decode<D, MASE_KV_MXFP4, false>(p, batch, st); break;
    default: rc = launch_decode<D, MASE_KV_MXFP4, true>(p, batch, st); break;
  }
  if (rc != MASE_OK || p.part_o == nullptr) return rc;
  const size_t shares = p.scores != nullptr ? ((size_t)p.max_length + kWeightSlots - 1) / kWeightSlots : (size_t)p.group;
  const dim3 grid((unsigned)(shares ? shares : 1), (unsigned)p.c.heads, (unsigned)batch);
  if (f16) hipLaunchKernelGGL((paged_decode_join_kernel<D, true>), grid, dim3(256), 0, st, p);
  else hipLaunchKernelGGL((paged_decode_join_kernel<D, false>), grid, dim3(256), 0, st, p);
  return MASE_OK;
}

}  // namespace
}  // namespace mase

extern "C" size_t mase_paged_attention_decode_workspace_bytes(size_t batch, size_t heads, size_t kv_heads, size_t head_dim,
                                                              size_t max_length, int with_weights) {
  if (kv_heads == 0 || heads % kv_heads != 0 || max_length > 0x7FFFFF00u) return 0;
  const mase::DecodePlan d = mase::decode_plan(batch, heads, kv_heads, head_dim, max_length, with_weights != 0);
  return (d.part_floats + d.ml_floats + d.score_floats) * sizeof(float);
}

extern "C" int mase_paged_attention_decode(const mase_paged_kv* cache, const void* q, size_t q_stride_b, size_t q_stride_h,
                                           size_t heads, const int32_t* lengths, size_t max_length, float scaling,
                                           const void* mask, int mask_dtype, size_t mask_stride_b, float* weights,
                                           size_t w_stride_b, size_t w_stride_h, void* out, void* workspace,
                                           size_t workspace_bytes, void* stream) {
  using namespace mase;
  DecodeParams p{};
  const int rc = paged_kv_params(cache, p.c);
  if (rc != MASE_OK) return rc;
  if (heads == 0 || heads % cache->kv_heads != 0 || heads / cache->kv_heads > (size_t)kMaxGroup) return MASE_ERR_SHAPE;
  if (max_length > 0x7FFFFF00u) return MASE_ERR_SHAPE;
  if (!(scaling > -3.0e38f && scaling < 3.0e38f)) return MASE_ERR_PARAM;
  if (mask != nullptr && mask_dtype != cache->dtype && mask_dtype != MASE_DT_F32) return MASE_ERR_DTYPE;
  if (cache->batch == 0) return MASE_OK;
  if (q == nullptr || lengths == nullptr || out == nullptr) return MASE_ERR_NULL;
  if (!aligned16(q) || !aligned16(out) || q_stride_b % 8 != 0 || q_stride_h % 8 != 0) return MASE_ERR_ALIGN;
  const DecodePlan d = decode_plan(cache->batch, heads, cache->kv_heads, cache->head_dim, max_length, weights != nullptr);
  if (cache->kv_heads * d.head_tiles > 65535) return MASE_ERR_SHAPE;
  const size_t need = (d.part_floats + d.ml_floats + d.score_floats) * sizeof(float);
  if (need != 0 && (workspace == nullptr || workspace_bytes < need)) return MASE_ERR_WORKSPACE;
  if (need != 0 && !aligned16(workspace)) return MASE_ERR_ALIGN;
  p.q = (const unsigned char*)q;
  p.q_sb = q_stride_b * 2;
  p.q_sh = q_stride_h * 2;
  p.lengths = lengths;
  p.mask = (const unsigned char*)mask;
  p.mask_sb = mask_stride_b;
  p.mask_f32 = mask_dtype == MASE_DT_F32;
  p.out = (unsigned char*)out;
  if (need != 0) {
    p.part_o = (float*)workspace;
    p.part_ml = p.part_o + d.part_floats;
    p.scores = weights != nullptr ? p.part_ml + d.ml_floats : nullptr;
  }
  p.weights = weights;
  p.w_sb = w_stride_b;
  p.w_sh = w_stride_h;
  p.score_stride = d.score_stride;
  p.heads = (int)heads;
  p.group = (int)(heads / cache->kv_heads);
  p.head_tiles = d.head_tiles;
  p.max_length = (int)max_length;
  p.chunk = d.chunk;
  p.splits = d.splits;
  p.scaling = scaling;
  hipStream_t st = (hipStream_t)stream;
  const bool f16 = cache->dtype == MASE_DT_F16;
  int lrc;
  if (cache->head_dim == 64) lrc = launch_decode_d<64>(p, cache->format, f16, cache->batch, st);
  else if (cache->head_dim == 128) lrc = launch_decode_d<128>(p, cache->format, f16, cache->batch, st);
  else lrc = launch_decode_d<256>(p, cache->format, f16, cache->batch, st);
  if (lrc != MASE_OK) return lrc;
  return hipGetLastError() == hipSuccess ? MASE_OK : MASE_ERR_LAUNCH;
}
