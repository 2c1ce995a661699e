// Attention of one new token per sequence over a paged key-value cache for gfx950: x = scaling (q . k) + mask,
// out = softmax(x) v, with the cache held in 16 bits or as MX codes (paged_kv.hpp).  The attention core of the reference's
// Llama block on a cache (models/llama/modeling_llama.py:362-480, nn/quantized/modules/llama/attention.py:182-187, 352-395)
// for one query.  Bound by HBM: every cached byte is read once for each tile of 16 query heads of its cached head.
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
//
// Whole calls, 64 sequences of 8192 slots, 8 cached heads for 32 query heads: heads of 128 in bf16 (2.15 GB) 355 us, MXINT8
// (1.11 GB) 198 us, MXFP8 e4m3 190 us, MXFP4 (0.57 GB) 112 us; heads of 64 in bf16 (1.07 GB) 181 us, of 256 (2.15 GB, 4096
// slots) 356 us: 5.1 .. 6.1 TB/s, where a large copy moves 4.9 (read and written).  What brought it there: shares of equal
// length over resident work-groups instead of parts of the longest sequence (64 sequences of 65 .. 4096 slots 150 -> 125 us);
// page numbers through the scalar cache, so that no load of a page number waits for the rows in flight (MXFP4 99 -> 79 us);
// two work-groups on a CU (three: 392 us for the bf16 case, one: 154 us for the MXFP4 case).  Vector instructions issue in
// 15 % of the cycles with bf16 rows, 69 % with MXINT8 (two conversions, two products and half a packing an element) and 62 %
// with MXFP4; rows two steps ahead instead of one, or steps of 64 slots, were no faster.
#pragma once
#include "paged_attention.hpp"

namespace mase {
namespace {

typedef __bf16 pa_bf16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 pa_f16x8_t __attribute__((ext_vector_type(8)));
typedef float pa_f32x4_t __attribute__((ext_vector_type(4)));

// int32 in memory that no kernel writes while this one runs: a uniform index reads it through the scalar cache, apart from
// the vector loads in flight (which a vector load of a page number would have to wait for)
typedef const __attribute__((address_space(4))) int32_t scalar_int;

constexpr int kWaves = 4;
constexpr int kHeadTile = 16;
constexpr float kLog2e = 1.4426950408889634f;

template <bool F16>
__device__ __forceinline__ pa_f32x4_t mfma16(const uint32_t* a, const uint32_t* b, pa_f32x4_t c) {
  const uint4 av = make_uint4(a[0], a[1], a[2], a[3]), bv = make_uint4(b[0], b[1], b[2], b[3]);
  if constexpr (F16)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(pa_f16x8_t, av), __builtin_bit_cast(pa_f16x8_t, bv), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(pa_bf16x8_t, av), __builtin_bit_cast(pa_bf16x8_t, bv), c, 0, 0, 0);
}

// low or high 16 bits of a word as a number
template <bool F16>
__device__ __forceinline__ float half_of(uint32_t w, int high) {
  if constexpr (F16) return f16_bits_to_f32(high ? w >> 16 : w & 0xFFFFu);
  return bits2f(high ? w & 0xFFFF0000u : w << 16);
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
  static constexpr int kSlots = 32;                 // per wavefront and step
  static constexpr int kUnit = kWaves * kSlots;      // per work-group and step
  static constexpr int kPerCu = D == 256 && kBits >= 8 ? 1 : 2;  // work-groups resident on a CU
};

// units (work-group steps) of a sequence's row; a sequence without a slot has one too, which writes its zeros
template <int UNIT>
__device__ __forceinline__ int row_units(int length) {
  return length > 0 ? (length + UNIT - 1) / UNIT : 1;
}

// The sequences with their units in one line are cut into equal shares; a share is taken by one work-group for each (cached
// head, head tile), all of them resident: sequences of any lengths keep every CU busy to the end, and the heads of a page,
// which lie side by side in memory, are read at about the same time.  A row (sequence, cached head, head tile) that lies in
// one share is finished by it; the pieces of a row that is cut go to the work-group's first or last place (2 wg, 2 wg + 1)
// and are joined by the second kernel.
template <int D, int FMT, bool F16, int EXTRA>
__global__ __launch_bounds__(256, (Rows<D, FMT>::kPerCu)) void paged_decode_kernel(DecodeParams p) {
  using R = Rows<D, FMT>;
  constexpr float kGrow = F16 ? 4.0f : 8.0f;   // see the reference point of the exponentials below
  constexpr float kShift = F16 ? 11.0f : 0.0f;
  extern __shared__ __attribute__((aligned(16))) float lds[];
  __shared__ uint32_t wave_sum[kWaves];
  __shared__ int start_b, start_at;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int i = lane & 15, g = lane >> 4;
  const int page_mask = (1 << p.c.page_shift) - 1;
  const int row_heads = p.c.heads * p.head_tiles;  // rows of a sequence
  const int rh = (int)blockIdx.x % row_heads, hk = rh / p.head_tiles, tile = rh % p.head_tiles;
  const int rows = min(kHeadTile, p.group - tile * kHeadTile);  // query heads here
  const int head0 = hk * p.group + tile * kHeadTile;
  auto length_of = [&](int b) __attribute__((always_inline)) { return kv_length(((const scalar_int*)p.lengths)[b], p.max_length, p.c.table_pages, p.c.page_shift); };

  // this work-group's share [u0, u1) of the units (32 bits: the host's limit), and where it starts
  const int per = (p.batch + 255) / 256, b_lo = min((int)threadIdx.x * per, p.batch), b_hi = min(b_lo + per, p.batch);
  uint32_t mine = 0;
  for (int b = b_lo; b < b_hi; ++b) mine += (unsigned)row_units<R::kUnit>(length_of(b));
  uint32_t run = mine;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const uint32_t o = __shfl_up(run, d, 64);
    if (lane >= d) run += o;
  }
  if (lane == 63) wave_sum[wave] = run;
  __syncthreads();
  uint32_t before = run - mine, total = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    before += w < wave ? wave_sum[w] : 0u;
    total += wave_sum[w];
  }
  const unsigned shares = gridDim.x / (unsigned)row_heads;
  const uint32_t share = (total + shares - 1) / shares;
  const uint32_t u0 = min(share * (blockIdx.x / (unsigned)row_heads), total), u1 = min(u0 + share, total);
  if (blockIdx.x == 0) {
    uint32_t at = before;
    for (int b = b_lo; b < b_hi; ++b) {
      p.plan[b] = at;
      at += (unsigned)row_units<R::kUnit>(length_of(b));
    }
    if (threadIdx.x == 0) {
      p.plan[p.batch] = total;
      p.plan[p.batch + 1] = share;
    }
  }
  if (u0 >= u1) return;
  if (before <= u0 && u0 < before + mine) {  // one thread
    uint32_t at = before;
    int b = b_lo;
    for (; b < b_hi - 1; ++b) {
      const uint32_t n = (unsigned)row_units<R::kUnit>(length_of(b));
      if (u0 < at + n) break;
      at += n;
    }
    start_b = b;
    start_at = (int)(u0 - at);
  }
  __syncthreads();
  int b = __builtin_amdgcn_readfirstlane(start_b);
  int a = __builtin_amdgcn_readfirstlane(start_at);
  int length = length_of(b), n_units = row_units<R::kUnit>(length);
  int left = __builtin_amdgcn_readfirstlane((int)(u1 - u0));

#pragma unroll 1
  for (bool first_piece = true;; first_piece = false) {
    const int e = min(n_units, a + left);  // this row's units a .. e - 1
    // (a lane's value read back keeps what follows from it, the addresses of pages above all, in scalar registers)
    const int lo = a * R::kUnit, hi = __builtin_amdgcn_readfirstlane(min(e * R::kUnit, length));
    const scalar_int* table = (const scalar_int*)(p.c.table + (size_t)b * p.c.table_stride);

    uint32_t qf[D / 32][4];
#pragma unroll
    for (int u = 0; u < R::kKeyLoads; ++u)
#pragma unroll
      for (int s = 0; s < R::kRun / 8; ++s) {
        uint32_t* f = qf[u * (R::kRun / 8) + s];
        if (i < rows) kv_load<16>(p.q + (size_t)b * p.q_sb + (size_t)(head0 + i) * p.q_sh + (u * 4 * R::kRun + g * R::kRun + s * 8) * 2, f);
        else f[0] = f[1] = f[2] = f[3] = 0;
      }

    // page and first row of a 16-slot tile (uniform); a page number that must not be followed reads page 0 and its slots
    // count as absent
    auto tile_page = [&](int slot, int& row) __attribute__((always_inline)) {
      row = slot & page_mask;
      // (an entry that is there is read even if the slot is not: no branch)
      const int at = min(slot >> p.c.page_shift, p.c.table_pages - 1);
      const int pg = table[at];
      return slot < hi && pg >= 0 && pg < p.c.num_pages ? pg : -1;
    };
    uint32_t kr[2][R::kKeyLoads][R::kKeyWords], ksc[2][R::kScaleWords];
    uint32_t vr[8][R::kValWords], vsc[2];
    constexpr bool kMask = EXTRA >= kMaskOwn;
    constexpr int kMaskSize = EXTRA == kMaskF32 ? 4 : 2, kMaskWords = kMaskSize;  // bytes of a value, words of four
    uint32_t mk[2][kMaskWords];
    const unsigned char* mask_row = kMask ? p.mask + (size_t)b * p.mask_sb * kMaskSize : nullptr;
    // lane offsets from a tile's first row
    const uint32_t k_lane = (uint32_t)i * p.c.k_slot + (uint32_t)(g * R::kKeyBytes);
    uint32_t v_lane[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) v_lane[j] = (uint32_t)(4 * g + j) * p.c.v_slot + (uint32_t)(i * R::kValBytes);
    const uint32_t vs_lane = ((uint32_t)((i * R::kC) / 32) << p.c.page_shift) + (uint32_t)(4 * g);
    auto load_keys = [&](const int* page, const int* row) __attribute__((always_inline)) {
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const int pg = max(page[t], 0);
        const unsigned char* base = p.c.k + (size_t)pg * p.c.k_page + (size_t)hk * p.c.k_head + (size_t)row[t] * p.c.k_slot;
#pragma unroll
        for (int u = 0; u < R::kKeyLoads; ++u)
          kv_load<R::kKeyBytes>(base + (k_lane + (uint32_t)(u * 4 * R::kKeyBytes)), kr[t][u]);
        if constexpr (R::kPacked)
          kv_load<D / 32>((const unsigned char*)p.c.ks + ((((size_t)pg * p.c.heads + hk) << p.c.page_shift) + row[t]) * (D / 32) + (uint32_t)(i * (D / 32)), ksc[t]);
      }
    };
    auto load_values = [&](const int* page, const int* row) __attribute__((always_inline)) {
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const int pg = max(page[t], 0);
        const unsigned char* base = p.c.v + (size_t)pg * p.c.v_page + (size_t)hk * p.c.v_head + (size_t)row[t] * p.c.v_slot;
#pragma unroll
        for (int j = 0; j < 4; ++j)
          kv_load<R::kValBytes>(base + v_lane[j], vr[4 * t + j]);
        if constexpr (R::kPacked)
          vsc[t] = *(const uint32_t*)(p.c.vs + ((((size_t)pg * p.c.heads + hk) * (D / 32)) << p.c.page_shift) + row[t] + vs_lane);
      }
    };
    // what is added to the scores of slots s0 + 16 t + 4 g + r, as it lies in memory, four at a time (rows have any
    // alignment); where the four reach past the row something else is read, and the step reads them one by one
    auto load_mask = [&](int s0) __attribute__((always_inline)) {
      if constexpr (kMask) {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const int s = s0 + 16 * t + 4 * g;
          const unsigned char* at = s <= p.max_length - 4 ? mask_row + (size_t)s * kMaskSize : p.q;
          __builtin_memcpy(mk[t], at, 4 * kMaskSize);
        }
      }
    };
    auto mask_value = [&](int t, int r, int slot, bool near_end) __attribute__((always_inline)) {
      uint32_t w = kMaskSize == 4 ? mk[t][r % kMaskWords] : mk[t][(r >> 1) % kMaskWords] >> (16 * (r & 1));
      if (near_end) {
        const unsigned char* at = mask_row + (size_t)min(slot, p.max_length - 1) * kMaskSize;
        w = kMaskSize == 4 ? *(const uint32_t*)at : *(const uint16_t*)at;
      }
      return kMaskSize == 4 ? bits2f(w) : half_of<F16>(w, 0);
    };

    pa_f32x4_t o[R::kC];
#pragma unroll
    for (int n = 0; n < R::kC; ++n) o[n] = pa_f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
    float m = -__builtin_inff(), l = 0.0f;

    // A step's keys are read while the step before turns scores into outputs, its values while the step itself computes the
    // scores: each overwrites the registers that were just used, so the loads need none of their own.  Page numbers are read
    // one step further ahead.  Past the end the last step's rows are read again (from the cache), which keeps the count of
    // loads in flight the same on every path.
    int page[2], row[2], page_n[2], row_n[2];
    const int first = lo + wave * R::kSlots;
    auto step = [&](int t0) __attribute__((always_inline)) {
      const bool more = t0 + R::kUnit < hi;
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
        if (R::kPacked) __builtin_amdgcn_sched_barrier(0);
      }
      const bool some_gone = t0 + R::kSlots > hi || page[0] < 0 || page[1] < 0 || kMask;  // perhaps
      uint32_t gone = 0;  // bit 4 t + r: the slot is absent
      if (some_gone) {
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            bool absent = page[t] < 0 || t0 + 16 * t + 4 * g + r >= hi;
            if constexpr (kMask) {
              const float add = mask_value(t, r, t0 + 16 * t + 4 * g + r, t0 + R::kSlots > p.max_length);
              x[t][r] += add;
              absent = absent || add == -__builtin_inff();
            }
            if (absent) {
              x[t][r] = -__builtin_inff();
              gone |= 1u << (4 * t + r);
            }
          }
      }
#pragma unroll
      for (int t = 0; t < 2; ++t) {  // the next step's pages, or the same again
        page[t] = more ? page_n[t] : page[t];
        row[t] = more ? row_n[t] : row[t];
      }
      load_mask(more ? t0 + R::kUnit : t0);
      load_keys(page, row);
#pragma unroll
      for (int t = 0; t < 2; ++t) page_n[t] = tile_page(t0 + 2 * R::kUnit + 16 * t, row_n[t]);
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (EXTRA != kPlain) {
        if ((EXTRA == kScores || p.scores != nullptr) && i < rows) {
          float* sp = p.scores + ((size_t)b * p.heads + head0 + i) * p.score_stride + t0 + 4 * g;
#pragma unroll
          for (int t = 0; t < 2; ++t) *(float4*)(sp + 16 * t) = make_float4(x[t][0], x[t][1], x[t][2], x[t][3]);
        }
      }
      // The reference point m of the exponentials moves only when some head has met a score more than kGrow (in the
      // exponent's unit) above it: probabilities then reach 2^kGrow, and most steps skip the rescaling and the exchange
      // between lanes.
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
      {
        // Probabilities enter the product with the values as two 16-bit numbers, the rounded one and what it left out (about 16
        // bits of bf16, 22 of fp16): rounded once, they alone would be as far off as the rounded result.  The second product
        // costs matrix instructions that the loads leave free.  fp16 ones are held 2^kShift up, where small ones keep their
        // bits (fp16 loses them below 2^-14).
        uint32_t pf[4], pl[4];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          float ex[4];
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            ex[r] = __builtin_amdgcn_exp2f((x[t][r] - ms) * kLog2e + kShift);
            l += ex[r];
          }
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const uint32_t w = kv_pack2<F16>(ex[2 * r], ex[2 * r + 1]);
            pf[2 * t + r] = w;
            pl[2 * t + r] = kv_pack2<F16>(ex[2 * r] - half_of<F16>(w, 0), ex[2 * r + 1] - half_of<F16>(w, 1));
          }
        }
        float vscale[8];
        if constexpr (R::kPacked) {
#pragma unroll
          for (int j = 0; j < 8; ++j) vscale[j] = kv_scale<FMT>((vsc[j >> 2] >> (8 * (j & 3))) & 0xFFu);
        }
        if (some_gone) {  // what an absent slot holds must not meet its probability of zero: it may be infinite or NaN
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if ((gone >> j) & 1u) {
              if constexpr (R::kPacked) vscale[j] = 0.0f;
#pragma unroll
              for (int n = 0; n < R::kValWords; ++n) vr[j][n] = 0;
            }
        }
        // values: two neighbouring elements of the 8 slots at a time, widened, pairs of slots joined
#pragma unroll
        for (int np = 0; np < R::kC / 2; ++np) {
          uint32_t f0[4], f1[4];
          if constexpr (FMT == MASE_KV_MXINT8) {
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              const uint32_t wa = vr[2 * q][np >> 1] >> (16 * (np & 1)), wb = vr[2 * q + 1][np >> 1] >> (16 * (np & 1));
              f0[q] = kv_pack2<F16>((float)(int)(int8_t)wa * vscale[2 * q], (float)(int)(int8_t)wb * vscale[2 * q + 1]);
              f1[q] = kv_pack2<F16>((float)(int)(int8_t)(wa >> 8) * vscale[2 * q], (float)(int)(int8_t)(wb >> 8) * vscale[2 * q + 1]);
            }
          } else {
            uint32_t w[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) w[j] = kv_widen_pair<FMT, F16>(vr[j], np, R::kPacked ? vscale[j] : 0.0f);
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              f0[q] = __builtin_amdgcn_perm(w[2 * q + 1], w[2 * q], 0x05040100u);
              f1[q] = __builtin_amdgcn_perm(w[2 * q + 1], w[2 * q], 0x07060302u);
            }
          }
          o[2 * np] = mfma16<F16>(f0, pf, o[2 * np]);
          o[2 * np + 1] = mfma16<F16>(f1, pf, o[2 * np + 1]);
          o[2 * np] = mfma16<F16>(f0, pl, o[2 * np]);
          o[2 * np + 1] = mfma16<F16>(f1, pl, o[2 * np + 1]);
          if (R::kPacked && (np & 1)) __builtin_amdgcn_sched_barrier(0);
        }
      }
      load_values(page, row);
      __builtin_amdgcn_sched_barrier(0);
    };
    if (first < hi) {
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        page[t] = tile_page(first + 16 * t, row[t]);
        page_n[t] = tile_page(first + R::kUnit + 16 * t, row_n[t]);
      }
      load_mask(first);
      load_keys(page, row);
      __builtin_amdgcn_sched_barrier(0);  // the order of the loop, which its waits count on
      load_values(page, row);
      __builtin_amdgcn_sched_barrier(0);
      for (int t0 = first; t0 < hi; t0 += R::kUnit) step(t0);
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
    const bool all = a == 0 && e == n_units;
    const float down = __builtin_amdgcn_exp2f(-kShift);
    const size_t place = 2 * (size_t)blockIdx.x + (first_piece ? 0 : 1);
    for (int el = threadIdx.x; el < rows * D; el += 256) {
      const int r = el / D, d = el % D;
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
      float* ml = nullptr;
      if (all) {
        const float y = sum == 0.0f ? 0.0f : acc / sum;
        DTypeTraits<F16 ? MASE_DT_F16 : MASE_DT_BF16>::store1(p.out, bh * D + d, y);
        if (EXTRA != kPlain && p.scores != nullptr) ml = p.row_ml + bh * 2;
      } else {
        p.part_o[(place * p.tile_rows + r) * D + d] = acc * down;
        ml = p.part_ml + (place * p.tile_rows + r) * 2;
      }
      if (ml != nullptr && d == 0) {
        ml[0] = top;
        ml[1] = sum * down;
      }
    }
    left -= e - a;
    if (left <= 0) break;
    __syncthreads();  // everyone has read the LDS
    a = 0;
    if (++b >= p.batch) break;  // lengths that change under the kernel must not lead past the last sequence
    length = length_of(b);
    n_units = row_units<R::kUnit>(length);
  }
}

// The pieces of row `rh` of sequence b: how many (1: the row was finished in one piece), and where piece k lies.
struct Pieces {
  int count, row_heads;
  size_t wg0;  // the first piece's work-group; the next ones' are row_heads apart
  bool from_start;
  __device__ __forceinline__ size_t place(int k) const { return 2 * (wg0 + (size_t)k * row_heads) + (k == 0 && !from_start ? 1 : 0); }
};
__device__ __forceinline__ Pieces row_pieces(const DecodeParams& p, int b, int rh, int row_heads) {
  const uint32_t at = p.plan[b], n = p.plan[b + 1] - at, share = p.plan[p.batch + 1], s0 = at / share;
  Pieces q;
  q.row_heads = row_heads;
  q.wg0 = (size_t)s0 * row_heads + rh;
  q.from_start = s0 * share == at;
  q.count = (int)((at + n - 1) / share - s0) + 1;
  return q;
}

// A running softmax: reference point, sum of exponentials, and (joining) their weighted sum.  Later terms are added with one
// rescaling at most; NaN stays.
__device__ __forceinline__ void ml_add(float& top, float& sum, float4& acc, float m, float l, const float4& v) {
  const float t = fmaxf(top, m);
  const float f = top == t ? 1.0f : __builtin_amdgcn_exp2f((top - t) * kLog2e), g = m == t ? 1.0f : __builtin_amdgcn_exp2f((m - t) * kLog2e);
  top = t;
  sum = sum * f + l * g;
  acc.x = acc.x * f + v.x * g;
  acc.y = acc.y * f + v.y * g;
  acc.z = acc.z * f + v.z * g;
  acc.w = acc.w * f + v.w * g;
}

constexpr int kWeightSlots = 1024;  // per work-group

// Joins the pieces of cut rows (blocks x < joins) and, with weights, adds the probabilities to them (the blocks behind).
// grid (x, row, sequence).
//
// Joining: a work-group takes `items` (a power of two from 16 to 256) of the row's rows * D / 4 groups of four outputs,
// 256 / items threads sharing the pieces of each; the host takes as few items as make 256 work-groups of all rows.  The
// pieces' sums are added in a fixed order.
template <int D, bool F16>
__device__ __forceinline__ void join_pieces(const DecodeParams& p, int items, int rh, int b, float* lds) {
  float4* acc_s = (float4*)lds;  // [256], then [256] reference points and [256] sums
  float *top_s = lds + 1024, *sum_s = lds + 1280;
  const int tid = threadIdx.x;
  const Pieces q = row_pieces(p, b, rh, p.c.heads * p.head_tiles);
  if (q.count == 1) return;
  const int hk = rh / p.head_tiles, tile = rh % p.head_tiles;
  const int rows = min(kHeadTile, p.group - tile * kHeadTile);
  const int item = (int)blockIdx.x * items + tid % items, r = item / (D / 4), col = item % (D / 4) * 4;
  const int parts = 256 / items;
  float top = -__builtin_inff(), sum = 0.0f;
  float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  if (r < rows) {
#pragma unroll 4
    for (int k = tid / items; k < q.count; k += parts) {
      const size_t place = q.place(k) * p.tile_rows + r;
      const float2 ml = *(const float2*)(p.part_ml + place * 2);
      ml_add(top, sum, acc, ml.x, ml.y, *(const float4*)(p.part_o + place * D + col));
    }
  }
  acc_s[tid] = acc;
  top_s[tid] = top;
  sum_s[tid] = sum;
  __syncthreads();
  if (tid >= items || r >= rows) return;
  for (int k = 1; k < parts; ++k) ml_add(top, sum, acc, top_s[k * items + tid], sum_s[k * items + tid], acc_s[k * items + tid]);
  const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
  const size_t bh = (size_t)b * p.heads + hk * p.group + tile * kHeadTile + r;
  uint2 y;
  y.x = kv_pack2<F16>(acc.x * inv, acc.y * inv);
  y.y = kv_pack2<F16>(acc.z * inv, acc.w * inv);
  *(uint2*)(p.out + (bh * D + col) * 2) = y;
}

// Weights: the probabilities of kWeightSlots slots, summed over the query heads of a cached head.
__device__ __forceinline__ void add_weights(const DecodeParams& p, int share, int hk, int b, float* lds) {
  float *top_s = lds, *inv_s = lds + kMaxGroup;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const size_t bh0 = (size_t)b * p.heads + (size_t)hk * p.group;
  const int s0 = share * kWeightSlots;
  const int length = kv_length(p.lengths[b], p.max_length, p.c.table_pages, p.c.page_shift);
  if (s0 >= length) return;
  for (int h = wave; h < p.group; h += 4) {
    const Pieces q = row_pieces(p, b, hk * p.head_tiles + h / kHeadTile, p.c.heads * p.head_tiles);
    float top = -__builtin_inff(), sum = 0.0f;
    float4 none = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    const float4 zero = none;
    for (int k = lane; k < q.count; k += 64) {
      const float2 ml = q.count == 1 ? *(const float2*)(p.row_ml + (bh0 + h) * 2)
                                     : *(const float2*)(p.part_ml + (q.place(k) * p.tile_rows + h % kHeadTile) * 2);
      ml_add(top, sum, none, ml.x, ml.y, zero);
    }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) ml_add(top, sum, none, __shfl_xor(top, d, 64), __shfl_xor(sum, d, 64), zero);
    if (lane == 0) {
      top_s[h] = top;
      inv_s[h] = sum == 0.0f ? 0.0f : 1.0f / sum;
    }
  }
  __syncthreads();
  float* wrow = p.weights + (size_t)b * p.w_sb + (size_t)hk * p.w_sh;
  float acc[kWeightSlots / 256];
#pragma unroll
  for (int j = 0; j < kWeightSlots / 256; ++j) acc[j] = 0.0f;
  const int last = length - 1;
  for (int h = 0; h < p.group; ++h) {
    const float* xs = p.scores + (bh0 + h) * p.score_stride;
    const float top = top_s[h], inv = inv_s[h];
#pragma unroll
    for (int j = 0; j < kWeightSlots / 256; ++j) {
      const float x = xs[min(s0 + 256 * j + tid, last)];
      acc[j] += (x == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f((x - top) * kLog2e)) * inv;
    }
  }
#pragma unroll
  for (int j = 0; j < kWeightSlots / 256; ++j) {
    const int s = s0 + 256 * j + tid;
    if (s < length) wrow[s] += acc[j];
  }
}

template <int D, bool F16>
__global__ __launch_bounds__(256) void paged_decode_join_kernel(DecodeParams p, int joins, int items) {
  __shared__ __attribute__((aligned(16))) float lds[1536];
  const int rh = blockIdx.y, b = blockIdx.z;
  if ((int)blockIdx.x < joins) join_pieces<D, F16>(p, items, rh, b, lds);
  else if (rh % p.head_tiles == 0) add_weights(p, (int)blockIdx.x - joins, rh / p.head_tiles, b, lds);
}

// What a call launches and keeps between its two kernels.
struct DecodePlan {
  size_t groups;   // work-groups
  int head_tiles, tile_rows;
  bool join;       // a row may be cut
  size_t score_stride, plan_bytes, part_floats, ml_floats, row_ml_floats, score_floats;
  size_t bytes() const { return plan_bytes + (part_floats + ml_floats + row_ml_floats + score_floats) * sizeof(float); }
};

template <int D, int FMT>
DecodePlan decode_plan(size_t batch, size_t heads, size_t kv_heads, size_t max_length, bool weights) {
  using R = Rows<D, FMT>;
  DecodePlan d{};
  const size_t group = heads / kv_heads;
  d.head_tiles = (int)((group + kHeadTile - 1) / kHeadTile);
  d.tile_rows = (int)(group < kHeadTile ? group : kHeadTile);
  int cus = device_cu_count();
  if (cus <= 0) cus = 256;
  const size_t steps = max_length ? (max_length + R::kUnit - 1) / R::kUnit : 1;
  const size_t row_heads = kv_heads * d.head_tiles, resident = (size_t)cus * R::kPerCu;
  size_t shares = resident / row_heads;
  if (shares < 1) shares = 1;
  if (shares > batch * steps) shares = batch * steps;
  d.groups = shares * row_heads;
  d.join = steps > 1;
  d.score_stride = steps * R::kUnit;
  d.plan_bytes = (batch + 2 + 3) / 4 * 4 * sizeof(uint32_t);
  d.part_floats = d.join ? 2 * d.groups * d.tile_rows * D : 0;
  d.ml_floats = d.join ? 2 * d.groups * d.tile_rows * 2 : 0;
  d.row_ml_floats = weights ? (batch * heads * 2 + 3) / 4 * 4 : 0;
  d.score_floats = weights ? batch * heads * d.score_stride : 0;
  return d;
}

template <int D, int FMT, bool F16, int EXTRA>
int launch_decode(const DecodeParams& p, const DecodePlan& d, hipStream_t st) {
  // as much LDS as lets exactly kPerCu work-groups on a CU: where one more would fit, some CUs take it and others are left
  // with one less, and the launch lasts as long as the fullest CU
  constexpr size_t kLdsCu = 160 * 1024, kOnly = kLdsCu / (Rows<D, FMT>::kPerCu + 1) + 64;
  constexpr size_t kMost = sizeof(float) * (2 * kWaves * kHeadTile + kWaves * kHeadTile * D);
  static_assert(kMost + 256 <= kLdsCu / Rows<D, FMT>::kPerCu && kOnly + 256 <= kLdsCu / Rows<D, FMT>::kPerCu, "kPerCu work-groups fit");
  const size_t need = sizeof(float) * (2 * kWaves * kHeadTile + (size_t)kWaves * d.tile_rows * D), lds = need > kOnly ? need : kOnly;
  static std::atomic<uint64_t> attr_done{0};
  const void* fn = (const void*)paged_decode_kernel<D, FMT, F16, EXTRA>;
  if (!set_dynamic_lds_once(attr_done, fn, (int)(kMost > kOnly ? kMost : kOnly))) return MASE_ERR_LAUNCH;
  hipLaunchKernelGGL((paged_decode_kernel<D, FMT, F16, EXTRA>), dim3((unsigned)d.groups), dim3(256), lds, st, p);
  const size_t rows = (size_t)p.c.heads * d.head_tiles, all = (size_t)d.tile_rows * (D / 4);
  int items = 256;
  while (items > 16 && ((size_t)items / 2 >= all || (size_t)p.batch * rows * ((all + items - 1) / items) < 256)) items /= 2;
  const unsigned joins = d.join ? blocks_for(all, (size_t)items) : 0;
  const unsigned shares = EXTRA != kPlain && p.scores != nullptr ? blocks_for((size_t)p.max_length, kWeightSlots) : 0;
  if (joins + shares > 0)
    hipLaunchKernelGGL((paged_decode_join_kernel<D, F16>), dim3(joins + shares, (unsigned)rows, (unsigned)p.batch), dim3(256), 0, st, p, (int)joins, items);
  return MASE_OK;
}

template <int D, int FMT>
int decode_call(DecodeCall& c) {
  const DecodePlan d = decode_plan<D, FMT>(c.batch, c.heads, c.kv_heads, c.max_length, c.with_weights);
  if (c.need != nullptr) {
    *c.need = d.bytes();
    return MASE_OK;
  }
  if (c.workspace == nullptr || c.workspace_bytes < d.bytes()) return MASE_ERR_WORKSPACE;
  if (!aligned16(c.workspace)) return MASE_ERR_ALIGN;
  // units are counted in 32 bits: all of them, rounded up to whole shares, and a share with a row's on top
  const size_t row = c.max_length / Rows<D, FMT>::kUnit + 1;
  if (row * c.batch > 0x3FFFFFFFu || c.kv_heads * d.head_tiles > 65535u) return MASE_ERR_SHAPE;
  c.p.plan = (uint32_t*)c.workspace;
  float* f = (float*)(c.workspace + d.plan_bytes);
  c.p.part_o = f;
  c.p.part_ml = f + d.part_floats;
  c.p.row_ml = c.p.part_ml + d.ml_floats;
  c.p.scores = c.with_weights ? c.p.row_ml + d.row_ml_floats : nullptr;
  c.p.score_stride = d.score_stride;
  c.p.head_tiles = d.head_tiles;
  c.p.tile_rows = d.tile_rows;
  switch (c.extra * 2 + (c.f16 ? 1 : 0)) {
    case kPlain * 2: return launch_decode<D, FMT, false, kPlain>(c.p, d, c.st);
    case kPlain * 2 + 1: return launch_decode<D, FMT, true, kPlain>(c.p, d, c.st);
    case kScores * 2: return launch_decode<D, FMT, false, kScores>(c.p, d, c.st);
    case kScores * 2 + 1: return launch_decode<D, FMT, true, kScores>(c.p, d, c.st);
    case kMaskOwn * 2: return launch_decode<D, FMT, false, kMaskOwn>(c.p, d, c.st);
    case kMaskOwn * 2 + 1: return launch_decode<D, FMT, true, kMaskOwn>(c.p, d, c.st);
    case kMaskF32 * 2: return launch_decode<D, FMT, false, kMaskF32>(c.p, d, c.st);
    default: return launch_decode<D, FMT, true, kMaskF32>(c.p, d, c.st);
  }
}

// one head dimension's formats
template <int D>
int decode_dim(int format, DecodeCall& c) {
  switch (format) {
    case MASE_KV_16BIT: return decode_call<D, MASE_KV_16BIT>(c);
    case MASE_KV_MXINT8: return decode_call<D, MASE_KV_MXINT8>(c);
    case MASE_KV_MXFP8_E4M3: return decode_call<D, MASE_KV_MXFP8_E4M3>(c);
    case MASE_KV_MXFP8_E5M2: return decode_call<D, MASE_KV_MXFP8_E5M2>(c);
    case MASE_KV_MXFP4: return decode_call<D, MASE_KV_MXFP4>(c);
    default: return MASE_ERR_PARAM;
  }
}

}  // namespace
}  // namespace mase
