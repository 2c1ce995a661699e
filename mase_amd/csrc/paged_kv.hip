// Paged key-value cache for gfx950: writing new tokens (with MX quantization on the way), reading sequences back dense, and
// eviction by accumulated attention weight.  What the reference's attention modules do through
// kv_cache_mxfp / kv_cache_mxint and past_key_value.update (nn/quantized/functional/kvcache.py:8-43,
// nn/quantized/modules/llama/attention.py:182-187), with the codes themselves held in pages.  All of it is bound by HBM.
#include "paged_kv.hpp"
#include "mxfp_core.hpp"
#include "mxint_core.hpp"

namespace mase {

int paged_kv_params(const mase_paged_kv* c, PagedKv& p) {
  if (c == nullptr || c->k == nullptr || c->v == nullptr || c->page_table == nullptr) return MASE_ERR_NULL;
  if (c->dtype != MASE_DT_BF16 && c->dtype != MASE_DT_F16) return MASE_ERR_DTYPE;
  if (c->format < MASE_KV_16BIT || c->format > MASE_KV_MXFP4) return MASE_ERR_PARAM;
  const bool packed = c->format != MASE_KV_16BIT;
  if (packed && (c->k_scales == nullptr || c->v_scales == nullptr)) return MASE_ERR_NULL;
  if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256) return MASE_ERR_SHAPE;
  const size_t ps = c->page_size;
  if (ps < 16 || ps > 4096 || (ps & (ps - 1)) != 0) return MASE_ERR_SHAPE;
  // slots are counted in 32 bits on the device, grids have at most 65535 sequences and heads
  if (c->num_pages == 0 || c->num_pages > 0x7FFFFFFFu || c->table_pages == 0 || c->table_pages > 0x7FFFFFFFu / ps ||
      c->table_stride < c->table_pages || c->batch > 65535 || c->kv_heads == 0 || c->kv_heads > 65535)
    return MASE_ERR_SHAPE;
  const size_t strides[6] = {c->k_stride_page, c->k_stride_head, c->k_stride_slot,
                             c->v_stride_page, c->v_stride_head, c->v_stride_slot};
  for (size_t s : strides)
    if (s % 16 != 0) return MASE_ERR_ALIGN;
  const size_t row = kv_row_bytes(c->format, c->head_dim);
  // a page's rows of one head lie within 32-bit byte offsets
  if (c->k_stride_slot < row || c->v_stride_slot < row || c->k_stride_slot > 0x7FFFFFFFu / ps ||
      c->v_stride_slot > 0x7FFFFFFFu / ps)
    return MASE_ERR_SHAPE;
  if (!aligned16(c->k) || !aligned16(c->v)) return MASE_ERR_ALIGN;
  if (packed && (((uintptr_t)c->k_scales | (uintptr_t)c->v_scales) & 7u) != 0) return MASE_ERR_ALIGN;
  if (((uintptr_t)c->page_table & 3u) != 0) return MASE_ERR_ALIGN;
  p.k = (unsigned char*)c->k;
  p.v = (unsigned char*)c->v;
  p.ks = c->k_scales;
  p.vs = c->v_scales;
  p.table = c->page_table;
  p.table_stride = c->table_stride;
  p.k_page = c->k_stride_page; p.k_head = c->k_stride_head; p.k_slot = (uint32_t)c->k_stride_slot;
  p.v_page = c->v_stride_page; p.v_head = c->v_stride_head; p.v_slot = (uint32_t)c->v_stride_slot;
  p.num_pages = (int)c->num_pages;
  p.page_shift = __builtin_ctzll((unsigned long long)ps);
  p.table_pages = (int)c->table_pages;
  p.heads = (int)c->kv_heads;
  return MASE_OK;
}

namespace {

// first scale byte of a row of keys, and of a slot's column of values (the other bytes follow at 1 and at page_size)
template <int D>
__device__ __forceinline__ size_t key_scale_at(const PagedKv& p, int page, int head, int row) {
  return ((((size_t)page * p.heads + head) << p.page_shift) + row) * (D / 32);
}
template <int D>
__device__ __forceinline__ size_t value_scale_at(const PagedKv& p, int page, int head, int row) {
  return ((((size_t)page * p.heads + head) * (D / 32)) << p.page_shift) + row;
}

// -------------------------------------------------------------------------------------------------
// append
// -------------------------------------------------------------------------------------------------
struct AppendParams {
  PagedKv c;
  const unsigned char* key;
  const unsigned char* value;
  size_t k_sb, k_sh, k_st, v_sb, v_sh, v_st;  // byte strides
  const int32_t* starts;
  const int32_t* counts;
  int32_t* positions;
  size_t pos_sb, pos_sh;
  const int32_t* first_positions;
  int tokens;
  uint32_t items;  // tokens * heads * D / 8
  MxintParams mxint;
  MxfpParams mxfp;
};

// 8 elements to their codes; the 4 lanes of a block of 32 hold it together.  Every lane of the wavefront takes part (the
// logarithm's table is exchanged between lanes).  Returns the block's scale byte.
template <int FMT, int DT>
__device__ __forceinline__ uint32_t encode8(const uint4& raw, const AppendParams& p, const WaveLog2& meta, uint32_t* w) {
  using TR = DTypeTraits<DT>;
  float x[8];
  TR::unpack(raw, x);
  uint32_t c[8];
  uint32_t scale;
  if constexpr (FMT == MASE_KV_MXINT8) {
    const uint32_t m = group_max_u32<4>(vec_absmax_bits<DT>(raw));
    int k = 0, kc = 0;
    const int state = block_exponent<DT>(m, p.mxint, k, kc, meta);
    // clamp(rint(y)) for the integer bounds is rint(clamp(y)), and adding 1.5 2^23 rounds to the nearest integer, ties to
    // even, and leaves it in the low byte
#pragma unroll
    for (int j = 0; j < 8; ++j) c[j] = f2bits(__builtin_amdgcn_fmed3f(ldexpf(x[j], 7 - k), -128.0f, 127.0f) + 12582912.0f);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const uint32_t lo = __builtin_amdgcn_perm(c[4 * j + 1], c[4 * j], 0x0C0C0400u), hi = __builtin_amdgcn_perm(c[4 * j + 3], c[4 * j + 2], 0x04000C0Cu);
      w[j] = state == 0 ? lo | hi : 0u;
    }
    return state == 0 ? (uint32_t)(kc + 127) : 255u;  // the quantizer's other blocks are NaN throughout
  } else {
    constexpr int E = FMT == MASE_KV_MXFP8_E4M3 ? 4 : (FMT == MASE_KV_MXFP8_E5M2 ? 5 : 2), F = FMT == MASE_KV_MXFP8_E4M3 ? 3 : (FMT == MASE_KV_MXFP8_E5M2 ? 2 : 1);
    const uint32_t m = group_max_u32<4>(vec_flushed_absmax<DT>(raw));
    int sh = 0;
    const int state = mxfp_block_scale(m, p.mxfp, sh, meta);
    float y[8];
    mxfp_elements<(E < 4), 8>(x, state, sh, p.mxfp, c, y);
    uint32_t reserved = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) reserved |= code_is_reserved<E, F>(c[j]) ? 1u : 0u;
    reserved = group_max_u32<4>(reserved);
    int sb = state == 1 ? sh + 127 : (state == 0 ? 0 : 255);
    if (state == 1 && reserved) {  // one scale up with halved codes, as the packing kernels write such blocks
      sb = min(sb + 1, 254);
#pragma unroll
      for (int j = 0; j < 8; ++j) c[j] = halve_code<E, F>(c[j]);
    }
    scale = (uint32_t)sb;
  }
  if constexpr (FMT == MASE_KV_MXFP4) {
    w[0] = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) w[0] |= (c[j] & 0xFu) << (4 * j);
  } else {
    w[0] = c[0] | (c[1] << 8) | (c[2] << 16) | (c[3] << 24);
    w[1] = c[4] | (c[5] << 8) | (c[6] << 16) | (c[7] << 24);
  }
  return scale;
}

// One 16-byte piece (8 elements) of keys and the same of values per lane; consecutive lanes go along the head dimension.
// 16-bit rows: then the heads, then the tokens, the order in which projections leave their outputs (18381 tokens, 8 heads of
// 128: 151 MB in 32.8 us; the other order 33.9).  Codes: then the tokens, then the heads, so that the scale bytes of the
// values, which lie slot by slot, meet in a line (9227 tokens in MXINT8, 57 MB: 15.1 us; the other order 16.4).  Bound by
// HBM for prompts in 16 bits, nearly so in MXINT8, and by the launch for single tokens (64 of them: 3 us).  MXFP writes no more
// bytes than MXINT8 but takes 30 us (e4m3), 28 (e5m2) and 24 (MXFP4) for the same tokens: the elements' arithmetic bounds it.
template <int D, int FMT, int DT>
__global__ __launch_bounds__(256) void kv_append_kernel(AppendParams p) {
  constexpr int kPieces = D / 8;
  const int b = blockIdx.y;
  const int count = p.counts == nullptr ? p.tokens : min(p.counts[b], p.tokens);
  const uint32_t idx = blockIdx.x * 256u + threadIdx.x;
  constexpr bool kTokensFirst = FMT != MASE_KV_16BIT;
  const uint32_t first = (blockIdx.x * 256u) / kPieces;  // of the work-group's rows
  if constexpr (kTokensFirst) {
    const uint32_t token = first % (uint32_t)p.tokens;
    if ((int)token >= count && token + 256u / kPieces <= (uint32_t)p.tokens) return;  // the whole work-group
  } else {
    if ((int)(first / (uint32_t)p.c.heads) >= count) return;
  }
  WaveLog2 meta;
  if constexpr (FMT == MASE_KV_MXINT8) meta.init(p.mxint.tab, 0);
  else if constexpr (FMT != MASE_KV_16BIT) meta.init(p.mxfp.tab, kLog2TabHalf);
  const int piece = (int)(idx % kPieces);
  const uint32_t r = idx / kPieces;
  const uint32_t inner = (uint32_t)(kTokensFirst ? p.tokens : p.c.heads);
  const int in = (int)(r % inner), out = (int)(r / inner);
  const int j = kTokensFirst ? in : out, h = kTokensFirst ? out : in;
  // the states are requested before the page is looked up: neither waits for the other
  uint4 kx = make_uint4(0, 0, 0, 0), vx = kx;
  int slot = -1, page = -1;
  if (idx < p.items && j < count) {
    kx = *(const uint4*)(p.key + (size_t)b * p.k_sb + (size_t)h * p.k_sh + (size_t)j * p.k_st + piece * 16);
    vx = *(const uint4*)(p.value + (size_t)b * p.v_sb + (size_t)h * p.v_sh + (size_t)j * p.v_st + piece * 16);
    slot = kv_new_slot(p.starts[b], count, j, p.c.table_pages, p.c.page_shift);
    page = kv_page(p.c.table + (size_t)b * p.c.table_stride, p.c.table_pages, p.c.page_shift, p.c.num_pages, slot);
  }
  const bool live = page >= 0;
  const int row = slot & ((1 << p.c.page_shift) - 1);
  const size_t ko = (size_t)page * p.c.k_page + (size_t)h * p.c.k_head + (size_t)row * p.c.k_slot;
  const size_t vo = (size_t)page * p.c.v_page + (size_t)h * p.c.v_head + (size_t)row * p.c.v_slot;
  if constexpr (FMT == MASE_KV_16BIT) {
    if (!live) return;
    *(uint4*)(p.c.k + ko + piece * 16) = kx;
    *(uint4*)(p.c.v + vo + piece * 16) = vx;
  } else {
    uint32_t kw[2], vw[2];
    const uint32_t ksb = encode8<FMT, DT>(kx, p, meta, kw), vsb = encode8<FMT, DT>(vx, p, meta, vw);
    if (!live) return;
    if constexpr (FMT == MASE_KV_MXFP4) {
      *(uint32_t*)(p.c.k + ko + piece * 4) = kw[0];
      *(uint32_t*)(p.c.v + vo + piece * 4) = vw[0];
    } else {
      *(uint2*)(p.c.k + ko + piece * 8) = make_uint2(kw[0], kw[1]);
      *(uint2*)(p.c.v + vo + piece * 8) = make_uint2(vw[0], vw[1]);
    }
    if ((piece & 3) == 0) {
      p.c.ks[key_scale_at<D>(p.c, page, h, row) + (piece >> 2)] = (uint8_t)ksb;
      p.c.vs[value_scale_at<D>(p.c, page, h, row) + ((size_t)(piece >> 2) << p.c.page_shift)] = (uint8_t)vsb;
    }
  }
  if (p.positions != nullptr && piece == 0)
    p.positions[(size_t)b * p.pos_sb + (size_t)h * p.pos_sh + slot] =
        (p.first_positions != nullptr ? p.first_positions[b] : p.starts[b]) + j;
}

template <int D, int FMT>
void launch_append(const AppendParams& p, int dtype, size_t batch, hipStream_t st) {
  const dim3 grid(blocks_for(p.items, 256), (unsigned)batch), block(256);
  if (FMT == MASE_KV_16BIT || dtype == MASE_DT_BF16)
    hipLaunchKernelGGL((kv_append_kernel<D, FMT, MASE_DT_BF16>), grid, block, 0, st, p);
  else
    hipLaunchKernelGGL((kv_append_kernel<D, FMT, MASE_DT_F16>), grid, block, 0, st, p);
}

// -------------------------------------------------------------------------------------------------
// gather
// -------------------------------------------------------------------------------------------------
struct GatherParams {
  PagedKv c;
  const int32_t* lengths;
  unsigned char* key;
  unsigned char* value;
  int max_length;
};

// 8 elements of keys and of values per lane: a store instruction writes 1 KB without gaps.  (Lanes of 16 codes, whose two
// stores leave gaps of 16 bytes between lanes, took 62 us where this takes 25: 8 x 8 heads of up to 4096 MXFP8 rows of 128,
// 36 MB read and 134 MB written; ordinary stores instead of streaming ones 30 us.)
template <int D, int FMT, bool F16>
__global__ __launch_bounds__(256) void kv_gather_kernel(GatherParams p) {
  constexpr int kPieces = D / 8;
  constexpr int kBytes = FMT == MASE_KV_16BIT ? 16 : (FMT == MASE_KV_MXFP4 ? 4 : 8);  // in storage
  const int b = blockIdx.z, h = blockIdx.y;
  const int piece = (int)threadIdx.x % kPieces, slot = (int)blockIdx.x * (256 / kPieces) + (int)threadIdx.x / kPieces;
  if (slot >= p.max_length) return;
  const int length = kv_length(p.lengths[b], p.max_length, p.c.table_pages, p.c.page_shift);
  const int page = slot < length ? kv_page(p.c.table + (size_t)b * p.c.table_stride, p.c.table_pages, p.c.page_shift, p.c.num_pages, slot) : -1;
  uint32_t kw[4] = {0, 0, 0, 0}, vw[4] = {0, 0, 0, 0};
  if (page >= 0) {
    const int row = slot & ((1 << p.c.page_shift) - 1);
    uint32_t kc[kBytes / 4], vc[kBytes / 4];
    kv_load<kBytes>(p.c.k + (size_t)page * p.c.k_page + (size_t)h * p.c.k_head + (size_t)row * p.c.k_slot + piece * kBytes, kc);
    kv_load<kBytes>(p.c.v + (size_t)page * p.c.v_page + (size_t)h * p.c.v_head + (size_t)row * p.c.v_slot + piece * kBytes, vc);
    float ks = 0.0f, vs = 0.0f;
    if constexpr (FMT != MASE_KV_16BIT) {
      ks = kv_scale<FMT>(p.c.ks[key_scale_at<D>(p.c, page, h, row) + piece / 4]);
      vs = kv_scale<FMT>(p.c.vs[value_scale_at<D>(p.c, page, h, row) + ((size_t)(piece / 4) << p.c.page_shift)]);
    }
    kv_widen<FMT, F16, 8>(kc, ks, kw);
    kv_widen<FMT, F16, 8>(vc, vs, vw);
  }
  const size_t at = ((((size_t)b * p.c.heads + h) * p.max_length + slot) * D + piece * 8) * 2;
  store_nt((uint4*)(p.key + at), make_uint4(kw[0], kw[1], kw[2], kw[3]));
  store_nt((uint4*)(p.value + at), make_uint4(vw[0], vw[1], vw[2], vw[3]));
}

template <int D, int FMT>
void launch_gather(const GatherParams& p, int dtype, size_t batch, hipStream_t st) {
  constexpr int kPieces = D / 8;
  const dim3 grid(blocks_for((size_t)p.max_length, 256 / kPieces), (unsigned)p.c.heads, (unsigned)batch), block(256);
  if (FMT == MASE_KV_16BIT || dtype == MASE_DT_BF16)
    hipLaunchKernelGGL((kv_gather_kernel<D, FMT, false>), grid, block, 0, st, p);
  else
    hipLaunchKernelGGL((kv_gather_kernel<D, FMT, true>), grid, block, 0, st, p);
}

// -------------------------------------------------------------------------------------------------
// evict
// -------------------------------------------------------------------------------------------------
struct EvictParams {
  PagedKv c;
  const int32_t* lengths;
  const float* weights;
  const int32_t* positions;
  float* weights_out;
  int32_t* positions_out;
  int32_t* lengths_out;
  int32_t* moves;    // [rows] number of moves (workspace)
  int32_t* holes;    // [rows][keep] slots below keep that become free, in order
  int32_t* fillers;  // [rows][keep] entry i: the i-th kept slot, for those at keep or behind
  int max_length, capacity, keep, recent, first;
};


// a number that orders slots: protected ones above every weight, NaN below
__device__ __forceinline__ uint32_t evict_key(float w, int pos, int newest, const EvictParams& p) {
  if (pos < p.first || (long long)pos > (long long)newest - p.recent) return 0xFFFFFFFFu;
  if (w != w) return 0u;
  const uint32_t u = f2bits(w + 0.0f);  // -0 equals +0
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

__device__ __forceinline__ int lanes_below(uint64_t mask) {
  return (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0u));
}

// sum of a value over this lane and those below it (quad and row shifts, then the last lanes of the rows before)
__device__ __forceinline__ int scan64(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false);  // row_shr:1
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);  // row_bcast:15 into rows 1 and 3
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);  // row_bcast:31 into rows 2 and 3
  return v;
}

// sum of the first `wave` of a work-group's per-wavefront numbers
template <int WAVES>
__device__ __forceinline__ int sum_before(const int* sums, int wave) {
  int s = 0;
#pragma unroll
  for (int i = 0; i < WAVES - 1; ++i) s += i < wave ? sums[i] : 0;
  return s;
}

// Histogram of 256 bins in kCopies interleaved copies: the lanes of a wavefront that meet in a bin (tokens never attended
// to, weights of one binade) are spread over as many addresses in as many banks.
constexpr int kCopies = 8;

// The bin, from the top, that the `want`-th largest key falls into (found[0]), and how many keys lie in bins above it
// (found[1]); the histogram is zero afterwards.  All threads (at least 256) call it.
__device__ __forceinline__ void find_bin(uint32_t* hist, int want, int* sums, int* found, int tid, int lane, int wave) {
  int mine = 0, run = 0;
  const int bin = 255 - tid;
  if (wave < 4) {
    uint4* c = (uint4*)(hist + bin * kCopies);
    const uint4 u = c[0], v = c[1];
    c[0] = c[1] = make_uint4(0, 0, 0, 0);
    mine = (int)(u.x + u.y + u.z + u.w + v.x + v.y + v.z + v.w);
    run = scan64(mine);
    if (lane == 63) sums[wave] = run;
  }
  __syncthreads();
  if (wave < 4) {
    const int before = run - mine + sum_before<4>(sums, wave);
    if (before < want && want <= before + mine) {  // one thread
      found[0] = bin;
      found[1] = before;
    }
  }
  __syncthreads();
}

// One work-group per (sequence, cached head); a wavefront owns a contiguous run of slots, 64 at a time, so that ranks in
// slot order come from counts per wavefront and ballots within it.  The key of the keep-th largest slot is found by four
// histograms over 8 bits of the keys each.  HELD: the row's keys stay in LDS (rows of up to kHeldSlots); otherwise
// they are made anew from L2 for each pass.
// It is bound by the latency of its dependent steps on one CU (two reads of the row, four histograms, the ranks): 39 us for
// 64 rows of 20001 .. 32768 slots (30 MB, 6 us at the rate of a copy), 11 us for 8 rows of 2047.  Weights and positions are read in runs of independent loads
// (one at a time, each waiting for L2: 103 us); keys in registers with every turn unrolled were no faster (45 us: the code
// itself came from memory).
constexpr int kHeldSlots = 36864;

template <int WAVES, bool HELD>
__global__ __launch_bounds__(64 * WAVES) void kv_evict_select_kernel(EvictParams p) {
  constexpr int kThreads = 64 * WAVES, kRun = 8, kFirstRun = 16;  // turns whose loads are in flight together
  extern __shared__ uint32_t held[];              // HELD: [turns * kThreads] keys by slot
  __shared__ __attribute__((aligned(16))) uint32_t hist[256 * kCopies];
  __shared__ int sums[WAVES], sums2[WAVES], found[2];
  const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const size_t rowi = (size_t)b * p.c.heads + h;
  const float* w = p.weights + rowi * p.capacity;
  const int32_t* pos = p.positions + rowi * p.capacity;
  float* wo = p.weights_out + rowi * p.capacity;
  int32_t* po = p.positions_out + rowi * p.capacity;
  const int n = kv_length(p.lengths[b], min(p.max_length, p.capacity), p.c.table_pages, p.c.page_shift);
  if (h == 0 && tid == 0) p.lengths_out[b] = min(n, p.keep);
  if (n <= p.keep) {
    for (int s = tid; s < p.capacity; s += kThreads) {
      wo[s] = s < n ? w[s] : 0.0f;
      po[s] = s < n ? pos[s] : -1;
    }
    if (tid == 0) p.moves[rowi] = 0;
    return;
  }
  const int turns = (n + kThreads - 1) / kThreads;    // of 64 slots, for each wavefront
  const int s_lo = wave * turns * 64 + lane;          // this lane's first slot, the next ones 64 apart
  auto there = [&](int k) __attribute__((always_inline)) { return k < turns && s_lo + 64 * k < n; };

  // The largest position; HELD: keys but for the recent slots' protection, which needs it.  Slots behind the last one of the
  // row have the smallest key, 0: they lie behind every slot that may have it too (NaN), and keep <= n slots come before.
  int newest = -0x7FFFFFFF - 1;
  for (int k = 0; k < turns; k += kFirstRun) {
    int pv[kFirstRun];
    float wv[kFirstRun];
#pragma unroll
    for (int j = 0; j < kFirstRun; ++j) {
      const int s = min(s_lo + 64 * (k + j), n - 1);
      pv[j] = pos[s];
      wv[j] = HELD ? w[s] : 0.0f;
    }
#pragma unroll
    for (int j = 0; j < kFirstRun; ++j) {
      newest = max(newest, pv[j]);
      if (HELD && k + j < turns) held[s_lo + 64 * (k + j)] = there(k + j) ? evict_key(wv[j], pv[j], 0x7FFFFFFF, p) : 0u;
    }
  }
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) newest = max(newest, __shfl_xor(newest, d, 64));
  if (lane == 0) sums[wave] = newest;
  for (int i = tid; i < 256 * kCopies; i += kThreads) hist[i] = 0;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < WAVES; ++i) newest = max(newest, sums[i]);
  if (HELD && p.recent > 0) {
    for (int k = 0; k < turns; k += kRun) {
      int pv[kRun];
#pragma unroll
      for (int j = 0; j < kRun; ++j) pv[j] = pos[min(s_lo + 64 * (k + j), n - 1)];
#pragma unroll
      for (int j = 0; j < kRun; ++j)
        if (there(k + j) && (long long)pv[j] > (long long)newest - p.recent) held[s_lo + 64 * (k + j)] = 0xFFFFFFFFu;
    }
  }
  // calls f(key) for each of this wavefront's turns of 64 slots
  auto for_keys = [&](auto f) __attribute__((always_inline)) {
    if constexpr (HELD) {
      for (int k = 0; k < turns; k += kRun) {
        uint32_t key[kRun];
#pragma unroll
        for (int j = 0; j < kRun; ++j) key[j] = held[s_lo + 64 * min(k + j, turns - 1)];
#pragma unroll
        for (int j = 0; j < kRun; ++j)
          if (k + j < turns) f(key[j]);
      }
    } else {
      for (int k = 0; k < turns; k += kRun) {
        float wv[kRun];
        int pv[kRun];
#pragma unroll
        for (int j = 0; j < kRun; ++j) {
          const int s = min(s_lo + 64 * (k + j), n - 1);
          wv[j] = w[s];
          pv[j] = pos[s];
        }
#pragma unroll
        for (int j = 0; j < kRun; ++j)
          if (k + j < turns) f(there(k + j) ? evict_key(wv[j], pv[j], newest, p) : 0u);
      }
    }
  };
  uint32_t cut = 0, cut_mask = 0;  // the keep-th largest key, as far as it is known
  int want = p.keep;               // how many of the slots with that key are kept: the first ones
#pragma unroll 1
  for (int shift = 24; shift >= 0; shift -= 8) {
    for_keys([&](uint32_t key) __attribute__((always_inline)) {
      if ((key & cut_mask) == cut) atomicAdd(&hist[((key >> shift) & 255u) * kCopies + (lane & (kCopies - 1))], 1u);
    });
    __syncthreads();
    find_bin(hist, want, sums, found, tid, lane, wave);
    want -= found[1];
    cut |= (uint32_t)found[0] << shift;
    cut_mask |= 255u << shift;
  }
  int gt = 0, eq = 0;  // slots above and at the cut: the lane's, the wavefront's, then those before the slot in hand
  for_keys([&](uint32_t key) __attribute__((always_inline)) {
    gt += key > cut ? 1 : 0;
    eq += key == cut ? 1 : 0;
  });
  gt = __builtin_amdgcn_readlane(scan64(gt), 63);
  eq = __builtin_amdgcn_readlane(scan64(eq), 63);
  if (lane == 0) {
    sums[wave] = gt;
    sums2[wave] = eq;
  }
  __syncthreads();
  gt = sum_before<WAVES>(sums, wave);
  eq = sum_before<WAVES>(sums2, wave);
  int32_t* holes = p.holes + rowi * p.keep;
  int32_t* fillers = p.fillers + rowi * p.keep;
#pragma unroll 1
  for (int k = 0; k < turns; k += kRun) {
    float wv[kRun];
    int pv[kRun];
    uint32_t kv[kRun];
#pragma unroll
    for (int j = 0; j < kRun; ++j) {
      const int s = min(s_lo + 64 * (k + j), n - 1);
      wv[j] = w[s];
      pv[j] = pos[s];
      if (HELD) kv[j] = held[s_lo + 64 * min(k + j, turns - 1)];
    }
#pragma unroll
    for (int j = 0; j < kRun; ++j) {
      const int s = s_lo + 64 * (k + j);
      const bool in = there(k + j);
      const uint32_t key = HELD ? kv[j] : evict_key(wv[j], pv[j], newest, p);
      const bool above = in && key > cut, at = in && key == cut;
      const uint64_t gm = __builtin_amdgcn_ballot_w64(above), em = __builtin_amdgcn_ballot_w64(at);
      const int eq_before = eq + lanes_below(em);
      const int kept_before = gt + lanes_below(gm) + min(eq_before, want);
      const bool kept = above || (at && eq_before < want);
      if (in) {
        if (s < p.keep) {
          if (kept) {
            wo[s] = wv[j];
            po[s] = pv[j];
          } else {
            holes[s - kept_before] = s;
          }
        } else if (kept) {
          fillers[kept_before] = s;  // kept_before < keep: exactly keep slots are kept
        }
        if (s == p.keep) p.moves[rowi] = p.keep - kept_before;
      }
      gt += __popcll(gm);
      eq += __popcll(em);
    }
  }
  for (int s = p.keep + tid; s < p.capacity; s += kThreads) {
    wo[s] = 0.0f;
    po[s] = -1;
  }
}

template <int WAVES, bool HELD>
int launch_evict_select(const EvictParams& p, size_t batch, size_t most, hipStream_t st) {
  // keys by slot, in whole turns of the work-group
  const size_t lds = HELD ? (most + 64 * WAVES - 1) / (64 * WAVES) * (64 * WAVES) * sizeof(uint32_t) : 0;
  if (HELD && WAVES == 16) {
    static std::atomic<uint64_t> attr_done{0};
    if (!set_dynamic_lds_once(attr_done, (const void*)kv_evict_select_kernel<WAVES, HELD>, kHeldSlots * (int)sizeof(uint32_t))) return MASE_ERR_LAUNCH;
  }
  hipLaunchKernelGGL((kv_evict_select_kernel<WAVES, HELD>), dim3((unsigned)p.c.heads, (unsigned)batch), dim3(64 * WAVES), lds, st, p);
  return MASE_OK;
}

// Moves kept rows from behind `keep` into the free slots: sources and targets are disjoint, so the order does not matter, and
// only rows that change place are touched.  16 bytes of keys and of values per lane.  8 x 8 heads of 20001 .. 32768 MXINT8
// rows of 128 cut to 16384: 380 thousand rows of 264 bytes read and written, 0.20 GB in 50 us, 4.0 TB/s where a large copy
// moves 4.9: single rows here and there, and the values' scale bytes one by one.
template <int D, int FMT>
__global__ __launch_bounds__(256) void kv_evict_move_kernel(EvictParams p) {
  constexpr int kRow = FMT == MASE_KV_16BIT ? 2 * D : (FMT == MASE_KV_MXFP4 ? D / 2 : D);
  constexpr int kLanes = kRow / 16, kMoves = 256 / kLanes;
  const int h = blockIdx.y, b = blockIdx.z;
  const size_t rowi = (size_t)b * p.c.heads + h;
  const int moves = p.moves[rowi];
  const int part = threadIdx.x % kLanes;
  const int32_t* table = p.c.table + (size_t)b * p.c.table_stride;
  const int mask = (1 << p.c.page_shift) - 1;
  for (int m = blockIdx.x * kMoves + (int)threadIdx.x / kLanes; m < moves; m += (int)gridDim.x * kMoves) {
    const int to = p.holes[rowi * p.keep + m], from = p.fillers[rowi * p.keep + (p.keep - moves) + m];
    if (part == 0) {
      p.weights_out[rowi * p.capacity + to] = p.weights[rowi * p.capacity + from];
      p.positions_out[rowi * p.capacity + to] = p.positions[rowi * p.capacity + from];
    }
    const int pf = kv_page(table, p.c.table_pages, p.c.page_shift, p.c.num_pages, from);
    const int pt = kv_page(table, p.c.table_pages, p.c.page_shift, p.c.num_pages, to);
    if (pf < 0 || pt < 0) continue;
    const int rf = from & mask, rt = to & mask;
    const size_t hk = (size_t)h * p.c.k_head + part * 16, hv = (size_t)h * p.c.v_head + part * 16;
    const uint4 kx = *(const uint4*)(p.c.k + (size_t)pf * p.c.k_page + (size_t)rf * p.c.k_slot + hk);
    const uint4 vx = *(const uint4*)(p.c.v + (size_t)pf * p.c.v_page + (size_t)rf * p.c.v_slot + hv);
    *(uint4*)(p.c.k + (size_t)pt * p.c.k_page + (size_t)rt * p.c.k_slot + hk) = kx;
    *(uint4*)(p.c.v + (size_t)pt * p.c.v_page + (size_t)rt * p.c.v_slot + hv) = vx;
    if constexpr (FMT != MASE_KV_16BIT) {
      if (part < D / 32) {
        p.c.ks[key_scale_at<D>(p.c, pt, h, rt) + part] = p.c.ks[key_scale_at<D>(p.c, pf, h, rf) + part];
        const size_t col = (size_t)part << p.c.page_shift;
        p.c.vs[value_scale_at<D>(p.c, pt, h, rt) + col] = p.c.vs[value_scale_at<D>(p.c, pf, h, rf) + col];
      }
    }
  }
}

template <int D, int FMT>
void launch_evict_move(const EvictParams& p, size_t batch, hipStream_t st) {
  constexpr int kLanes = (FMT == MASE_KV_16BIT ? 2 * D : (FMT == MASE_KV_MXFP4 ? D / 2 : D)) / 16;
  const int most = min(p.keep, p.max_length - p.keep);  // of moves in a row
  const dim3 grid(blocks_for((size_t)most, 256 / kLanes), (unsigned)p.c.heads, (unsigned)batch);
  hipLaunchKernelGGL((kv_evict_move_kernel<D, FMT>), grid, dim3(256), 0, st, p);
}

// calls fn<D, FMT>(args...) for the pool's head dimension and format
#define MASE_KV_DISPATCH(cache, fn, ...)                                               \
  do {                                                                                 \
    switch ((int)(cache)->head_dim * 8 + (cache)->format) {                            \
      MASE_KV_CASES(64, fn, __VA_ARGS__)                                               \
      MASE_KV_CASES(128, fn, __VA_ARGS__)                                              \
      MASE_KV_CASES(256, fn, __VA_ARGS__)                                              \
      default: return MASE_ERR_SHAPE;                                                  \
    }                                                                                  \
  } while (0)
#define MASE_KV_CASES(D, fn, ...)                                                      \
  case D * 8 + MASE_KV_16BIT: fn<D, MASE_KV_16BIT>(__VA_ARGS__); break;                \
  case D * 8 + MASE_KV_MXINT8: fn<D, MASE_KV_MXINT8>(__VA_ARGS__); break;              \
  case D * 8 + MASE_KV_MXFP8_E4M3: fn<D, MASE_KV_MXFP8_E4M3>(__VA_ARGS__); break;      \
  case D * 8 + MASE_KV_MXFP8_E5M2: fn<D, MASE_KV_MXFP8_E5M2>(__VA_ARGS__); break;      \
  case D * 8 + MASE_KV_MXFP4: fn<D, MASE_KV_MXFP4>(__VA_ARGS__); break;

MxfpParams mxfp_params(int format, const uint32_t* tab) {
  MxfpParams q{};
  q.m.E = format == MASE_KV_MXFP8_E4M3 ? 4 : (format == MASE_KV_MXFP8_E5M2 ? 5 : 2);
  q.m.F = format == MASE_KV_MXFP8_E4M3 ? 3 : (format == MASE_KV_MXFP8_E5M2 ? 2 : 1);
  q.m.bias = (1 << (q.m.E - 1)) - 1;
  q.m.e_hi = (1 << q.m.E) - 1;
  q.m.frac_hi = (1 << q.m.F) - 1;
  q.m.is_finite = 1;
  q.m.round_mode = 0;
  q.el_emax = q.m.e_hi - q.m.bias;
  q.tab = tab;
  return q;
}

}  // namespace
}  // namespace mase

extern "C" int mase_paged_kv_append(const mase_paged_kv* cache, const void* key, const void* value, size_t tokens,
                                    size_t key_stride_b, size_t key_stride_h, size_t key_stride_t, size_t value_stride_b,
                                    size_t value_stride_h, size_t value_stride_t, const int32_t* starts,
                                    const int32_t* counts, int32_t* positions, size_t pos_stride_b, size_t pos_stride_h,
                                    const int32_t* first_positions, const uint32_t* log2_tab, void* stream) {
  using namespace mase;
  AppendParams p{};
  const int rc = paged_kv_params(cache, p.c);
  if (rc != MASE_OK) return rc;
  if (cache->batch == 0 || tokens == 0) return MASE_OK;
  if (key == nullptr || value == nullptr || starts == nullptr) return MASE_ERR_NULL;
  if (cache->format != MASE_KV_16BIT && log2_tab == nullptr) return MASE_ERR_NULL;
  if (!aligned16(key) || !aligned16(value)) return MASE_ERR_ALIGN;
  const size_t strides[6] = {key_stride_b, key_stride_h, key_stride_t, value_stride_b, value_stride_h, value_stride_t};
  for (size_t s : strides)
    if (s % 8 != 0) return MASE_ERR_ALIGN;
  if (tokens > 0x7FFFFF00u / (cache->kv_heads * (cache->head_dim / 8))) return MASE_ERR_SHAPE;
  p.key = (const unsigned char*)key;
  p.value = (const unsigned char*)value;
  p.k_sb = key_stride_b * 2; p.k_sh = key_stride_h * 2; p.k_st = key_stride_t * 2;
  p.v_sb = value_stride_b * 2; p.v_sh = value_stride_h * 2; p.v_st = value_stride_t * 2;
  p.starts = starts;
  p.counts = counts;
  p.positions = positions;
  p.pos_sb = pos_stride_b;
  p.pos_sh = pos_stride_h;
  p.first_positions = first_positions;
  p.tokens = (int)tokens;
  p.items = (uint32_t)(tokens * cache->kv_heads * (cache->head_dim / 8));
  if (cache->format == MASE_KV_MXINT8) {
    p.mxint.qshift = 7;
    p.mxint.bias = 127;
    p.mxint.scale_max = 255;
    p.mxint.lo = -128.0f;
    p.mxint.hi = 127.0f;
    p.mxint.tab = log2_tab;
  } else if (cache->format != MASE_KV_16BIT) {
    p.mxfp = mxfp_params(cache->format, log2_tab);
  }
  MASE_KV_DISPATCH(cache, launch_append, p, cache->dtype, cache->batch, (hipStream_t)stream);
  return hipGetLastError() == hipSuccess ? MASE_OK : MASE_ERR_LAUNCH;
}

extern "C" int mase_paged_kv_gather(const mase_paged_kv* cache, const int32_t* lengths, size_t max_length, void* key,
                                    void* value, void* stream) {
  using namespace mase;
  GatherParams p{};
  const int rc = paged_kv_params(cache, p.c);
  if (rc != MASE_OK) return rc;
  if (cache->batch == 0 || max_length == 0) return MASE_OK;
  if (lengths == nullptr || key == nullptr || value == nullptr) return MASE_ERR_NULL;
  if (!aligned16(key) || !aligned16(value)) return MASE_ERR_ALIGN;
  if (max_length > 0x7FFFFF00u / (cache->head_dim / 8)) return MASE_ERR_SHAPE;
  p.lengths = lengths;
  p.key = (unsigned char*)key;
  p.value = (unsigned char*)value;
  p.max_length = (int)max_length;
  MASE_KV_DISPATCH(cache, launch_gather, p, cache->dtype, cache->batch, (hipStream_t)stream);
  return hipGetLastError() == hipSuccess ? MASE_OK : MASE_ERR_LAUNCH;
}

extern "C" size_t mase_paged_kv_evict_workspace_bytes(size_t batch, size_t kv_heads, size_t keep) {
  const size_t rows = batch * kv_heads;
  return ((rows + 3) / 4 * 4 + 2 * rows * keep) * sizeof(int32_t);
}

extern "C" int mase_paged_kv_evict(const mase_paged_kv* cache, const int32_t* lengths, size_t max_length,
                                   const float* weights, const int32_t* positions, size_t capacity, size_t keep,
                                   size_t recent, size_t first, float* weights_out, int32_t* positions_out,
                                   int32_t* lengths_out, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace mase;
  EvictParams p{};
  const int rc = paged_kv_params(cache, p.c);
  if (rc != MASE_OK) return rc;
  if (keep == 0 || recent > keep || first > keep - recent) return MASE_ERR_PARAM;
  if (cache->batch == 0) return MASE_OK;
  if (lengths == nullptr || weights == nullptr || positions == nullptr || weights_out == nullptr ||
      positions_out == nullptr || lengths_out == nullptr)
    return MASE_ERR_NULL;
  if (weights == weights_out || positions == positions_out) return MASE_ERR_PARAM;
  if (max_length > 0x7FFFFFFFu - 1024u || capacity == 0 || capacity > 0x7FFFFFFFu - 1024u || keep > 0x7FFFFFFFu) return MASE_ERR_SHAPE;
  const size_t rows = cache->batch * cache->kv_heads;
  if (workspace == nullptr || workspace_bytes < mase_paged_kv_evict_workspace_bytes(cache->batch, cache->kv_heads, keep))
    return MASE_ERR_WORKSPACE;
  if (!aligned16(workspace)) return MASE_ERR_ALIGN;
  p.lengths = lengths;
  p.weights = weights;
  p.positions = positions;
  p.weights_out = weights_out;
  p.positions_out = positions_out;
  p.lengths_out = lengths_out;
  p.moves = (int32_t*)workspace;
  p.holes = p.moves + (rows + 3) / 4 * 4;
  p.fillers = p.holes + rows * keep;
  p.max_length = (int)max_length;
  p.capacity = (int)capacity;
  p.keep = (int)keep;
  p.recent = (int)recent;
  p.first = (int)first;
  hipStream_t st = (hipStream_t)stream;
  const size_t most = max_length < capacity ? max_length : capacity;  // slots of a row
  // Short rows: four wavefronts, whose barriers are shorter; longer ones: sixteen, which have fewer turns.  Rows of 1024, 2048,
  // 4096 and 8192 slots, 8 rows cut to half: 10.2, 11.3, 15.8 and 26.6 us with four, 12.3, 12.6, 13.3 and 14.9 with sixteen
  // (64 rows alike).
  const int src = most <= 2048 ? launch_evict_select<4, true>(p, cache->batch, most, st)
                  : most <= (size_t)kHeldSlots ? launch_evict_select<16, true>(p, cache->batch, most, st)
                                               : launch_evict_select<16, false>(p, cache->batch, most, st);
  if (src != MASE_OK) return src;
  if (max_length > keep && capacity > keep) MASE_KV_DISPATCH(cache, launch_evict_move, p, cache->batch, st);
  return hipGetLastError() == hipSuccess ? MASE_OK : MASE_ERR_LAUNCH;
}
