// Shared by the kernels of the paged key-value cache: the pool's parameters on the device and the widening of its codes.
#pragma once
#include "common.hpp"
#include "paged_kv_index.hpp"

namespace mase {

struct PagedKv {
  unsigned char* k;
  unsigned char* v;
  uint8_t* ks;  // [pages][heads][slots][D / 32]
  uint8_t* vs;  // [pages][heads][D / 32][slots]
  const int32_t* table;
  size_t table_stride;                     // entries between the rows of two sequences
  size_t k_page, k_head, v_page, v_head;   // byte strides
  uint32_t k_slot, v_slot;
  int num_pages, page_shift, table_pages, heads;
};

// checks what the host can see of a pool and fills the kernels' form of it; MASE_OK or an error code
int paged_kv_params(const mase_paged_kv* c, PagedKv& p);

// bytes of one row's elements (keys or values of one token and head)
static inline size_t kv_row_bytes(int format, size_t head_dim) {
  return format == MASE_KV_16BIT ? 2 * head_dim : (format == MASE_KV_MXFP4 ? head_dim / 2 : head_dim);
}

#if defined(__HIPCC__)
typedef __bf16 kv_bf16x2_t __attribute__((ext_vector_type(2)));
typedef _Float16 kv_f16x2_t __attribute__((ext_vector_type(2)));

// The shared scale of a block as the widening below takes it.  Byte 255 is NaN in every format (a block with an element
// that the format cannot hold).  MXINT8: code * 2^(byte - 134) is one multiplication by this power of two (subnormal for
// bytes below 8).  MXFP: the conversion instructions take the power of two itself, 2^(byte - 127), as an fp32 number of
// which they read the exponent field.
template <int FMT>
__device__ __forceinline__ float kv_scale(uint32_t byte) {
  if constexpr (FMT == MASE_KV_MXINT8) return byte == 255u ? qnan() : ldexpf(1.0f, (int)byte - 134);
  return bits2f(byte << 23);
}

// two values as a dword of two 16-bit numbers.  Every code times its scale is exact in bf16 (at most 8 significant bits),
// and in fp16 as long as it stays in that type's range.
template <bool F16>
__device__ __forceinline__ uint32_t kv_pack2(float a, float b) {
  if constexpr (F16) return f32_to_f16_bits(a) | (f32_to_f16_bits(b) << 16);
  return f32x2_to_bf16x2_bits(a, b);
}

// elements 2 q and 2 q + 1 of a dword of codes (8-bit formats: q = 0, 1; 4-bit: q = 0 .. 3) as a dword of two 16-bit numbers
template <int FMT, bool F16, int Q>
__device__ __forceinline__ uint32_t kv_widen2(uint32_t w, float scale) {
  if constexpr (FMT == MASE_KV_MXINT8) {
    const float a = (float)(int)(int8_t)(w >> (16 * Q)), b = (float)(int)(int8_t)(w >> (16 * Q + 8));
    return kv_pack2<F16>(a * scale, b * scale);
  } else if constexpr (FMT == MASE_KV_MXFP8_E4M3) {
    if constexpr (F16) return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, scale, Q != 0));
    else return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, Q != 0));
  } else if constexpr (FMT == MASE_KV_MXFP8_E5M2) {
    if constexpr (F16) return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_bf8(w, scale, Q != 0));
    else return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(w, scale, Q != 0));
  } else {
    static_assert(FMT == MASE_KV_MXFP4, "codes");
    if constexpr (F16) return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, Q));
    else return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, Q));
  }
}

// N elements (N even; one block) from their storage words to N / 2 dwords of two 16-bit numbers
template <int FMT, bool F16, int N>
__device__ __forceinline__ void kv_widen(const uint32_t* w, float scale, uint32_t* out) {
  if constexpr (FMT == MASE_KV_16BIT) {
#pragma unroll
    for (int j = 0; j < N / 2; ++j) out[j] = w[j];
  } else if constexpr (FMT == MASE_KV_MXFP4) {
#pragma unroll
    for (int j = 0; j < N; j += 8) {
      out[j / 2] = kv_widen2<FMT, F16, 0>(w[j / 8], scale);
      out[j / 2 + 1] = kv_widen2<FMT, F16, 1>(w[j / 8], scale);
      if constexpr (N >= 8) {
        out[j / 2 + 2] = kv_widen2<FMT, F16, 2>(w[j / 8], scale);
        out[j / 2 + 3] = kv_widen2<FMT, F16, 3>(w[j / 8], scale);
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < N; j += 4) {
      out[j / 2] = kv_widen2<FMT, F16, 0>(w[j / 4], scale);
      out[j / 2 + 1] = kv_widen2<FMT, F16, 1>(w[j / 4], scale);
    }
  }
}

// elements 2 np and 2 np + 1 of a run in its storage words
template <int FMT, bool F16>
__device__ __forceinline__ uint32_t kv_widen_pair(const uint32_t* w, int np, float scale) {
  if constexpr (FMT == MASE_KV_16BIT) {
    return w[np];
  } else if constexpr (FMT == MASE_KV_MXFP4) {
    switch (np & 3) {
      case 0: return kv_widen2<FMT, F16, 0>(w[np >> 2], scale);
      case 1: return kv_widen2<FMT, F16, 1>(w[np >> 2], scale);
      case 2: return kv_widen2<FMT, F16, 2>(w[np >> 2], scale);
      default: return kv_widen2<FMT, F16, 3>(w[np >> 2], scale);
    }
  } else {
    return (np & 1) ? kv_widen2<FMT, F16, 1>(w[np >> 1], scale) : kv_widen2<FMT, F16, 0>(w[np >> 1], scale);
  }
}

// BYTES (2 .. 32) from memory to words; a 2-byte piece fills the low half of one word
template <int BYTES>
__device__ __forceinline__ void kv_load(const unsigned char* p, uint32_t* w) {
  if constexpr (BYTES == 2) {
    w[0] = *(const uint16_t*)p;
  } else if constexpr (BYTES == 4) {
    w[0] = *(const uint32_t*)p;
  } else if constexpr (BYTES == 8) {
    const uint2 t = *(const uint2*)p;
    w[0] = t.x; w[1] = t.y;
  } else {
#pragma unroll
    for (int j = 0; j < BYTES / 16; ++j) {
      const uint4 t = ((const uint4*)p)[j];
      w[4 * j] = t.x; w[4 * j + 1] = t.y; w[4 * j + 2] = t.z; w[4 * j + 3] = t.w;
    }
  }
}
#endif

}  // namespace mase
