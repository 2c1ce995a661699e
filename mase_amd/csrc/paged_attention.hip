// Entry points of the attention of one new token over a paged key-value cache (kernels: paged_attention_kernels.hpp).
#include "paged_attention.hpp"

namespace mase {
namespace {
int decode_dispatch(size_t head_dim, int format, DecodeCall& c) {
  switch (head_dim) {
    case 64: return paged_decode_d64(format, c);
    case 128: return paged_decode_d128(format, c);
    case 256: return paged_decode_d256(format, c);
    default: return MASE_ERR_SHAPE;
  }
}
}  // namespace
}  // namespace mase

extern "C" size_t mase_paged_attention_decode_workspace_bytes(size_t batch, size_t heads, size_t kv_heads, size_t head_dim,
                                                              int format, size_t max_length, int with_weights) {
  using namespace mase;
  if (batch == 0 || batch > 65535 || kv_heads == 0 || heads == 0 || heads % kv_heads != 0 || heads / kv_heads > (size_t)kMaxGroup ||
      max_length > 0x7FFF0000u || (head_dim != 64 && head_dim != 128 && head_dim != 256))
    return 0;
  size_t need = 0;
  DecodeCall c{};
  c.batch = batch;
  c.heads = heads;
  c.kv_heads = kv_heads;
  c.max_length = max_length;
  c.with_weights = with_weights != 0;
  c.need = &need;
  return decode_dispatch(head_dim, format, c) == MASE_OK ? need : 0;
}

extern "C" int mase_paged_attention_decode(const mase_paged_kv* cache, const void* q, size_t q_stride_b, size_t q_stride_h,
                                           size_t heads, const int32_t* lengths, size_t max_length, float scaling,
                                           const void* mask, int mask_dtype, size_t mask_stride_b, float* weights,
                                           size_t w_stride_b, size_t w_stride_h, void* out, void* workspace,
                                           size_t workspace_bytes, void* stream) {
  using namespace mase;
  DecodeCall call{};
  DecodeParams& p = call.p;
  const int rc = paged_kv_params(cache, p.c);
  if (rc != MASE_OK) return rc;
  if (heads == 0 || heads % cache->kv_heads != 0 || heads / cache->kv_heads > (size_t)kMaxGroup) return MASE_ERR_SHAPE;
  if (max_length > 0x7FFF0000u) return MASE_ERR_SHAPE;  // a step looks a little past the last slot
  if (!(scaling > -3.0e38f && scaling < 3.0e38f)) return MASE_ERR_PARAM;
  if (mask != nullptr && mask_dtype != cache->dtype && mask_dtype != MASE_DT_F32) return MASE_ERR_DTYPE;
  if (cache->batch == 0) return MASE_OK;
  if (q == nullptr || lengths == nullptr || out == nullptr) return MASE_ERR_NULL;
  if (!aligned16(q) || !aligned16(out) || q_stride_b % 8 != 0 || q_stride_h % 8 != 0) return MASE_ERR_ALIGN;
  p.q = (const unsigned char*)q;
  p.q_sb = q_stride_b * 2;
  p.q_sh = q_stride_h * 2;
  p.lengths = lengths;
  p.mask = (const unsigned char*)mask;
  p.mask_sb = mask_stride_b;
  p.out = (unsigned char*)out;
  p.weights = weights;
  p.w_sb = w_stride_b;
  p.w_sh = w_stride_h;
  p.batch = (int)cache->batch;
  p.heads = (int)heads;
  p.group = (int)(heads / cache->kv_heads);
  p.max_length = (int)max_length;
  p.scaling = scaling;
  call.batch = cache->batch;
  call.heads = heads;
  call.kv_heads = cache->kv_heads;
  call.max_length = max_length;
  call.f16 = cache->dtype == MASE_DT_F16;
  call.extra = mask != nullptr ? (mask_dtype == MASE_DT_F32 ? kMaskF32 : kMaskOwn) : (weights != nullptr ? kScores : kPlain);
  call.with_weights = weights != nullptr;
  call.workspace = (unsigned char*)workspace;
  call.workspace_bytes = workspace_bytes;
  call.st = (hipStream_t)stream;
  const int lrc = decode_dispatch(cache->head_dim, cache->format, call);
  if (lrc != MASE_OK) return lrc;
  return hipGetLastError() == hipSuccess ? MASE_OK : MASE_ERR_LAUNCH;
}
