// What the entry point of the paged attention and the files that hold its kernels (one per head dimension) share.
#pragma once
#include "paged_kv.hpp"

namespace mase {

constexpr int kMaxGroup = 256;  // query heads of one cached head
// what a step does besides: nothing; scores kept (for weights); a mask of the states' type or fp32 (scores kept if asked for)
enum { kPlain = 0, kScores = 1, kMaskOwn = 2, kMaskF32 = 3 };

struct DecodeParams {
  PagedKv c;
  const unsigned char* q;
  size_t q_sb, q_sh;  // bytes
  const int32_t* lengths;
  const unsigned char* mask;
  size_t mask_sb;  // elements
  unsigned char* out;
  uint32_t* plan;  // [batch + 1] units of the sequences before each, then the units of a share
  float* part_o;    // [2 * work-groups][heads of a tile][D]
  float* part_ml;   // [2 * work-groups][heads of a tile][2]
  float* row_ml;    // [batch * heads][2], with weights
  float* scores;    // [batch * heads][score_stride], NULL without weights
  float* weights;
  size_t w_sb, w_sh;
  size_t score_stride;
  int batch, heads, group, head_tiles, tile_rows, max_length;
  float scaling;
};

// a call's arguments; need != NULL: only say how much workspace it takes
struct DecodeCall {
  DecodeParams p;
  size_t batch, heads, kv_heads, max_length;
  bool f16, with_weights;
  int extra;
  unsigned char* workspace;
  size_t workspace_bytes;
  size_t* need;
  hipStream_t st;
};

int paged_decode_d64(int format, DecodeCall& c);
int paged_decode_d128(int format, DecodeCall& c);
int paged_decode_d256(int format, DecodeCall& c);

}  // namespace mase
