// Paged attention kernels for heads of 64 elements.
#include "paged_attention_kernels.hpp"

namespace mase {
int paged_decode_d64(int format, DecodeCall& c) { return decode_dim<64>(format, c); }
}  // namespace mase
