// Paged attention kernels for heads of 256 elements.
#include "paged_attention_kernels.hpp"

namespace mase {
int paged_decode_d256(int format, DecodeCall& c) { return decode_dim<256>(format, c); }
}  // namespace mase
