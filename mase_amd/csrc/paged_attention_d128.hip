// Paged attention kernels for heads of 128 elements.
#include "paged_attention_kernels.hpp"

namespace mase {
int paged_decode_d128(int format, DecodeCall& c) { return decode_dim<128>(format, c); }
}  // namespace mase
