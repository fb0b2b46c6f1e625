// Attention over the KV cache in blocks for f16 rows.
#include "paged_attention_few.hpp"
#include "paged_attention_many.hpp"

namespace llaisys::kernels {
template void launchPagedFew<F16>(const PagedAttnArgs &, unsigned, hipStream_t);
template void launchPagedMany<F16>(const PagedAttnArgs &, unsigned, hipStream_t);
} // namespace llaisys::kernels
