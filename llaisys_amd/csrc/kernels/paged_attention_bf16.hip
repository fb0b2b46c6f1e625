// Attention over the KV cache in blocks for bf16 rows.
#include "paged_attention_few.hpp"
#include "paged_attention_many.hpp"

namespace llaisys::kernels {
template void launchPagedFew<BF16>(const PagedAttnArgs &, unsigned, hipStream_t);
template void launchPagedMany<BF16>(const PagedAttnArgs &, unsigned, hipStream_t);
} // namespace llaisys::kernels
