// Attention over the KV cache in blocks for f32 rows.
#include "paged_attention_few.hpp"
#include "paged_attention_many.hpp"

namespace llaisys::kernels {
template void launchPagedFew<F32>(const PagedAttnArgs &, unsigned, hipStream_t);
template void launchPagedMany<F32>(const PagedAttnArgs &, unsigned, hipStream_t);
} // namespace llaisys::kernels
