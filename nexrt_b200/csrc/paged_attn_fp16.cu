// The fp16 kernels of the attention over a paged cache.
#include "paged_attn.cuh"

namespace nexrt {
template int paged_dispatch<__half>(const PagedAttnArgs&, int, bool, cudaStream_t);
}  // namespace nexrt
