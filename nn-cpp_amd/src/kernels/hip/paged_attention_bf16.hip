// paged_attention_bf16.hip - the kernels of attention over pages of bf16 (paged_attention_fwd.hpp).
#include "paged_attention_fwd.hpp"

namespace nnh {
namespace attn {
template hipError_t paged_of<__bf16>(const PagedAttentionArgs&, bool, hipStream_t);
}
}  // namespace nnh
