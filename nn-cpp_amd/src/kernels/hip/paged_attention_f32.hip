// paged_attention_f32.hip - the kernels of attention over pages of f32 (paged_attention_fwd.hpp).
#include "paged_attention_fwd.hpp"

namespace nnh {
namespace attn {
template hipError_t paged_of<float>(const PagedAttentionArgs&, bool, hipStream_t);
}
}  // namespace nnh
