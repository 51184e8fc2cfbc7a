// masked_attention_fwd_bf16.hip - masked attention's forward kernels over bf16 (masked_attention_fwd.hpp).
#include "masked_attention_fwd.hpp"

namespace nnh {
namespace attn {
template hipError_t forward_of<__bf16>(const MaskedAttentionArgs&, bool, bool, hipStream_t);
}
}  // namespace nnh
