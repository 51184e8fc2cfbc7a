// masked_attention_bwd_bf16.hip - masked attention's backward kernels over bf16 (masked_attention_bwd.hpp).
#include "masked_attention_bwd.hpp"

namespace nnh {
namespace attn {
template hipError_t backward_of<__bf16>(const MaskedAttentionArgs&, bool, hipStream_t);
}
}  // namespace nnh
