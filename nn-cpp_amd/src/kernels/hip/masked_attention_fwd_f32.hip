// masked_attention_fwd_f32.hip - masked attention's forward kernels over f32 (masked_attention_fwd.hpp).
#include "masked_attention_fwd.hpp"

namespace nnh {
namespace attn {
template hipError_t forward_of<float>(const MaskedAttentionArgs&, bool, bool, hipStream_t);
}
}  // namespace nnh
