// masked_attention_bwd_f32.hip - masked attention's backward kernels over f32 (masked_attention_bwd.hpp).
#include "masked_attention_bwd.hpp"

namespace nnh {
namespace attn {
template hipError_t backward_of<float>(const MaskedAttentionArgs&, bool, hipStream_t);
}
}  // namespace nnh
