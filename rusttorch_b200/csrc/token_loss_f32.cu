// token_loss_f32.cu — the token loss of f32 logits.
#include "token_loss.cuh"

namespace rt {
RT_TOKEN_LOSS_TYPE(float, f32)
}  // namespace rt
