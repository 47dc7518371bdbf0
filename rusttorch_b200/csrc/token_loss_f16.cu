// token_loss_f16.cu — the token loss of f16 logits.
#include "token_loss.cuh"

namespace rt {
RT_TOKEN_LOSS_TYPE(f16, f16)
}  // namespace rt
