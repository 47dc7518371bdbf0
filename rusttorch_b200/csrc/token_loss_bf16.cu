// token_loss_bf16.cu — the token loss of bf16 logits.
#include "token_loss.cuh"

namespace rt {
RT_TOKEN_LOSS_TYPE(bf16, bf16)
}  // namespace rt
