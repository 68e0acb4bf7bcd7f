// The operators on device tensors (include/hat.h): argument checks, the choice of a
// kernel and its launch on the caller's stream.
#pragma once
#include "../../include/hat.h"

namespace hat {

void op_rotary(const hat_rotary* a, void* stream);
size_t op_attention_workspace(const hat_attention* a);
void op_attention(const hat_attention* a, void* stream);
void op_residual_norm(const hat_residual_norm* a, void* stream);

}  // namespace hat
