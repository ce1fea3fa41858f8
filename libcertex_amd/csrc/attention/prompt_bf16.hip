// The attention of prompts over bfloat16 elements.
#include "prompt.hpp"

namespace certex_amd::attention {

size_t prompt_workspace_bf16(prompt_args const& a) { return workspace_for<bf16_t>(a); }
void prompt_bf16(prompt_args const& a, hipStream_t stream) { launch<bf16_t>(a, stream); }

}  // namespace certex_amd::attention
