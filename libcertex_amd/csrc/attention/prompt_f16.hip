// The attention of prompts over float16 elements.
#include "prompt.hpp"

namespace certex_amd::attention {

size_t prompt_workspace_f16(prompt_args const& a) { return workspace_for<f16_t>(a); }
void prompt_f16(prompt_args const& a, hipStream_t stream) { launch<f16_t>(a, stream); }

}  // namespace certex_amd::attention
