// The attention of prompts over float32 elements.
#include "prompt.hpp"

namespace certex_amd::attention {

size_t prompt_workspace_f32(prompt_args const& a) { return workspace_for<float>(a); }
void prompt_f32(prompt_args const& a, hipStream_t stream) { launch<float>(a, stream); }

}  // namespace certex_amd::attention
