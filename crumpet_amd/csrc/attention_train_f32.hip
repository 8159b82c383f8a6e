// Window attention with gradients, float instantiations.
#include "attention_train_kernels.h"

namespace crumpet {
namespace train {

int attention_forward_f32(const AttnArgs& a, int D, void* stream) { return forward_any<float>(a, D, stream); }
int attention_backward_f32(const AttnArgs& a, int D, void* stream) { return backward_any<float>(a, D, stream); }

}  // namespace train
}  // namespace crumpet
