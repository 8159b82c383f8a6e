// Window attention with gradients, __bf16 instantiations.
#include "attention_train_kernels.h"

namespace crumpet {
namespace train {

int attention_forward_bf16(const AttnArgs& a, int D, void* stream) { return forward_any<__bf16>(a, D, stream); }
int attention_backward_bf16(const AttnArgs& a, int D, void* stream) { return backward_any<__bf16>(a, D, stream); }

}  // namespace train
}  // namespace crumpet
