// Window attention with gradients, _Float16 instantiations.
#include "attention_train_kernels.h"

namespace crumpet {
namespace train {

int attention_forward_f16(const AttnArgs& a, int D, void* stream) { return forward_any<_Float16>(a, D, stream); }
int attention_backward_f16(const AttnArgs& a, int D, void* stream) { return backward_any<_Float16>(a, D, stream); }

}  // namespace train
}  // namespace crumpet
