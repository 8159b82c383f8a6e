// Window attention with gradients, bias-stationary kernels: _Float16, a mask tensor.
#include "attention_train_tuned.h"

namespace crumpet {
namespace train {

int attention_tuned_f16_mask(const AttnArgs& a, const Order& o, int D, bool grad, void* stream) {
    return tuned_any<_Float16, true>(a, o, D, grad, stream);
}

}  // namespace train
}  // namespace crumpet
