// Window attention with gradients, bias-stationary kernels: __bf16, a mask tensor.
#include "attention_train_tuned.h"

namespace crumpet {
namespace train {

int attention_tuned_bf16_mask(const AttnArgs& a, const Order& o, int D, bool grad, void* stream) {
    return tuned_any<__bf16, true>(a, o, D, grad, stream);
}

}  // namespace train
}  // namespace crumpet
