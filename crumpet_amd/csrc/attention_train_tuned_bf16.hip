// Window attention with gradients, bias-stationary kernels: __bf16, shifted windows or no mask.
#include "attention_train_tuned.h"

namespace crumpet {
namespace train {

int attention_tuned_bf16(const AttnArgs& a, const Order& o, int D, bool grad, void* stream) {
    return tuned_any<__bf16, false>(a, o, D, grad, stream);
}

}  // namespace train
}  // namespace crumpet
