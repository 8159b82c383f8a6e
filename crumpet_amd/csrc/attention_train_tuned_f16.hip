// Window attention with gradients, bias-stationary kernels: _Float16, shifted windows or no mask.
#include "attention_train_tuned.h"

namespace crumpet {
namespace train {

int attention_tuned_f16(const AttnArgs& a, const Order& o, int D, bool grad, void* stream) {
    return tuned_any<_Float16, false>(a, o, D, grad, stream);
}

}  // namespace train
}  // namespace crumpet
