// The attention gradients in bf16.
#include "attention_bwd.hpp"

namespace nsh {
template int attention_backward_launch<bf16>(const Att&, hipStream_t);
}
