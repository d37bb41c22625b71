// The attention gradients in fp16.
#include "attention_bwd.hpp"

namespace nsh {
template int attention_backward_launch<f16>(const Att&, hipStream_t);
}
