// The attention gradients in fp32.
#include "attention_bwd.hpp"

namespace nsh {
template int attention_backward_launch<float>(const Att&, hipStream_t);
}
