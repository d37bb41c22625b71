// The forward attention kernels in fp16.
#include "attention_fwd.hpp"

namespace nsh {
template int attention_forward_launch<f16>(const Att&, hipStream_t);
}
