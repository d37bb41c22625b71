// The forward attention kernels in fp32.
#include "attention_fwd.hpp"

namespace nsh {
template int attention_forward_launch<float>(const Att&, hipStream_t);
}
