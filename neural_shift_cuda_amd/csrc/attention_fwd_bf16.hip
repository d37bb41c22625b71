// The forward attention kernels in bf16.
#include "attention_fwd.hpp"

namespace nsh {
template int attention_forward_launch<bf16>(const Att&, hipStream_t);
}
