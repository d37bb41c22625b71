#include "gated.hpp"

namespace nsh {
NSH_GATED_ENTRIES(, bf16)
}  // namespace nsh
