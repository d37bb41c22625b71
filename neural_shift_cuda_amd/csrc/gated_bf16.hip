#include "gated.hpp"

namespace nsh {
NSH_GATED_ENTRIES(, bf16, false)
NSH_GATED_FEW_ROWS(, bf16)
}  // namespace nsh
