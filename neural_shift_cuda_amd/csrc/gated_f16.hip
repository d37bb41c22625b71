#include "gated.hpp"

namespace nsh {
NSH_GATED_ENTRIES(, f16, false)
NSH_GATED_FEW_ROWS(, f16)
}  // namespace nsh
