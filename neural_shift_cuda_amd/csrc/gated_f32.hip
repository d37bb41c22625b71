#include "gated.hpp"

namespace nsh {
NSH_GATED_ENTRIES(, float, false)
NSH_GATED_FEW_ROWS(, float)
}  // namespace nsh
