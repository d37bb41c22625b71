#include "gated.hpp"

namespace nsh {
NSH_GATED_ENTRIES(, float, true)
}  // namespace nsh
