#include "gated.hpp"

namespace nsh {
NSH_GATED_ENTRIES(, f16)
}  // namespace nsh
