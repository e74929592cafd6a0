#include "tmoe_norm_launch.hpp"

namespace tmoe {
TMOE_NORM_TYPE(uint16_t)
}  // namespace tmoe
