#include "tmoe_norm_launch.hpp"

namespace tmoe {
TMOE_NORM_TYPE(float)
}  // namespace tmoe
