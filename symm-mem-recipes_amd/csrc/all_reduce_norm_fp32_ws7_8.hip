// fp32 kernels of all_reduce_norm.hpp for world sizes 7 to 8.
#include "all_reduce_norm.hpp"

SMR_INSTANTIATE_FORWARD(false, 7)
SMR_INSTANTIATE_FORWARD(false, 8)
