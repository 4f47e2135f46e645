// fp32 kernels of all_reduce_norm.hpp for world sizes 1 to 4.
#include "all_reduce_norm.hpp"

SMR_INSTANTIATE_FORWARD(false, 1)
SMR_INSTANTIATE_FORWARD(false, 2)
SMR_INSTANTIATE_FORWARD(false, 3)
SMR_INSTANTIATE_FORWARD(false, 4)
