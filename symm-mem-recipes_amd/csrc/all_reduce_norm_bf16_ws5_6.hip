// bf16 kernels of all_reduce_norm.hpp for world sizes 5 to 6.
#include "all_reduce_norm.hpp"

SMR_INSTANTIATE_FORWARD(true, 5)
SMR_INSTANTIATE_FORWARD(true, 6)
