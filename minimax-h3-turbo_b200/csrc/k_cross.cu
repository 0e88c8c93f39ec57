// Translation unit: cross attention and its gradients (cross_attn.cuh).
#include "cross_attn.cuh"

namespace h3b {

H3B_DEVICE_ERROR_ACCESSOR(device_error_cross)

}  // namespace h3b
