// Translation unit: low-rank adapters beside a shared projection, and their gradients (lowrank.cuh).
#include "lowrank.cuh"

namespace h3b {

H3B_DEVICE_ERROR_ACCESSOR(device_error_lowrank)

}  // namespace h3b
