// Translation unit: rotary embedding from positions on several axes (rope_axes.cuh).
#include <type_traits>

#include "rope_axes.cuh"
