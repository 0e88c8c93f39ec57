// Translation unit: the residual's addition with its norm and 8-bit output, and their gradients (resnorm.cuh).
#include "resnorm.cuh"
