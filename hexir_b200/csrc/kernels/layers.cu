// layers.cu -- the translation unit of the layer kernels (linear_16.cu,
// layer_norm.cu): a CUBIN of its own in libhexir_b200.so, apart from
// kernels.cu's, because that one is written into every cuda-placed .hxb.

#include "common.cuh"

extern "C" __device__ unsigned int hexir_device_error_word = 0u;

#include "linear_16.cu"
#include "layer_norm.cu"
