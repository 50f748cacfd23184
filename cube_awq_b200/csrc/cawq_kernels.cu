// cawq_kernels.cu — the GEMM, dequantize and tensor-parallel kernels of
// libcube_awq.so, one translation unit so they share a device error word
// without relocatable device code (cawq_layer.cu has the other one).
#include "cawq_common.cuh"

namespace cawq {

cudaError_t read_device_error(uint32_t* word, int reset) {
  cudaError_t e = cudaDeviceSynchronize();
  if (e != cudaSuccess) return e;
  *word = 0;
  if ((e = read_own_error_word(word, reset)) != cudaSuccess) return e;
  return read_layer_error(word, reset);
}

}  // namespace cawq

#include "cawq_decode.cuh"
#include "cawq_dequant.cuh"
#include "cawq_generic.cuh"
#include "cawq_prefill.cuh"
#include "cawq_prefill_f32.cuh"
#include "cawq_prefill_tw.cuh"
#include "cawq_tp.cuh"
