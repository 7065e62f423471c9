// The language-model tuning operators: a translation unit of its own beside memintelli_b200.cu, with its own device
// error flag.
#include <atomic>
#include <type_traits>
#include <utility>

#include "embedding.cu"
#include "token_loss.cu"
#include "grad_clip.cu"
#include "lm_abi.cu"

namespace mib {

cudaError_t lm_take_device_error(int* code) {
  cudaError_t e = cudaMemcpyFromSymbol(code, g_device_error, sizeof(int));
  if (e == cudaSuccess && *code != 0) {
    const int zero = 0;
    e = cudaMemcpyToSymbol(g_device_error, &zero, sizeof(int));
  }
  return e;
}

}  // namespace mib
