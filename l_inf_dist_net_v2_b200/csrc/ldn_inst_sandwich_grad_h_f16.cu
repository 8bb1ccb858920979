#include "ldn_sandwich_grad.cuh"

namespace ldn {

template int sandwich_grad_rows<__half, false>(Gate, const SandwichGradArgs&, const DeviceCtx*, int*, const cudaStream_t*);

}  // namespace ldn
