#include "ldn_sandwich_forward.cuh"

namespace ldn {

template bool sandwich_rows<__nv_bfloat16>(Gate, const SandwichArgs&, const DeviceCtx*, cudaStream_t, int*);

}  // namespace ldn
