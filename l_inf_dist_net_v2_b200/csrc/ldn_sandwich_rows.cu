// (simple kernels only so far)
#include "ldn_sandwich.cuh"
namespace ldn {
bool sandwich_in_registers(Gate, const SandwichArgs&, int, const DeviceCtx*, cudaStream_t, int*) { return false; }
bool sandwich_grad_in_registers(Gate, const SandwichGradArgs&, int, const DeviceCtx*, int*) { return false; }
int launch_sandwich_grad_in_registers(Gate, const SandwichGradArgs&, int, const DeviceCtx*, cudaStream_t) { return kBadArgument; }
}  // namespace ldn
