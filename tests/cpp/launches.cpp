// HIP calls of a process without a GPU: devices of 256 and 64 compute units, of which one is
// current, and the grid of the last launch. Loaded before the library, whose own calls come here.
#include <hip/hip_runtime_api.h>

#include <cstddef>

namespace {
int g_device = 0;
dim3 g_grid, g_block;
}  // namespace

extern "C" {

void launches_set_device(int device) { g_device = device; }
unsigned launches_grid() { return g_grid.x; }

hipError_t hipGetDevice(int* device) {
  *device = g_device;
  return hipSuccess;
}
hipError_t hipDeviceGetAttribute(int* value, hipDeviceAttribute_t attribute, int device) {
  *value = attribute == hipDeviceAttributeMultiprocessorCount ? (device == 0 ? 256 : 64) : 0;
  return hipSuccess;
}
hipError_t hipFuncSetAttribute(const void*, hipFuncAttribute, int) { return hipSuccess; }
hipError_t hipGetLastError() { return hipSuccess; }
hipError_t __hipPushCallConfiguration(dim3 grid, dim3 block, std::size_t, hipStream_t) {
  g_grid = grid;
  g_block = block;
  return hipSuccess;
}
hipError_t __hipPopCallConfiguration(dim3* grid, dim3* block, std::size_t* lds, hipStream_t* stream) {
  *grid = g_grid;
  *block = g_block;
  *lds = 0;
  *stream = nullptr;
  return hipSuccess;
}
hipError_t hipLaunchKernel(const void*, dim3 grid, dim3, void**, std::size_t, hipStream_t) {
  g_grid = grid;
  return hipSuccess;
}

}  // extern "C"
