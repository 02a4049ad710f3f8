// launches.cpp -- the kernels that a call would launch, without a GPU: a library that
// is loaded before libark_opt.so and stands in for the parts of the runtime that its
// entry points use.  Every address is device memory, nothing runs, and a launch is a
// line of text: grid, block and the kernel's (mangled) name.  (tests/launches.py)
#include <hip/hip_runtime_api.h>

#include <map>
#include <string>

static std::map<const void*, std::string> names;
static std::string lines;

extern "C" {

void launches_clear() { lines.clear(); }
const char* launches_lines() { return lines.c_str(); }

void __hipRegisterFunction(void**, const void* host, char*, const char* name, unsigned, void*,
                           void*, void*, void*, int*) {
  names[host] = name;
}

// what <<<grid, block>>> hands to the kernel's stub
static dim3 next_grid, next_block;
static size_t next_lds;
static hipStream_t next_stream;
hipError_t __hipPushCallConfiguration(dim3 grid, dim3 block, size_t lds, hipStream_t stream) {
  next_grid = grid, next_block = block, next_lds = lds, next_stream = stream;
  return hipSuccess;
}
hipError_t __hipPopCallConfiguration(dim3* grid, dim3* block, size_t* lds, hipStream_t* stream) {
  *grid = next_grid, *block = next_block, *lds = next_lds, *stream = next_stream;
  return hipSuccess;
}

hipError_t hipLaunchKernel(const void* fn, dim3 grid, dim3 block, void**, size_t, hipStream_t) {
  const auto it = names.find(fn);
  lines += std::to_string(grid.x) + " " + std::to_string(grid.y) + " " + std::to_string(block.x) +
           " " + (it == names.end() ? "?" : it->second) + "\n";
  return hipSuccess;
}

hipError_t hipFuncSetAttribute(const void*, hipFuncAttribute, int) { return hipSuccess; }
hipError_t hipGetLastError() { return hipSuccess; }
hipError_t hipGetDevice(int* dev) {
  *dev = 0;
  return hipSuccess;
}
hipError_t hipPointerGetAttributes(hipPointerAttribute_t* a, const void* p) {
  *a = hipPointerAttribute_t{};
  a->type = hipMemoryTypeDevice;
  a->devicePointer = (void*)p;
  return hipSuccess;
}
hipError_t hipMemGetAddressRange(hipDeviceptr_t*, size_t*, hipDeviceptr_t) {
  return hipErrorNotFound;  // an allocation of unknown size: taken as it is
}

}  // extern "C"
