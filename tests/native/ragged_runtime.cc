// host_runtime.cc with more of a machine behind it, for the host side of the
// grouped and 4-bit products: two devices, memory that can run out, frees,
// kernel attributes and the kernels' argument blocks in the list of calls.
#include <hip/hip_runtime_api.h>

#define hipMalloc standin_base_malloc
#define hipFree standin_base_free
#define hipLaunchKernel standin_base_launch
#define hipGetDeviceCount standin_base_count
#define hipSetDevice standin_base_set_device
#include "host_runtime.cc"
#undef hipMalloc
#undef hipFree
#undef hipLaunchKernel
#undef hipGetDeviceCount
#undef hipSetDevice

namespace {
size_t g_limit = ~(size_t)0;  // the largest allocation that there is memory for
int g_device = 0;
bool g_attributes = true;  // whether kernel attributes can be set
int g_arguments = 0;       // bytes of the product kernels' argument block that are listed with a launch

void note_bytes(const void *from, int count) {
  g_log += "arguments ";
  for (int i = 0; i < count; ++i) {
    char hex[3];
    std::snprintf(hex, sizeof(hex), "%02x", ((const unsigned char *)from)[i]);
    g_log += hex;
  }
  g_log += '\n';
}

// A program that cannot call the functions below (node) is given what to list
// and where to write the list at its end in its environment.
struct Environment {
  Environment() {
    if (const char *bytes = std::getenv("STANDIN_ARGUMENTS")) g_arguments = std::atoi(bytes);
  }
  ~Environment() {
    if (const char *path = std::getenv("STANDIN_LOG"))
      if (std::FILE *file = std::fopen(path, "w")) {
        std::fwrite(g_log.data(), 1, g_log.size(), file);
        std::fclose(file);
      }
  }
} g_environment;
}  // namespace

extern "C" {

void standin_memory(size_t largest) { g_limit = largest; }
void standin_attributes(int work) { g_attributes = work != 0; }
void standin_arguments(int bytes) { g_arguments = bytes; }

hipError_t hipMalloc(void **ptr, size_t bytes) {
  if (bytes > g_limit) {
    note("out_of_memory %zu", bytes);
    return hipErrorOutOfMemory;
  }
  const hipError_t e = standin_base_malloc(ptr, bytes);
  note("at %zx", (size_t)*ptr);
  return e;
}
hipError_t hipFree(void *ptr) {
  note("free %zx", (size_t)ptr);
  return hipSuccess;
}
hipError_t hipLaunchKernel(const void *host, dim3 grid, dim3 block, void **args, size_t shared, hipStream_t stream) {
  const hipError_t e = standin_base_launch(host, grid, block, args, shared, stream);
  note("device %d shared %zu", g_device, shared);
  const std::string &name = g_kernels[host];
  if (g_arguments && name.find("ragged_kernel") != std::string::npos) {
    note_bytes(args[0], g_arguments);
  } else if (g_arguments && name.find("quantize") != std::string::npos) {
    for (int i = 0; i < 7; ++i) note_bytes(args[i], 8);  // pointers and sizes come first in all of them
  }
  return e;
}
hipError_t hipFuncSetAttribute(const void *host, hipFuncAttribute, int value) {
  note("attribute %d %d %s", g_device, value, g_kernels[host].c_str());
  return g_attributes ? hipSuccess : hipErrorInvalidValue;
}
hipError_t hipGetDeviceCount(int *count) {
  *count = 2;
  return hipSuccess;
}
hipError_t hipSetDevice(int device) {
  g_device = device;
  return hipSuccess;
}

}  // extern "C"
