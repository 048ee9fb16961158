// A CUDA runtime for the latent attention's host code that launches nothing: it records each launch and fails the one it
// is told to.
#include <cuda_runtime.h>

#include <map>
#include <string>

namespace {
std::map<const void*, std::string>& names() {
  static std::map<const void*, std::string> m;
  return m;
}
std::string text, message;
int launches, fail_at = -1;
}  // namespace

extern "C" {
void fake_begin(int fail) { text.clear(), launches = 0, fail_at = fail; }
const char* fake_launches() { return text.c_str(); }
const char* fake_message() { return message.c_str(); }

void** __cudaRegisterFatBinary(void*) { static void* h; return &h; }
void __cudaRegisterFatBinaryEnd(void**) {}
void __cudaUnregisterFatBinary(void**) {}
void __cudaRegisterFunction(void**, const char* host, char*, const char* name, int, uint3*, uint3*, dim3*, dim3*, int*) { names()[host] = name; }
unsigned __cudaPushCallConfiguration(dim3, dim3, size_t, cudaStream_t) { return 0; }
cudaError_t __cudaPopCallConfiguration(dim3*, dim3*, size_t*, void*) { return cudaSuccess; }
cudaError_t cudaLaunchKernel(const void*, dim3, dim3, void**, size_t, cudaStream_t) { return cudaErrorUnknown; }
cudaError_t cudaLaunchKernelExC(const cudaLaunchConfig_t* c, const void* f, void**) {
  text += names()[f] + " " + std::to_string(c->gridDim.x) + " " + std::to_string(c->gridDim.y) + " " + std::to_string(c->blockDim.x) + " " +
          std::to_string(c->dynamicSmemBytes) + (c->numAttrs > 0 ? " early" : "") + "\n";
  return launches++ == fail_at ? cudaErrorLaunchOutOfResources : cudaSuccess;
}
const char* cudaGetErrorString(cudaError_t) { return "a launch that was told to fail"; }
cudaError_t cudaGetDevice(int* d) { *d = 0; return cudaSuccess; }
cudaError_t cudaDeviceGetAttribute(int* v, cudaDeviceAttr, int) { *v = 148; return cudaSuccess; }
cudaError_t cudaFuncSetAttribute(const void*, cudaFuncAttribute, int) { return cudaSuccess; }
static int encode() { return 0; }
cudaError_t cudaGetDriverEntryPoint(const char*, void** fn, unsigned long long, cudaDriverEntryPointQueryResult* q) {
  *fn = reinterpret_cast<void*>(encode), *q = cudaDriverEntryPointSuccess;
  return cudaSuccess;
}
cudaError_t cudaGetDriverEntryPoint_ptsz(const char* s, void** fn, unsigned long long f, cudaDriverEntryPointQueryResult* q) { return cudaGetDriverEntryPoint(s, fn, f, q); }
cudaError_t cudaGetDriverEntryPointByVersion(const char* s, void** fn, unsigned, unsigned long long f, cudaDriverEntryPointQueryResult* q) { return cudaGetDriverEntryPoint(s, fn, f, q); }
}

namespace mk {
int set_last_error(int code, const char* msg) { message = msg; return code; }
}
