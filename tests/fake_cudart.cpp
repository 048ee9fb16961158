// A CUDA runtime for the batch operators' host code that launches nothing: it records each launch, fails the
// one it is told to, and keeps the last error until it is asked for, as the runtime does.
#include <cuda_runtime.h>

#include <cstdint>
#include <map>
#include <string>

namespace {
std::map<const void*, std::string>& names() {
  static std::map<const void*, std::string> m;
  return m;
}
std::string text, message;
int launches, fail_at = -1;
cudaError_t last = cudaSuccess;
dim3 grid_, block_;
size_t smem_;
cudaStream_t stream_;

cudaError_t launch(const std::string& name, dim3 g, dim3 b, bool overlaps) {
  text += name + " " + std::to_string(g.x) + " " + std::to_string(g.y) + " " + std::to_string(b.x) + (overlaps ? " overlaps" : "") + "\n";
  const cudaError_t e = launches++ == fail_at ? cudaErrorLaunchOutOfResources : cudaSuccess;
  if (e != cudaSuccess) last = e;
  return e;
}
}  // namespace

extern "C" {
void fake_begin(int fail, int pending) { text.clear(), launches = 0, fail_at = fail, last = static_cast<cudaError_t>(pending); }
const char* fake_launches() { return text.c_str(); }

void** __cudaRegisterFatBinary(void*) { static void* h; return &h; }
void __cudaRegisterFatBinaryEnd(void**) {}
void __cudaUnregisterFatBinary(void**) {}
void __cudaRegisterFunction(void**, const char* host, char*, const char* name, int, uint3*, uint3*, dim3*, dim3*, int*) { names()[host] = name; }
unsigned __cudaPushCallConfiguration(dim3 g, dim3 b, size_t smem, cudaStream_t s) { grid_ = g, block_ = b, smem_ = smem, stream_ = s; return 0; }
cudaError_t __cudaPopCallConfiguration(dim3* g, dim3* b, size_t* smem, void* s) {
  *g = grid_, *b = block_, *smem = smem_, *static_cast<cudaStream_t*>(s) = stream_;
  return cudaSuccess;
}
cudaError_t cudaLaunchKernel(const void* f, dim3 g, dim3 b, void**, size_t, cudaStream_t) { return launch(names()[f], g, b, false); }
cudaError_t cudaLaunchKernelExC(const cudaLaunchConfig_t* c, const void* f, void**) { return launch(names()[f], c->gridDim, c->blockDim, c->numAttrs > 0); }
cudaError_t cudaGetLastError() { const cudaError_t e = last; last = cudaSuccess; return e; }
const char* cudaGetErrorString(cudaError_t e) { return e == cudaSuccess ? "no error" : "a launch that was told to fail"; }
cudaError_t cudaGetDevice(int* d) { *d = 0; return cudaSuccess; }
cudaError_t cudaDeviceGetAttribute(int* v, cudaDeviceAttr, int) { *v = 148; return cudaSuccess; }
}

namespace mk {
int set_last_error(int code, const char* msg) { message = msg; return code; }
}
namespace w4 {   // the products' own launches, which are instantiated in files of their own
struct Args;
int product(const char* type, bool two, bool xr, int grid) {
  const std::string name = std::string(type) + (two ? " two" : " one") + (xr ? " xr" : "");
  return launch(name, dim3(grid), dim3(0), false) == cudaSuccess ? 0 : mk::set_last_error(-2, "a product that was told to fail");
}
int launch_bf16(const Args&, int, bool two, bool xr, int grid, cudaStream_t) { return product("bf16", two, xr, grid); }
int launch_fp16(const Args&, int, bool two, bool xr, int grid, cudaStream_t) { return product("fp16", two, xr, grid); }
}
extern "C" const char* fake_message() { return message.c_str(); }
