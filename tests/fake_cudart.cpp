// Host-only stand-in for the CUDA runtime calls of csrc/paged_prefill.cu: two devices, one
// current, and no GPU.  A launch fails, as the runtime's does, unless the function's limit of
// dynamic shared memory has been raised on the current device.
#include <cuda.h>
#include <cuda_runtime.h>

#include <map>
#include <utility>

namespace {
int g_device = 0, g_launches = 0, g_sets = 0, g_regs = 0;
bool g_refuse = false;                      // the next attributes cannot be set
cudaError_t g_last = cudaSuccess;
dim3 g_grid, g_block;
size_t g_smem = 0;
std::map<std::pair<const void *, int>, int> g_limit;

CUresult encode(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *,
                const cuuint64_t *, const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave,
                CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill) {
  return CUDA_SUCCESS;
}
}  // namespace

extern "C" {

void fake_reset(int device, int regs, int refuse) {
  g_device = device;
  g_regs = regs;
  g_refuse = refuse;
  g_last = cudaSuccess;
}
int fake_launches() { return g_launches; }
int fake_sets() { return g_sets; }

cudaError_t cudaGetDevice(int *d) {
  *d = g_device;
  return cudaSuccess;
}
cudaError_t cudaFuncSetAttribute(const void *f, cudaFuncAttribute, int value) {
  if (g_refuse) return cudaErrorUnknown;
  ++g_sets;
  g_limit[{f, g_device}] = value;
  return cudaSuccess;
}
cudaError_t cudaFuncGetAttributes(cudaFuncAttributes *a, const void *) {
  *a = {};
  a->numRegs = g_regs;
  return cudaSuccess;
}
cudaError_t cudaGetDriverEntryPoint(const char *, void **fn, unsigned long long,
                                    cudaDriverEntryPointQueryResult *q) {
  *fn = reinterpret_cast<void *>(encode);
  *q = cudaDriverEntryPointSuccess;
  return cudaSuccess;
}
cudaError_t cudaGetLastError() {
  const cudaError_t e = g_last;
  g_last = cudaSuccess;
  return e;
}
unsigned __cudaPushCallConfiguration(dim3 grid, dim3 block, size_t smem, struct CUstream_st *) {
  g_grid = grid;
  g_block = block;
  g_smem = smem;
  return 0;
}
cudaError_t __cudaPopCallConfiguration(dim3 *grid, dim3 *block, size_t *smem, void *stream) {
  *grid = g_grid;
  *block = g_block;
  *smem = g_smem;
  *static_cast<void **>(stream) = nullptr;
  return cudaSuccess;
}
cudaError_t cudaLaunchKernel(const void *f, dim3, dim3, void **, size_t smem, cudaStream_t) {
  const auto it = g_limit.find({f, g_device});
  if (smem > 48 * 1024 && (it == g_limit.end() || smem > static_cast<size_t>(it->second)))
    return g_last = cudaErrorInvalidValue;
  ++g_launches;
  return cudaSuccess;
}
char __cudaInitModule(void **) { return 1; }
void **__cudaRegisterFatBinary(void *) { return nullptr; }
void __cudaRegisterFatBinaryEnd(void **) {}
void __cudaUnregisterFatBinary(void **) {}
void __cudaRegisterFunction(void **, const char *, char *, const char *, int, uint3 *, uint3 *, dim3 *,
                            dim3 *, int *) {}
void __cudaRegisterVar(void **, char *, char *, const char *, int, size_t, int, int) {}

}  // extern "C"
