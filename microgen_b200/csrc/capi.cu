// C-ABI plumbing: status strings, error words, version, TMA descriptors.
#include <cstdlib>
#include <mutex>

#include "common.cuh"

__device__ int g_mg_dev_error = 0;
__device__ int g_mg_dev_error_info = 0;

static thread_local int t_last_cuda_error = 0;

bool mg_pdl_enabled() {
  static const bool on = [] {
    const char* v = getenv("MG_PDL");
    return !(v && v[0] == '0');
  }();
  return on;
}

int mg_set_cuda_error(cudaError_t e) {
  t_last_cuda_error = static_cast<int>(e);
  return MG_ERR_CUDA;
}

typedef CUresult (*PFN_encodeTiled_t)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                      const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                      CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

static PFN_encodeTiled_t get_encode_fn() {
  static PFN_encodeTiled_t fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PFN_encodeTiled_t>(p);
  });
  return fn;
}

int mg_make_map_2d(CUtensorMap* map, CUtensorMapDataType dt, const void* base, uint64_t inner, uint64_t outer,
                   uint64_t row_bytes, uint32_t box_inner, uint32_t box_outer, CUtensorMapSwizzle swizzle) {
  PFN_encodeTiled_t enc = get_encode_fn();
  if (!enc) return MG_ERR_CUDA;
  cuuint64_t dims[2] = {inner, outer};
  cuuint64_t strides[1] = {row_bytes};
  cuuint32_t box[2] = {box_inner, box_outer};
  cuuint32_t es[2] = {1, 1};
  CUresult r = enc(map, dt, 2, const_cast<void*>(base), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
                   swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? MG_OK : MG_ERR_INVALID_ARG;
}

int mg_make_map_3d(CUtensorMap* map, CUtensorMapDataType dt, const void* base, const uint64_t (&dims)[3],
                   const uint64_t (&strides)[2], const uint32_t (&box)[3], CUtensorMapSwizzle swizzle) {
  PFN_encodeTiled_t enc = get_encode_fn();
  if (!enc) return MG_ERR_CUDA;
  cuuint64_t d[3] = {dims[0], dims[1], dims[2]}, st[2] = {strides[0], strides[1]};
  cuuint32_t b[3] = {box[0], box[1], box[2]}, es[3] = {1, 1, 1};
  CUresult r = enc(map, dt, 3, const_cast<void*>(base), d, st, b, es, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle,
                   CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? MG_OK : MG_ERR_INVALID_ARG;
}

int mg_error_words(int** code, int** info) {
  static int* addr[64][2] = {};
  static std::mutex mu;
  int dev = 0;
  MG_CUDA_TRY(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64) return MG_ERR_UNSUPPORTED;
  std::lock_guard<std::mutex> lock(mu);
  if (!addr[dev][1]) {
    void *c = nullptr, *i = nullptr;
    MG_CUDA_TRY(cudaGetSymbolAddress(&c, g_mg_dev_error));
    MG_CUDA_TRY(cudaGetSymbolAddress(&i, g_mg_dev_error_info));
    addr[dev][0] = static_cast<int*>(c);
    addr[dev][1] = static_cast<int*>(i);
  }
  *code = addr[dev][0];
  *info = addr[dev][1];
  return MG_OK;
}

extern "C" int mg_abi_version(void) { return MG_ABI_VERSION; }

extern "C" const char* mg_status_string(int status) {
  switch (status) {
    case MG_OK: return "ok";
    case MG_ERR_INVALID_ARG: return "invalid argument";
    case MG_ERR_UNSUPPORTED: return "unsupported shape";
    case MG_ERR_CUDA: return "CUDA runtime error";
    case MG_ERR_TIMEOUT: return "bounded device wait timed out";
    case MG_ERR_DEVICE: return "device-side check failed";
    default: return "unknown status";
  }
}

extern "C" int mg_last_cuda_error(void) { return t_last_cuda_error; }

extern "C" int mg_device_error(void* stream, int clear, int* code, int* info) {
  if (!code) return MG_ERR_INVALID_ARG;
  cudaStream_t s = mg_stream(stream);
  int vals[2] = {0, 0};
  MG_CUDA_TRY(cudaMemcpyFromSymbolAsync(&vals[0], g_mg_dev_error, sizeof(int), 0, cudaMemcpyDeviceToHost, s));
  MG_CUDA_TRY(cudaStreamSynchronize(s));
  if (vals[0] != MG_OK) {  // the common case (no error) costs one read and one synchronisation
    MG_CUDA_TRY(cudaMemcpyFromSymbolAsync(&vals[1], g_mg_dev_error_info, sizeof(int), 0, cudaMemcpyDeviceToHost, s));
    MG_CUDA_TRY(cudaStreamSynchronize(s));
  }
  *code = vals[0];
  if (info) *info = vals[1];
  if (clear && vals[0] != MG_OK) {
    const int zero[2] = {0, 0};
    MG_CUDA_TRY(cudaMemcpyToSymbolAsync(g_mg_dev_error, &zero[0], sizeof(int), 0, cudaMemcpyHostToDevice, s));
    MG_CUDA_TRY(cudaMemcpyToSymbolAsync(g_mg_dev_error_info, &zero[1], sizeof(int), 0, cudaMemcpyHostToDevice, s));
    MG_CUDA_TRY(cudaStreamSynchronize(s));
  }
  return MG_OK;
}
