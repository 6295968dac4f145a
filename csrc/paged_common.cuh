// What the kernels that serve from paged caches share.
#pragma once
#include "common.cuh"
#include <atomic>

namespace ats {

// bf16 [rows, heads, d], rows `ld` elements apart, as boxes of 64 columns x `box_heads` heads x `box_rows` rows, 128-byte swizzle; rows behind the last
// read as zero.
inline int make_tmap_tokens(CUtensorMap* out, const void* base, uint64_t rows, uint64_t heads, uint64_t d, uint64_t ld, uint32_t box_heads, uint32_t box_rows) {
  EncodeTiledFn enc = get_encode_tiled();
  if (!enc) return 1000;
  if ((reinterpret_cast<uintptr_t>(base) & 15) || (ld & 7) || (d & 7)) return 1001;
  cuuint64_t dims[3] = {d, heads, rows};
  cuuint64_t strides[2] = {d * 2, ld * 2};
  cuuint32_t box[3] = {64, box_heads, box_rows};
  cuuint32_t estr[3] = {1, 1, 1};
  const CUresult r = enc(out, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? 0 : 1100 + int(r);
}

// Pages [rows, n_kv, d] (rows = pages * page): `box_rows` tokens of one head.
inline int make_tmap_pages(CUtensorMap* out, const void* base, uint64_t rows, uint64_t n_kv, uint64_t d, uint32_t box_rows) {
  return make_tmap_tokens(out, base, rows, n_kv, d, n_kv * d, 1, box_rows);
}

// Operands that are read or written 16 bytes at a time begin at multiples of 16 bytes.
template <typename... P>
inline bool off_16(const P*... p) {
  return ((reinterpret_cast<uintptr_t>(p) | ...) & 15) != 0;
}

// Launches a kernel that begins with pdl_prologue() right behind one of the same operator that asks for it (griddepcontrol.launch_dependents behind its own
// wait): it is set up while that one ends, whatever launches the thread makes else.
template <typename... KArgs, typename... Args>
inline cudaError_t launch_behind(void (*kernel)(KArgs...), dim3 grid, dim3 block, cudaStream_t stream, size_t smem, Args&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, std::forward<Args>(args)...);
}

// Makes the device's context the calling thread's (tensor maps are encoded by the driver).  In the mode in which it may be asked for during a capture, this thread's
// or another's: the first call of a thread may be a captured one.
inline void bind_context() {
  static thread_local bool bound = false;
  if (bound) return;
  cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
  cudaThreadExchangeStreamCaptureMode(&mode);
  cudaFree(0);
  cudaThreadExchangeStreamCaptureMode(&mode);
  bound = true;
}

// A kernel's shared-memory limit, raised once per device.
struct DeviceOnce {
  std::atomic<unsigned long long> done{0};
  template <typename K>
  cudaError_t smem(K kernel, int bytes) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess || (dev < 64 && (done.load(std::memory_order_acquire) >> dev & 1))) return e;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess && dev < 64) done.fetch_or(1ull << dev, std::memory_order_release);
    return e;
  }
};

struct PagedRows {
  const int* starts;    // [R + 1] packed starts of the rows' new tokens
  const int* lengths;   // [R] tokens of a row, the new ones among them
  const int* tables;    // [R, width]
  int R, width, pages, page_log, tokens;   // tokens: rows of the packed batch
};
// New tokens and keys of row r, as far as the batch and the table hold them: no index that follows from these leaves its buffer, whatever the plan says.
__device__ __forceinline__ void paged_row(const PagedRows& p, int r, int* first, int* fresh, int* keys) {
  const int a = min(max(p.starts[r], 0), p.tokens), b = min(max(p.starts[r + 1], a), p.tokens);
  const long long room = (long long)p.width << p.page_log;
  const int len = (int)min((long long)max(p.lengths[r], 0), room);
  *first = a;
  *fresh = b - a;
  *keys = len;
}

}  // namespace ats
