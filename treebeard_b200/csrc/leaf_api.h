// What the translation units behind include/tbk_leaf.h share: checks, the current device, workspaces.
#pragma once
#include "../../include/tbk_leaf.h"
#include "last_error.h"

#include <algorithm>
#include <atomic>
#include <cstdint>
#include <cuda_runtime.h>

#define CUDA_TRY(expr)                                                                                            \
  do {                                                                                                            \
    cudaError_t e__ = (expr);                                                                                     \
    if (e__ != cudaSuccess)                                                                                       \
      return fail(TBK_ERR_CUDA, "%s failed: %s (%s:%d)", #expr, cudaGetErrorString(e__), __FILE__, __LINE__);     \
  } while (0)

namespace {

using tb::fail;

// Makes a device current for a call's launches and puts the old one back.
struct OnDevice {
  int before = -1;
  cudaError_t error;
  explicit OnDevice(int device) {
    error = cudaGetDevice(&before);
    if (error == cudaSuccess && before != device) error = cudaSetDevice(device);
    else if (error == cudaSuccess) before = -1;
  }
  ~OnDevice() {
    if (before >= 0) cudaSetDevice(before);
  }
};

constexpr int64_t kMost = 0x7ffff000; // of every size: coordinates of tiles behind the last one fit 32 bits

// A workspace cut into 256-byte aligned parts; with a null base only their sizes are added up.
struct Parts {
  unsigned char *base;
  uint64_t used = 0;
  template <class P> P *take(uint64_t count) {
    P *p = base ? reinterpret_cast<P *>(base + used) : nullptr;
    used += (count * sizeof(P) + 255) / 256 * 256;
    return p;
  }
};

int64_t tiles_of(int64_t n, int64_t tile) { return (n + tile - 1) / tile; }

int check_sizes(const char *what, int64_t n, int64_t a, int64_t b) {
  if (n < 0 || a < 1 || b < 1) return fail(TBK_ERR_INVALID, "%s: sizes %lld, %lld, %lld are not >= 0, >= 1, >= 1", what, (long long)n, (long long)a, (long long)b);
  if (n > kMost || a > kMost || b > kMost) return fail(TBK_ERR_UNSUPPORTED, "%s: a size is above %lld", what, (long long)kMost);
  return TBK_OK;
}

// size: bytes of an element (the kernels read whole elements, and misaligned ones end a program)
int check_address(const char *what, const void *p, int size) {
  if (reinterpret_cast<uintptr_t>(p) % size) return fail(TBK_ERR_INVALID, "%s does not begin at a multiple of its elements' %d bytes", what, size);
  return TBK_OK;
}

int check_matrix(const char *what, const void *p, int64_t ld, int64_t rows, int64_t cols, int size) {
  if (!p && rows > 0) return fail(TBK_ERR_INVALID, "%s is null", what);
  if (const int rc = check_address(what, p, size)) return rc;
  if (ld < cols && rows > 1) return fail(TBK_ERR_INVALID, "%s: %lld elements from row to row are less than its %lld columns", what, (long long)ld, (long long)cols);
  if (ld > ((int64_t)1 << 38)) return fail(TBK_ERR_UNSUPPORTED, "%s: %lld elements from row to row", what, (long long)ld);
  return TBK_OK;
}

int check_workspace(const void *p, uint64_t have, uint64_t need) {
  if (need == 0) return TBK_OK;
  if (!p || have < need) return fail(TBK_ERR_INVALID, "the workspace has %llu of %llu bytes", (unsigned long long)(p ? have : 0), (unsigned long long)need);
  if (reinterpret_cast<uintptr_t>(p) % 256) return fail(TBK_ERR_INVALID, "the workspace is not 256-byte aligned");
  return TBK_OK;
}

#define TRY(expr)               \
  do {                          \
    const int rc__ = (expr);    \
    if (rc__) return rc__;      \
  } while (0)

// Launches a kernel that begins with after_previous_kernel(): it may come while the one before it still runs.
template <class... P, class... A> int launch(void (*kernel)(P...), dim3 grid, unsigned threads, size_t smem, cudaStream_t stream, unsigned cluster, A... args) {
  cudaLaunchConfig_t config = {};
  config.gridDim = grid;
  config.blockDim = dim3(threads);
  config.dynamicSmemBytes = smem;
  config.stream = stream;
  cudaLaunchAttribute attrs[2];
  attrs[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attrs[0].val.programmaticStreamSerializationAllowed = 1;
  attrs[1].id = cudaLaunchAttributeClusterDimension;
  attrs[1].val.clusterDim.x = cluster, attrs[1].val.clusterDim.y = 1, attrs[1].val.clusterDim.z = 1;
  config.attrs = attrs;
  config.numAttrs = cluster > 1 ? 2 : 1;
  CUDA_TRY(cudaLaunchKernelEx(&config, kernel, P(args)...));
  return TBK_OK;
}

int64_t up8(int64_t n) { return (n + 7) / 8 * 8; }

// Multiprocessors of a device; the figure of the architecture where there is none (workspace sizes on a host).
int multiprocessors(int device) {
  static std::atomic<int> known[64];
  if (device >= 0 && device < 64 && known[device].load() > 0) return known[device].load();
  int n = 0;
  if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, device) != cudaSuccess || n < 2) {
    cudaGetLastError();
    return 148;
  }
  if (device < 64) known[device].store(n);
  return n;
}

} // namespace
