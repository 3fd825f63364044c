// What the extern "C" files share: the per-call device checks and the TMA
// tensor-map encoder (defined in capi.cu), and small argument checks.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include <atomic>

namespace b2a {

// Current device is sm_100 and its error word is known: B2A_OK and *err, or
// the status to return.
int api_prologue(int** err);

// SMs of the current device (148 where it cannot be asked).
int api_sm_count();

// Tiled bf16 tensor map with 128-byte swizzle, out-of-range elements read as
// zero. dims / box have `rank` entries (innermost first), byte_strides
// rank - 1 (dimension i + 1). Returns B2A_OK or B2A_ERR_TMA.
int api_tensor_map(CUtensorMap* m, const void* base, int rank, const unsigned long long* dims,
                   const unsigned long long* byte_strides, const unsigned* box);

// The same of bytes, with the swizzle of box[0] bytes (64 or 128).
int api_tensor_map_bytes(CUtensorMap* m, const void* base, int rank, const unsigned long long* dims,
                         const unsigned long long* byte_strides, const unsigned* box);

inline bool api_aligned(const void* p, unsigned bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

// Strides are not negative and multiples of `mult` elements.
inline bool api_strides_ok(const long long* s, int n, long long mult) {
  for (int i = 0; i < n; ++i)
    if (s[i] < 0 || (s[i] % mult) != 0) return false;
  return true;
}

inline size_t api_align256(size_t x) { return (x + 255) & ~(size_t)255; }

// Launches a kernel whose attributes `prepare` sets: once per device, since the
// runtime's attribute calls cost about a microsecond each and attributes stay
// with the kernel. A device that was reset, or another context of it, has lost
// them, and the launch fails: it is then prepared and launched once more.
// `launch` returns the launch's status and leaves no error behind. Returns 0,
// or -1 on failure.
struct OncePerDevice {
  std::atomic<unsigned long long> done{0};
  template <typename Prepare, typename Launch>
  int run(Prepare&& prepare, Launch&& launch) {
    int dev = 0;
    const bool known = cudaGetDevice(&dev) == cudaSuccess && dev >= 0 && dev < 64;
    const unsigned long long bit = known ? 1ull << dev : 0;
    if ((done.load(std::memory_order_acquire) & bit) && launch() == cudaSuccess) return 0;
    if (prepare() && launch() == cudaSuccess) {
      done.fetch_or(bit, std::memory_order_release);
      return 0;
    }
    done.fetch_and(~bit, std::memory_order_release);
    return -1;
  }
};

// Both give this launch's status: an error that somebody left in the runtime
// before is not taken for it, and a failed launch leaves none (the next
// cudaGetLastError would report it as somebody else's).
template <typename... Params, typename... Args>
inline cudaError_t launch_config(const cudaLaunchConfig_t& cfg, void (*kernel)(Params...), const Args&... args) {
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, args...);
  if (e != cudaSuccess) cudaGetLastError();
  return e;
}

template <typename... Params, typename... Args>
inline cudaError_t launch_plain(void (*kernel)(Params...), dim3 grid, unsigned threads, size_t smem, cudaStream_t st,
                                const Args&... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  return launch_config(cfg, kernel, args...);
}

// Launch as a programmatic dependent: the grid may be scheduled while the
// kernel before it in the stream drains. Its threads wait (grid_dep_wait)
// before they touch memory.
template <typename... Params, typename... Args>
inline cudaError_t launch_dependent(void (*kernel)(Params...), dim3 grid, unsigned threads, size_t smem,
                                    cudaStream_t st, int cluster, const Args&... args) {
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)cluster;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 0 ? 2 : 1;
  return launch_config(cfg, kernel, args...);
}

constexpr float kApiLog2e = 1.4426950408889634f;

}  // namespace b2a
