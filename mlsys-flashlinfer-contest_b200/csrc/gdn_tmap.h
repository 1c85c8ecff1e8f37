// Tensor maps on the host: the driver's encoder, and a small cache of encoded maps.
#pragma once

#include <cuda.h>
#include <cudaTypedefs.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace gdn {

// cuTensorMapEncodeTiled, or nullptr where the driver has none.
inline PFN_cuTensorMapEncodeTiled_v12000 tmap_encoder() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = [] {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      ptr = nullptr;
    return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(ptr);
  }();
  return fn;
}

// What an encoding depends on: the base address and up to three sizes.
struct TmapKey {
  const void* base;
  int64_t size[3];
  bool operator==(const TmapKey& o) const {
    return base == o.base && size[0] == o.size[0] && size[1] == o.size[1] && size[2] == o.size[2];
  }
};

// Encoding a tensor map costs about a microsecond of host time and a call needs four to six; a small
// per-thread cache of encoded maps (one for each `Encode` type) skips it when a caller reuses its buffers
// (a serving loop, or the caching allocator handing back a block).
template <class Encode>
cudaError_t cached_tmap(CUtensorMap* m, const TmapKey& key, Encode encode) {
  struct Entry {
    TmapKey key;
    CUtensorMap map;
  };
  constexpr int kEntries = 16;
  thread_local Entry cache[kEntries];
  thread_local int used = 0, next = 0;
  for (int i = 0; i < used; ++i)
    if (cache[i].key == key) {
      *m = cache[i].map;
      return cudaSuccess;
    }
  const cudaError_t e = encode(m);
  if (e != cudaSuccess) return e;
  cache[next] = Entry{key, *m};
  next = (next + 1) % kEntries;
  if (used < kEntries) ++used;
  return cudaSuccess;
}

}  // namespace gdn
