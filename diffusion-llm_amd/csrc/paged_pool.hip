// paged_pool.hip - attention of ragged batches over paged caches held in 8 bits, and
// over the pages of a list: the tiles of paged_tiles.h for every kind of pool.
#include "paged_tiles.h"

namespace bd3 {

hipError_t launch_paged_pool(const PagedArgs& a, int pool, hipStream_t stream) {
  if (a.columns != nullptr) {
    if (pool == kPoolInt8) return launch_paged_tiles<kPoolInt8, true>(a, stream);
    if (pool == kPoolE4m3) return launch_paged_tiles<kPoolE4m3, true>(a, stream);
    return launch_paged_tiles<kPoolBf16, true>(a, stream);
  }
  if (pool == kPoolInt8) return launch_paged_tiles<kPoolInt8, false>(a, stream);
  return launch_paged_tiles<kPoolE4m3, false>(a, stream);
}

}  // namespace bd3
