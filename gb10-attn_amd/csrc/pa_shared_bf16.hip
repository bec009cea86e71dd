// pa_shared_bf16.hip -- instances of pa_shared.hpp over bf16 caches.
#include "pa_shared.hpp"

namespace pa {
hipError_t launch_shared_bf16(const SharedParams& p, hipStream_t stream) { return launch_shared_kv<KvBF16, true>(p, stream); }
}  // namespace pa
