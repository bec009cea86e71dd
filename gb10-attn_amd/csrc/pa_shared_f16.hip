// pa_shared_f16.hip -- instances of pa_shared.hpp over fp16 caches.
#include "pa_shared.hpp"

namespace pa {
hipError_t launch_shared_f16(const SharedParams& p, hipStream_t stream) { return launch_shared_kv<KvF16, false>(p, stream); }
}  // namespace pa
