// pa_shared_fp8.hip -- instances of pa_shared.hpp over FP8 caches: the codes widen
// to bf16 under a bf16 q, to fp16 otherwise.
#include "pa_shared.hpp"

namespace pa {
hipError_t launch_shared_fp8(const SharedParams& p, hipStream_t stream) {
  return p.q_dtype == kBF16 ? launch_shared_kv<KvFP8, true>(p, stream) : launch_shared_kv<KvFP8, false>(p, stream);
}
}  // namespace pa
