// kv_prefix_q8.hip -- kv_prefix.h's kernel for this cache type.
#include "kv_prefix.h"

namespace llapis {

hipError_t launch_kv_prefix_q8(const KvPrefix & p, int head_dim, hipStream_t s) {
    return dev::launch_kv_prefix_type<dev::KV_Q8>(p, head_dim, s);
}

}  // namespace llapis
