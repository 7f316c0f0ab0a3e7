// kv_prefix_f16.hip -- kv_prefix.h's kernel for this cache type.
#include "kv_prefix.h"

namespace llapis {

hipError_t launch_kv_prefix_f16(const KvPrefix & p, int head_dim, hipStream_t s) {
    return dev::launch_kv_prefix_type<dev::KV_F16>(p, head_dim, s);
}

}  // namespace llapis
