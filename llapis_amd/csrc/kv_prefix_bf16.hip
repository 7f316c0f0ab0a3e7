// kv_prefix_bf16.hip -- kv_prefix.h's kernel for this cache type.
#include "kv_prefix.h"

namespace llapis {

hipError_t launch_kv_prefix_bf16(const KvPrefix & p, int head_dim, hipStream_t s) {
    return dev::launch_kv_prefix_type<dev::KV_BF16>(p, head_dim, s);
}

}  // namespace llapis
