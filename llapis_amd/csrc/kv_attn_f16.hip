// kv_attn_f16.hip -- kv_attn.h's kernel for this cache type.
#include "kv_attn.h"

namespace llapis {

hipError_t launch_kv_attn_f16(const KvAttn & p, int head_dim, hipStream_t s) {
    return dev::launch_kv_attn_type<dev::KV_F16>(p, head_dim, s);
}

}  // namespace llapis
