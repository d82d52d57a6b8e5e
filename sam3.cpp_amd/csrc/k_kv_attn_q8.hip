// k_kv_attn_q8.hip — attention over a Q8_0 cache.
#include "k_kv_attn.h"

namespace s3e {

hipError_t launch_kv_attn_q8(const KvAttnArgs &a, bool f32, hipStream_t st) { return launch_kv_attn<8>(a, f32, st); }

}  // namespace s3e
