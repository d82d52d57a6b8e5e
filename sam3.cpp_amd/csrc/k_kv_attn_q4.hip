// k_kv_attn_q4.hip — attention over a Q4_0 cache.
#include "k_kv_attn.h"

namespace s3e {

hipError_t launch_kv_attn_q4(const KvAttnArgs &a, bool f32, hipStream_t st) { return launch_kv_attn<4>(a, f32, st); }

int kv_attn_nt(int type, int D, bool f32, int64_t cols) {
    if (cols <= 16) return 1;
    switch (D) {
        case 32: return f32 ? kv_most_tiles<1, true>() : kv_most_tiles<1, false>();
        case 64: return f32 ? kv_most_tiles<2, true>() : kv_most_tiles<2, false>();
        case 96: return f32 ? kv_most_tiles<3, true>() : kv_most_tiles<3, false>();
        case 128: return f32 ? kv_most_tiles<4, true>() : kv_most_tiles<4, false>();
        default: return f32 ? kv_most_tiles<8, true>() : kv_most_tiles<8, false>();
    }
}

}  // namespace s3e
