// k_kv_attn_q4.hip — attention over a Q4_0 cache.
#include "k_kv_attn.h"

namespace s3e {

hipError_t launch_kv_attn_q4(const KvAttnArgs &a, bool f32, hipStream_t st) { return launch_kv_attn<4>(a, f32, st); }

void kv_attn_columns(KvAttnArgs &a, int D, bool f32, int64_t cols) {
    const int NB = D / 32;
    int64_t per;
    a.tile = cols > 32;
    if (a.tile) {
        a.nt = kv_tile_nt(NB, f32);
        per = kv_tile_cols(NB, f32);
        // no more than run at once: a few left over would take as long again (4096
        // × 28 736 at head dim 256: 242 work-groups 235 µs, 264 294)
        a.goal = 256 * (kv_tile_fill(NB, f32) * 4 / kv_tile_waves(NB, f32));
    } else {
        a.nt = cols <= 16 || NB == 8 ? 1 : 2;
        per = 16 * a.nt;
        // sequences of unlike length fill the CUs better in more, shorter ranges
        // (µs by goal, 64 of up to 4096 keys / one of 131 072: 512 62.5 / 41.1, 768
        // 57.7 / 40.8, 1536 53.4 / 45.5, 3072 54.8 / 50.5)
        a.goal = a.n_seq > 1 ? 1536 : 768;
    }
    a.ctiles = (int)((cols + per - 1) / per);
}

}  // namespace s3e
