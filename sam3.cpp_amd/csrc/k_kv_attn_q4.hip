// k_kv_attn_q4.hip — attention over a Q4_0 cache.
#include <algorithm>
#include "k_kv_attn.h"

namespace s3e {

hipError_t launch_kv_attn_q4(const KvAttnArgs &a, bool f32, hipStream_t st) { return launch_kv_attn<4>(a, f32, st); }

// Which kernel, by columns.  At head dim 256 and Q8_0 a work-group's rings leave
// a CU one of them, and the kernel that converts once for 192 columns is ahead
// from about 64 (µs, one kernel / the other, 16 sequences of up to 4096 keys, 4
// heads: 64 columns 77 / 77, 128 150 / 83, 512 502 / 324), with Q4_0 from about
// 256 (192 122 / 96, 256 148 / 167, 384 206 / 171; 64 sequences of 8 heads: 256
// 583 / 755, 512 1096 / 1031).  At the smaller head dims a wave holds two column
// tiles and four or three work-groups share a CU: ahead at every count (4 × 2048
// queries, 16 heads of 64: 109 against 117; 64 × 256 columns of 128: 278 against 379).
void kv_attn_columns(KvAttnArgs &a, int D, bool f32, int64_t cols, int64_t all_cols) {
    const int NB = D / 32;
    const bool q4 = a.c.type == S3E_TYPE_Q4_0;
    int64_t per;
    a.tile = NB == KV_TILE_NB && cols > (q4 ? 256 : 64);
    if (a.tile) {
        a.nt = 1;
        per = kv_tile_cols(f32);
        // no more than run at once: a few left over would take as long again (4096
        // × 28 736 at head dim 256: 242 work-groups 235 µs, 264 294)
        a.goal = 256;
    } else {
        a.nt = cols <= 16 ? 1 : kv_most_tiles(NB);
        per = 16 * a.nt;
        // as many as run at once; sequences of unlike length fill the CUs better in
        // more, shorter ranges where three or more share a CU (µs by goal, one of
        // 131 072 keys, 8 heads: Q4_0 × 128 512 39.0, 768 39.3, 1536 43.0; Q8_0 × 128
        // 512 53.1, 768 62.9; Q8_0 × 256 256 110.8, 512 121.0.  64 of up to 8192:
        // Q4_0 × 128 768 101.5, 1536 91.5; Q8_0 × 256 512 303, 1536 312)
        const int ring = KV_WAVES * KV_STAGES * (q4 ? 36 : 68) * D;
        const int fit = std::min(kv_waves(q4 ? 4 : 8, NB, a.nt), (160 << 10) / ring);
        a.goal = a.n_seq > 1 && fit > 2 ? 1536 : 256 * fit;
    }
    a.ctiles = (int)((cols + per - 1) / per);
    // a prompt among single tokens: work-groups for the rows there are, each of which
    // looks its sequence up, where the bounds alone would start over twice as many
    // (a prompt of 2048 and 63 tokens, 8 heads of 128, Q4_0: 127 µs, 514 without)
    const int64_t tiles = all_cols / per + a.n_seq;
    a.tiles = a.n_seq > 1 && (int64_t)a.n_seq * a.ctiles > 2 * tiles ? (int)tiles : 0;
}

}  // namespace s3e
