// k_kv.h — the quantized key/value cache's layout in memory and its kernels'
// arguments (k_kv.hip: writing, reading back, joining partial results;
// k_kv_attn.h: attention over it).
#pragma once

#include "s3e_internal.h"

namespace s3e {

// A cache is pages of P tokens; a page holds, for each key/value head, P/32
// chunks of 32 tokens.  A chunk of D = 32·NB channels is
//   K words | K scales | V words | V scales.
// A word is eight codes (4 bytes of Q4_0 nibbles, 8 bytes of Q8_0): what one
// lane feeds to one 16 × 16 × 32 fp16 MFMA as eight consecutive values of the
// summed dimension, so attention takes words as they lie, without shuffles.  K:
// key r = 8a + 4t + i of the chunk (a, i < 4, t < 2) and channels 32b + 8g + j
// (j < 8) are word t·NB + b of lane 16g + 4a + i.  V: channel 16w + m and keys
// 8g + j are word w of lane 16g + m.  Either way a lane has 2·NB words; they
// lie in pieces of up to 16 bytes a lane, all 64 lanes of a piece together, so
// that a wave's load of a piece is contiguous. Code j of a Q4_0 word is nibble
// (j >> 1) + 4·(j & 1) (two codes of one shift then sit 16 bits apart, as an
// fp16 pair needs them), of a Q8_0 word byte j.
// Scales are fp16 [NB][32 keys].
template <int Q, int NB>
struct KvChunk {
    static constexpr int WB = Q;                   // bytes of a word
    static constexpr int PER = 16 / WB;            // words of a whole piece
    static constexpr int WORDS = 2 * NB;           // words of a lane
    static constexpr int PIECES = (WORDS + PER - 1) / PER;
    static constexpr int CODES = 64 * WORDS * WB;  // bytes of the K (or V) words
    static constexpr int SCALES = NB * 64;         // bytes of the K (or V) scales
    static constexpr int HALF = CODES + SCALES;    // K or V
    static constexpr int BYTES = 2 * HALF;
    // words of a lane in piece p, and a word's byte offset
    __host__ __device__ static constexpr int width(int p) { return WORDS - p * PER < PER ? WORDS - p * PER : PER; }
    __host__ __device__ static constexpr int word(int w, int lane) {
        const int p = w / PER;
        return p * PER * 64 * WB + (lane * width(p) + w % PER) * WB;
    }
};

struct KvCache {
    uint8_t *data = nullptr;
    int64_t slots = 0;      // n_pages · page
    int type = 0;           // S3E_TYPE_Q4_0 or S3E_TYPE_Q8_0
    int heads = 0, D = 0, page_shift = 0;
};

// K and V rows by element strides (token, head), fp16 or f32; tensor 0 is K.
struct KvWriteArgs {
    const void *x[2] = {nullptr, nullptr};
    int64_t st[2] = {0, 0}, sh[2] = {0, 0};
    int vec[2] = {0, 0};    // rows allow 16-byte loads
    const int32_t *slots = nullptr;
    int n = 0;
    KvCache c;
};
hipError_t launch_kv_write(const KvWriteArgs &a, bool f32, hipStream_t st);
// y: [n][heads][D], null: left out
struct KvReadArgs {
    void *y[2] = {nullptr, nullptr};
    const int32_t *slots = nullptr;
    int n = 0;
    KvCache c;
};
hipError_t launch_kv_read(const KvReadArgs &a, bool f32, hipStream_t st);

struct KvAttnArgs {
    KvCache c;
    const void *q = nullptr;
    int64_t q_st = 0, q_sh = 0;  // element strides: token, head
    int q_vec = 0;
    const int32_t *q_start = nullptr, *kv_len = nullptr, *pages = nullptr;
    int64_t pages_ld = 0;
    const _Float16 *mask = nullptr;
    int64_t mask_ld = 0;
    int mask_vec = 0;
    void *o = nullptr;
    float scale = 0.f;      // |scale| · log2(e), of a zero scale 1
    int sign = 1;           // the scale's: −1, 0 or 1
    int causal = 0;
    int n_seq = 0, n_tokens = 0, max_q = 0, nh = 0;
    int64_t max_kv = 0;
    int tile = 0;           // the kernel for many columns
    int nt = 1;             // column tiles of 16 a wave
    int ctiles = 1;         // work-groups over the columns of a sequence and head
    // > 0: work-groups over the columns of all sequences and one head, found by
    // q_start, instead of ctiles for each
    int tiles = 0;
    int goal = 0;           // work-groups to aim at with the split over keys
    // keys a work-group takes (a multiple of 128) and the number of such
    // ranges; nsplit > 1: unnormalised outputs to part_o [nsplit][tokens][nh][D]
    // and (reference, sum) to part_ml [nsplit][tokens][nh][2]
    int64_t chunk = 0;
    int nsplit = 1;
    float *part_o = nullptr, *part_ml = nullptr;
};
hipError_t launch_kv_attn_q4(const KvAttnArgs &a, bool f32, hipStream_t st);
hipError_t launch_kv_attn_q8(const KvAttnArgs &a, bool f32, hipStream_t st);
hipError_t launch_kv_combine(const KvAttnArgs &a, bool f32, hipStream_t st);
// The kernel, column tiles and work-groups over the columns where a sequence and
// head have up to `cols` of them, all sequences `all_cols`.
void kv_attn_columns(KvAttnArgs &a, int D, bool f32, int64_t cols, int64_t all_cols);

// The reference exponent of a column that has seen no key.
constexpr float KV_NONE = -3.0e38f;

}  // namespace s3e
