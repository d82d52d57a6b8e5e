// k_kv_attn.h — attention over the quantized key/value cache (k_kv_attn_q4.hip
// and k_kv_attn_q8.hip instantiate it for their type).
//
// O = softmax(scale·Q·Kᵀ + mask)·V for the columns (query, head) of one
// sequence and key/value head, in one pass over the keys with a running
// reference and sum.  Both products run transposed on the 16 × 16 × 32 fp16
// MFMA: Sᵀ = K·Qᵀ, then Oᵀ = Vᵀ·Pᵀ, so that a lane's scores (column lane % 16,
// keys 8·(lane / 16) .. + 8 of a chunk of 32) are its operand of the second
// product as they stand, and so are the words of both tensors (k_kv.h) once
// their codes are fp16.
//
// Codes are exact in fp16, and a block of 32 channels is the summed dimension
// of one MFMA, so K's scale multiplies each block sum in fp32: scores carry no
// rounding but q's own.  V's scale varies along the summed dimension and goes
// into the probabilities: P·d is rounded once, to fp16 (fp32 operands: kept as
// a pair hi + lo, as is q, scaled by its row's power of two; over few keys in
// fp16 too, KV_FEW_KEYS).  So that P·d
// stays below fp16's largest and well above its smallest, a column's exponents
// are measured from a reference: its largest score so far plus the exponent of
// the largest scale of V among the keys it has seen; both are taken again, and
// the accumulators scaled, when a score exceeds its by 6 or a scale is over
// twice to four times the largest (P·d is at most 2^7 then, 2^15 in between).
// One reference serves every key and block of channels: of a key or block whose
// scale is 2^-13 of the largest, a pair's low half ends at fp16's 2^-24, 2^-19 of
// the product.
#pragma once

#include "k_kv.h"

namespace s3e {
namespace {

typedef _Float16 kv_h8 __attribute__((ext_vector_type(8)));
typedef _Float16 kv_h4 __attribute__((ext_vector_type(4)));
typedef _Float16 kv_h2 __attribute__((ext_vector_type(2)));
typedef float kv_f4 __attribute__((ext_vector_type(4)));
typedef uint32_t kv_u4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ kv_h2 as_h2(uint32_t x) { return __builtin_bit_cast(kv_h2, x); }

// (x & mask) | magic as one v_and_or_b32: with both constants literal the
// compiler makes two instructions of it, so they are kept in registers.
struct KvMagic {
    uint32_t lo = 0x000f000fu, hi = 0x00f000f0u, e = 0x64006400u;
    __device__ __forceinline__ KvMagic() { __asm__("" : "+v"(lo), "+v"(hi), "+v"(e)); }
};

// The eight codes of a word as fp16, exactly.  A code's bits below the exponent
// of 1024 are 1024 + code (of 64 after the scale, for the nibbles four bits up).
__device__ __forceinline__ kv_h8 word_h8_q4(uint32_t x, const KvMagic &M) {
    const uint32_t y = x >> 8;
    const kv_h2 k = {(_Float16)1032.f, (_Float16)1032.f}, k16 = {(_Float16)-72.f, (_Float16)-72.f},
                s16 = {(_Float16)0.0625f, (_Float16)0.0625f};
    const kv_h2 a = as_h2((x & M.lo) | M.e) - k;
    const kv_h2 b = __builtin_elementwise_fma(as_h2((x & M.hi) | M.e), s16, k16);
    const kv_h2 c = as_h2((y & M.lo) | M.e) - k;
    const kv_h2 d = __builtin_elementwise_fma(as_h2((y & M.hi) | M.e), s16, k16);
    return kv_h8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}
__device__ __forceinline__ kv_h8 word_h8_q8(uint32_t x, uint32_t y) {
    x ^= 0x80808080u;
    y ^= 0x80808080u;
    const kv_h2 k = {(_Float16)1152.f, (_Float16)1152.f};
    // bytes (b, 0x64, b', 0x64): 1024 + 128 + code
    const kv_h2 a = as_h2(__builtin_amdgcn_perm(0x64646464u, x, 0x04010400u)) - k;
    const kv_h2 b = as_h2(__builtin_amdgcn_perm(0x64646464u, x, 0x04030402u)) - k;
    const kv_h2 c = as_h2(__builtin_amdgcn_perm(0x64646464u, y, 0x04010400u)) - k;
    const kv_h2 d = as_h2(__builtin_amdgcn_perm(0x64646464u, y, 0x04030402u)) - k;
    return kv_h8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// K's or V's half of a chunk in LDS, as a wave's lanes read it: their words, and
// the scales of keys 8a .. 8a + 8 of each block.
typedef __attribute__((address_space(3))) const uint8_t *kv_lds;
__device__ __forceinline__ kv_u4 lds16(kv_lds p) { return *(__attribute__((address_space(3))) const kv_u4 *)p; }
__device__ __forceinline__ uint64_t lds8(kv_lds p) { return *(__attribute__((address_space(3))) const uint64_t *)p; }
template <int Q, int NB>
struct KvHalf {
    using C = KvChunk<Q, NB>;
    uint32_t w[C::WORDS * Q / 4];
    __device__ __forceinline__ void load(kv_lds p, int lane) {
#pragma unroll
        for (int i = 0; i < C::PIECES; i++) {
            const kv_lds q = p + i * 1024 + lane * (C::width(i) * Q);
            const int n = C::width(i) * Q / 4, at = i * 4;
            if (n == 4) {
                const kv_u4 x = lds16(q);
                w[at] = x[0], w[at + 1] = x[1], w[at + 2] = x[2], w[at + 3] = x[3];
            } else {
                const uint64_t x = lds8(q);
                w[at] = (uint32_t)x, w[at + 1] = (uint32_t)(x >> 32);
            }
        }
    }
    __device__ __forceinline__ kv_h8 word(int i, const KvMagic &M) const {
        if constexpr (Q == 4) return word_h8_q4(w[i], M);
        else return word_h8_q8(w[2 * i], w[2 * i + 1]);
    }
};
// The scales of block b for the keys of a lane group.
template <int Q, int NB>
__device__ __forceinline__ kv_u4 scales_of(kv_lds half, int b, int ka) { return lds16(half + KvChunk<Q, NB>::CODES + b * 64 + ka * 16); }

__device__ __forceinline__ float max_over_keys(float x) {
    x = fmaxf(x, __shfl_xor(x, 16, 64));
    return fmaxf(x, __shfl_xor(x, 32, 64));
}
__device__ __forceinline__ float sum_over_keys(float x) {
    x += __shfl_xor(x, 16, 64);
    return x + __shfl_xor(x, 32, 64);
}

// P·d of eight keys in fp16, each product rounded once.  (The compiler puts no
// wait states around asm: one before it, behind the exponential that made p,
// and two at its end, before the MFMA that reads the pairs.)
__device__ __forceinline__ kv_u4 scaled_eight(const float *p, kv_u4 d) {
    uint32_t r0, r1, r2, r3;
#define S3E_KV_PAIR(R, P0, P1, D)                                        \
    "v_fma_mixlo_f16 " R ", " P0 ", " D ", 0 op_sel_hi:[0,1,0]\n\t"      \
    "v_fma_mixhi_f16 " R ", " P1 ", " D ", 0 op_sel:[0,1,0] op_sel_hi:[0,1,0]\n\t"
    __asm__("s_nop 0\n\t" S3E_KV_PAIR("%0", "%4", "%5", "%12") S3E_KV_PAIR("%1", "%6", "%7", "%13") S3E_KV_PAIR("%2", "%8", "%9", "%14")
                S3E_KV_PAIR("%3", "%10", "%11", "%15") "s_nop 1"
            : "=&v"(r0), "=&v"(r1), "=&v"(r2), "=&v"(r3)
            : "v"(p[0]), "v"(p[1]), "v"(p[2]), "v"(p[3]), "v"(p[4]), "v"(p[5]), "v"(p[6]), "v"(p[7]), "v"(d[0]), "v"(d[1]), "v"(d[2]), "v"(d[3]));
#undef S3E_KV_PAIR
    return kv_u4{r0, r1, r2, r3};
}

// A mask over the fp16 pair of keys 2j, 2j + 1: zeros for those in `hidden`.
__device__ __forceinline__ uint32_t keep_pair(uint32_t hidden, int j) {
    return (hidden >> 2 * j & 1 ? 0u : 0xffffu) | (hidden >> 2 * j & 2 ? 0u : 0xffff0000u);
}

// The larger of each of two 16-bit numbers.
__device__ __forceinline__ uint32_t max_u16(uint32_t a, uint32_t b) {
    typedef uint16_t u2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u2, a), __builtin_bit_cast(u2, b)));
}

// 2^e as fp16 bits, e ≥ −24 (past fp16: larger than any).
__device__ __forceinline__ uint32_t half_of(int e) { return e >= -14 ? (uint32_t)(e + 15) << 10 : 1u << (e + 24); }

// s_waitcnt's field for at most n vector-memory operations under way.
constexpr int vm_wait(int n) { return (n & 15) | ((n >> 4) << 14) | (7 << 4) | (15 << 8); }

// Of the batch's arrays: read by scalar loads (a vector load would wait behind
// every chunk under way).
typedef __attribute__((address_space(4))) const int32_t c_i32;

// Up to so many keys a row's P·d are pairs in fp16 too: the roundings of few hardly
// average (up to as much again as the output's own).  A work-group decides it by the
// keys its first row sees, so that neither the batch's bounds nor other sequences nor
// a prompt's later rows cost such a row its pairs.  µs rounded once and as pairs for every row: 64 sequences' tokens over up
// to 4096 keys (8 heads of 128, Q4_0) 50 and 61, 4 × 2048 queries (16 heads of 64) 109
// and 148, 4096 × 28 736 at head dim 256 240 and 359; with few keys, where both take the
// loads' and the launch's time, 64 × 512 × 128 at head dim 256 53 and 61.
constexpr int KV_FEW_KEYS = 128;

// What a work-group is to do: its sequence, key/value head, key range and
// first column; `some` where there is anything.
struct KvTask {
    bool some;
    bool few;  // of the work-group's rows the first sees at most KV_FEW_KEYS keys (by length and causal limit)
    int split, kvh, q0, nq, ncols, len, c0, G;
    int before;          // under a causal mask row i sees the first before + i + 1 keys, of len (which may end before them)
    int k_begin, k_end;  // of the tile: keys some of its columns see
};
template <int COLS>
__device__ __forceinline__ KvTask kv_task(const KvAttnArgs &a, int &s) {
    // work-group → (sequence, head, key range) unit and column tile: an XCD (every
    // eighth work-group) takes a contiguous eighth of them, unit by unit, so that
    // the tiles that read the same keys share its L2; whole units tile by tile,
    // the later (under a causal mask longer) ones of every unit first, so that the
    // short ones fill the gaps
    KvTask t;
    t.some = false;
    const int shs = (a.tiles ? 1 : a.n_seq) * a.c.heads, ctiles = a.tiles ? a.tiles : a.ctiles;
    const int units = shs * a.nsplit, total = units * ctiles, per = (total + 7) >> 3;
    const int i = blockIdx.x >> 3, at = (blockIdx.x & 7) * per + i;
    if (i >= per || at >= total) return t;
    int unit, ct;
    if (units % 8 == 0) {
        const int u = units >> 3;
        unit = (i % u) * 8 + (blockIdx.x & 7);  // (dealt out: a long sequence's heads to every XCD)
        ct = ctiles - 1 - i / u;
    } else {
        unit = at / ctiles;
        ct = ctiles - 1 - at % ctiles;
    }
    // (every sequence's first range, then the second of those that have one: the
    // short ones last; sequence by sequence a batch of 64 took 53 µs, so 51)
    t.split = unit / shs;
    const int sh = unit - t.split * shs;
    s = sh / a.c.heads;
    t.kvh = sh - s * a.c.heads;
    const int G = a.nh / a.c.heads;
    if (a.tiles) {
        // tiles of all sequences: s begins at q_start[s]·G / COLS + s, which leaves each
        // at least as many as it has
        const c_i32 *starts = (c_i32 *)a.q_start;
        auto first = [&](int x) { return min(max(starts[x], 0), a.n_tokens) * G / COLS + x; };
        int end = a.n_seq;
        while (end - s > 1) {
            const int mid = (s + end) >> 1;
            if (first(mid) <= ct) s = mid;
            else end = mid;
        }
        ct -= first(s);
        if (ct < 0) return t;
    }
    t.G = G;
    t.q0 = min(max(a.q_start[s], 0), a.n_tokens);
    t.nq = min(max(a.q_start[s + 1], t.q0), a.n_tokens) - t.q0;
    t.ncols = min(t.nq, a.max_q) * t.G;
    t.c0 = ct * COLS;
    if (t.c0 >= t.ncols) return t;
    const int kv = max(a.kv_len[s], 0);
    t.len = (int)min((int64_t)kv, a.max_kv);
    t.before = kv - t.nq;
    const int64_t kb = t.split * a.chunk;
    if (kb >= t.len && t.split > 0) return t;  // past the sequence: no range the joining pass reads
    const int i_first = t.c0 / t.G, i_last = (min(t.c0 + COLS, t.ncols) - 1) / t.G;
    t.few = (a.causal ? min(t.len, t.before + i_first + 1) : t.len) <= KV_FEW_KEYS;
    t.k_begin = (int)kb;
    t.k_end = (int)min((int64_t)(a.causal ? min(t.len, t.before + i_last + 1) : t.len), kb + a.chunk);
    t.some = true;
    return t;
}

// Where a sequence's chunks lie.
struct KvPlaces {
    const c_i32 *pages;
    const uint8_t *base;     // of this head in page 0
    int64_t stride;          // bytes from page to page
    int n_pages, gsh, bytes;
    __device__ __forceinline__ KvPlaces(const KvAttnArgs &a, int s, int kvh, int bytes_)
        : pages((c_i32 *)(a.pages + s * a.pages_ld)), n_pages((int)(a.c.slots >> a.c.page_shift)), gsh(a.c.page_shift - 5), bytes(bytes_) {
        base = a.c.data + ((int64_t)kvh << gsh) * bytes;
        stride = ((int64_t)a.c.heads << gsh) * bytes;
    }
    // chunk g; a page that the cache does not have is read as page 0 and masked
    __device__ __forceinline__ const uint8_t *at(int g, bool &have) const {
        const int p = pages[g >> gsh];
        have = (unsigned)p < (unsigned)n_pages;
        return base + (have ? p : 0) * stride + (g & ((1 << gsh) - 1)) * bytes;
    }
};

// NT · 16 columns of one wave: queries, running sums and output.
// PAIRS: P·d as fp16 pairs too (fp32 operands: always).
template <int NB, bool F32, int NT, bool AHEAD, bool PAIRS>
struct KvColumns {
    static constexpr int D = 32 * NB, W = 2 * NB;  // W: 16-channel tiles of V
    static constexpr int PARTS = F32 ? 2 : 1;      // fp16 operands of an fp32 value
    static constexpr int PP = PAIRS ? 2 : 1;       // of a P·d
    static_assert(PAIRS || !F32, "fp32 is pairs throughout");
    static constexpr int VD = (NB * 16 + 63) / 64;

    int c0, see_all;
    int tok[NT];
    float cs[NT];            // a score's units of log2
    kv_h8 qf[NT][NB][PARTS];
    kv_f4 acc[NT][W];
    float ref[NT], sum[NT];  // reference (log2) and this lane's part of the sum
    float room[NT];          // 15 − e, |scales of V of the keys seen so far| ≤ 2^e
    uint32_t bound;          // fp16 bits of the least 2^e of the wave's columns that have seen a key
    const KvMagic M;

    // This lane's column of each tile: its query, head and limit (past the last
    // column: the last one's again, not stored).
    __device__ __forceinline__ void start(const KvAttnArgs &a, const KvTask &k, int first, int lane) {
        const int col = lane & 15, ka = lane >> 4;
        c0 = first;
        const int i_first = min(c0, k.ncols - 1) / k.G;
        see_all = a.causal ? min(k.len, k.before + i_first + 1) : k.len;
        bound = 0x7fff;
#pragma unroll
        for (int n = 0; n < NT; n++) {
            room[n] = 39.f;
            ref[n] = KV_NONE;
            sum[n] = 0.f;
#pragma unroll
            for (int w = 0; w < W; w++) acc[n][w] = kv_f4{0.f, 0.f, 0.f, 0.f};
            const int c = min(c0 + 16 * n + col, k.ncols - 1), i = c / k.G;
            tok[n] = k.q0 + i;
            const int64_t at = tok[n] * a.q_st + (k.kvh * k.G + (c - i * k.G)) * a.q_sh + 8 * ka;
            if constexpr (!F32) {
                cs[n] = a.scale;
                const _Float16 *q = (const _Float16 *)a.q + at;
#pragma unroll
                for (int b = 0; b < NB; b++) {
                    kv_h8 x;
                    if (a.q_vec) {
                        x = *(const kv_h8 *)(q + 32 * b);
                    } else {
#pragma unroll
                        for (int j = 0; j < 8; j++) x[j] = q[32 * b + j];
                    }
                    qf[n][b][0] = a.sign < 0 ? -x : (a.sign == 0 ? x * (_Float16)0.f : x);
                }
            } else {
                const float *q = (const float *)a.q + at;
                float v[NB][8], top = 0.f;
#pragma unroll
                for (int b = 0; b < NB; b++) {
                    if (a.q_vec) {
                        const float4 x = *(const float4 *)(q + 32 * b), y = *(const float4 *)(q + 32 * b + 4);
                        v[b][0] = x.x, v[b][1] = x.y, v[b][2] = x.z, v[b][3] = x.w;
                        v[b][4] = y.x, v[b][5] = y.y, v[b][6] = y.z, v[b][7] = y.w;
                    } else {
#pragma unroll
                        for (int j = 0; j < 8; j++) v[b][j] = q[32 * b + j];
                    }
#pragma unroll
                    for (int j = 0; j < 8; j++) top = fmaxf(top, fabsf(v[b][j]));
                }
                top = max_over_keys(top);
                // q = 2^e · (hi + lo), the row's largest in [2^14, 2^15): hi + lo is
                // 22 bits of each value down to 2^-14 of that, 2^-39 of it below
                int e = 0;
                if (top > 0.f && top < INFINITY) e = __builtin_amdgcn_frexp_expf(top) - 15;
                // (neither zero nor infinite, which would make −∞ or 0 no number)
                cs[n] = fminf(fmaxf(__builtin_amdgcn_ldexpf(a.scale, e), 1.17549435e-38f), 3.40282347e38f);
#pragma unroll
                for (int b = 0; b < NB; b++)
#pragma unroll
                    for (int j = 0; j < 8; j++) {
                        float x = __builtin_amdgcn_ldexpf(v[b][j], -e) * (float)a.sign;
                        __asm__("" : "+v"(x));  // one value for hi and for lo
                        const _Float16 hi = (_Float16)x;
                        qf[n][b][0][j] = hi;
                        qf[n][b][PARTS - 1][j] = (_Float16)(x - (float)hi);
                    }
            }
        }
    }

    // One chunk: keys 32g .. 32g + 32 (`have`: of a page the cache has).  The
    // operands come by word: kword(i), vword(i) as fp16, kscale(b), vscale(b)
    // the scales of this lane's eight keys, vbits(i) dwords of V's scales, of
    // which each of the chunk's NB · 16 is some lane's.
    template <typename KW, typename KS, typename VW, typename VS, typename VB>
    __device__ __forceinline__ void chunk(const KvAttnArgs &a, const KvTask &k, int g, bool have, int lane, KW kword, KS kscale, VW vword,
                                          VS vscale, VB vbits) {
        // ---- Sᵀ = K·Qᵀ, times K's scales: the next block's words are made
        // between a block's MFMAs and their use.  (The scheduling barriers keep
        // the compiler from making every word before the first MFMA: it would
        // spill.)
        float t[NT][8];
        kv_h8 kw[2] = {kword(0), kword(NB)};
#pragma unroll
        for (int b = 0; b < NB; b++) {
            kv_f4 m[NT][2];
#pragma unroll
            for (int h = 0; h < 2; h++)
#pragma unroll
                for (int n = 0; n < NT; n++) {
                    kv_f4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int i = PARTS - 1; i >= 0; i--) x = __builtin_amdgcn_mfma_f32_16x16x32_f16(kw[h], qf[n][b][i], x, 0, 0, 0);
                    m[n][h] = x;
                }
            const kv_h8 kd = __builtin_bit_cast(kv_h8, kscale(b));
            if (b + 1 < NB) kw[0] = kword(b + 1), kw[1] = kword(NB + b + 1);
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    t[n][j] = __builtin_fmaf((float)kd[j], m[n][j >> 2][j & 3], b == 0 ? 0.f : t[n][j]);
                    __asm__ volatile("" : "+v"(t[n][j]));  // (here, not behind the next branch with every block's sums held)
                }
            __builtin_amdgcn_sched_barrier(0);
        }
        uint32_t vds[VD];
#pragma unroll
        for (int i = 0; i < VD; i++) vds[i] = vbits(i);

        // ---- masked scores −∞; with a mask the scores are in powers of two
        const int key0 = 32 * g + 8 * (lane >> 4);
        const bool special = a.mask || !have || 32 * g + 32 > see_all;
        uint32_t hidden[NT], all = 0;  // bit j: key key0 + j is masked, in a column, in all of the lane's
        bool partly = false;  // a scale that is no number, at a key that some columns see and others do not
        if (special) {
#pragma unroll
            for (int n = 0; n < NT; n++) {
                if (a.mask) {
                    const _Float16 *mp = a.mask + tok[n] * a.mask_ld + key0;
                    float mv[8];
                    if (a.mask_vec && key0 + 8 <= a.max_kv) {
                        const kv_h8 x = *(const kv_h8 *)mp;
#pragma unroll
                        for (int j = 0; j < 8; j++) mv[j] = (float)x[j];
                    } else {
#pragma unroll
                        for (int j = 0; j < 8; j++) mv[j] = (float)mp[min(j, k.len - 1 - key0)];  // (all at once: past the end any value does)
                    }
#pragma unroll
                    for (int j = 0; j < 8; j++)
                        t[n][j] = mv[j] == -INFINITY ? -INFINITY : __builtin_fmaf(mv[j], 1.4426950408889634f, t[n][j] * cs[n]);
                }
                hidden[n] = 0;
                const int lim = a.causal ? min(k.len, k.before + tok[n] - k.q0 + 1) : k.len;
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    if (!have || key0 + j >= lim) t[n][j] = -INFINITY;
                    hidden[n] |= t[n][j] == -INFINITY ? 1u << j : 0u;
                }
            }
            // a masked key's probability is zero, but V's scale there may be no
            // number: zero below where none of this lane's columns sees the key
            all = hidden[0];
            uint32_t any = hidden[0];
#pragma unroll
            for (int n = 1; n < NT; n++) all &= hidden[n], any |= hidden[n];
            if constexpr (NT > 1) {
                uint32_t odd = 0;  // keys with a scale that is no number
#pragma unroll
                for (int b = 0; b < NB; b++) {
                    const kv_u4 d = vscale(b);
#pragma unroll
                    for (int j = 0; j < 4; j++)
                        odd |= ((d[j] & 0x7c00u) == 0x7c00u ? 1u << 2 * j : 0u) | ((d[j] & 0x7c000000u) == 0x7c000000u ? 2u << 2 * j : 0u);
                }
                partly = __builtin_amdgcn_ballot_w64(odd & any & ~all) != 0;
            }
        }

        // ---- the references, where a score or a scale outgrew them
        float mx[NT], c1[NT];
        bool grow = false;
#pragma unroll
        for (int n = 0; n < NT; n++) {
            c1[n] = a.mask ? 1.f : cs[n];
            float x = fmaxf(fmaxf(t[n][0], t[n][1]), t[n][2]);
            x = fmaxf(fmaxf(x, t[n][3]), t[n][4]);
            mx[n] = fmaxf(fmaxf(x, t[n][5]), fmaxf(t[n][6], t[n][7])) * c1[n];
            grow = grow || mx[n] > ref[n] + room[n];
        }
#pragma unroll
        for (int i = 0; i < VD; i++) grow = grow || (vds[i] & 0x7fffu) > bound || ((vds[i] >> 16) & 0x7fffu) > bound;
        if (__builtin_amdgcn_ballot_w64(grow)) {
            // the largest scales of V by key; not those that are no numbers
            uint32_t dk[4] = {0, 0, 0, 0};
#pragma unroll
            for (int b = 0; b < NB; b++) {
                const kv_u4 d = vscale(b);
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const uint32_t x = d[j] & 0x7fff7fffu;
                    dk[j] = max_u16(dk[j], x & ~(((x + 0x04000400u) >> 15 & 0x00010001u) * 0xffffu));
                }
            }
            uint32_t low = 0x7fff;
#pragma unroll
            for (int n = 0; n < NT; n++) {
                // of those of the keys that the column sees
                uint32_t dm = 0;
#pragma unroll
                for (int j = 0; j < 4; j++) dm = max_u16(dm, dk[j] & (special ? keep_pair(hidden[n], j) : ~0u));
                dm = max(dm & 0xffffu, dm >> 16);
                dm = max(dm, (uint32_t)__shfl_xor((int)dm, 16, 64));
                dm = max(dm, (uint32_t)__shfl_xor((int)dm, 32, 64));
                // 2^e ≥ four times every scale (so that it is seldom outgrown): three
                // above the exponent, or of a subnormal its bit length − 22
                const int e = dm >= 0x400u ? (int)(dm >> 10) - 12 : 10 - (dm ? __builtin_clz(dm) : 32);
                // the reference is the largest score + e − 9 (of a column that
                // outgrew its own: what others see changes nothing of it)
                const float best = ref[n] == KV_NONE ? KV_NONE : ref[n] - (6.f - room[n]), up = max_over_keys(mx[n]);
                if (up > ref[n] + room[n] || dm > half_of(15 - (int)room[n])) {
                    const float top = fmaxf(best, up);
                    room[n] = fminf(room[n], (float)(15 - e));
                    const float ref_n = top <= KV_NONE ? KV_NONE : top + (6.f - room[n]);
                    const float alpha = ref_n == ref[n] ? 1.f : __builtin_amdgcn_exp2f(ref[n] - ref_n);
                    ref[n] = ref_n;
                    sum[n] *= alpha;
#pragma unroll
                    for (int w = 0; w < W; w++) acc[n][w] *= alpha;
                }
                if (ref[n] != KV_NONE) low = min(low, half_of(15 - (int)room[n]));
            }
#pragma unroll
            for (int x = 1; x < 16; x *= 2) low = min(low, (uint32_t)__shfl_xor((int)low, x, 64));
            bound = __builtin_amdgcn_readfirstlane(low);
        }

        // ---- probabilities, in units of the reference (AHEAD: V's first words on their way)
        kv_h8 vw[2];
        kv_u4 d;
        if constexpr (AHEAD) vw[0] = vword(0), vw[1] = vword(1), d = vscale(0);
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int j = 0; j < 8; j++) {
                t[n][j] = __builtin_amdgcn_exp2f(__builtin_fmaf(t[n][j], c1[n], -ref[n]));
                sum[n] += t[n][j];
            }

        // ---- Oᵀ += Vᵀ·(P·d)ᵀ, block by block of V's channels (AHEAD: the next block's words before this one's products)
#pragma unroll
        for (int b = 0; b < NB; b++) {
            if constexpr (!AHEAD) vw[0] = vword(2 * b), vw[1] = vword(2 * b + 1), d = vscale(b);
            kv_h8 vn[2];
            kv_u4 dn;
            if (AHEAD && b + 1 < NB) vn[0] = vword(2 * b + 2), vn[1] = vword(2 * b + 3), dn = vscale(b + 1);
            kv_u4 p[NT][PP];
            if (special) {
                uint32_t h = all;
                __asm__ volatile("" : "+v"(h));  // (nothing of this ahead of the branch)
#pragma unroll
                for (int j = 0; j < 4; j++) d[j] &= keep_pair(h, j);
            }
#pragma unroll
            for (int n = 0; n < NT; n++) {
                if constexpr (!PAIRS) {
                    p[n][0] = scaled_eight(t[n], d);
                } else {
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const kv_h2 dd = as_h2(d[j]);
                        float x = t[n][2 * j] * (float)dd[0], y = t[n][2 * j + 1] * (float)dd[1];
                        // one value for hi and for lo: folded into a mixed fma, hi alone would be rounded from the exact product
                        __asm__("" : "+v"(x), "+v"(y));
                        const kv_h2 hi = {(_Float16)x, (_Float16)y};
                        p[n][0][j] = __builtin_bit_cast(uint32_t, hi);
                        p[n][PP - 1][j] = __builtin_bit_cast(uint32_t, kv_h2{(_Float16)(x - (float)hi[0]), (_Float16)(y - (float)hi[1])});
                    }
                }
            }
            if (NT > 1 && partly) {
#pragma unroll
                for (int n = 0; n < NT; n++) {
                    uint32_t h = hidden[n];
                    __asm__ volatile("" : "+v"(h));  // (nothing of this ahead of the branch)
#pragma unroll
                    for (int x = 0; x < PP; x++)
#pragma unroll
                        for (int j = 0; j < 4; j++) p[n][x][j] &= keep_pair(h, j);
                }
            }
#pragma unroll
            for (int w = 2 * b; w < 2 * b + 2; w++)
#pragma unroll
                for (int n = 0; n < NT; n++)
#pragma unroll
                    for (int x = 0; x < PP; x++)
                        acc[n][w] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vw[w & 1], __builtin_bit_cast(kv_h8, p[n][x]), acc[n][w], 0, 0, 0);
            if (AHEAD && b + 1 < NB) vw[0] = vn[0], vw[1] = vn[1], d = dn;
            __builtin_amdgcn_sched_barrier(0);
        }
    }

    __device__ __forceinline__ void join_lanes() {
#pragma unroll
        for (int n = 0; n < NT; n++) sum[n] = sum_over_keys(sum[n]);
    }

    // Accumulators and sums through LDS (`at` by lane, NT · (W · 1024 + 512) bytes
    // of a wave) into another wave's of the same columns.
    __device__ __forceinline__ void give(uint8_t *at, int lane) const {
#pragma unroll
        for (int n = 0; n < NT; n++) {
#pragma unroll
            for (int w = 0; w < W; w++) *(kv_f4 *)(at + (n * W + w) * 1024) = acc[n][w];
            *(float2 *)(at - lane * 8 + NT * W * 1024 + n * 512) = make_float2(ref[n], sum[n]);
        }
    }
    __device__ __forceinline__ void take(const uint8_t *at, int lane) {
#pragma unroll
        for (int n = 0; n < NT; n++) {
            const float2 o = *(const float2 *)(at - lane * 8 + NT * W * 1024 + n * 512);
            const float top = fmaxf(ref[n], o.x);
            const float wa = ref[n] == top ? 1.f : __builtin_amdgcn_exp2f(ref[n] - top);
            const float wb = o.x == top ? 1.f : __builtin_amdgcn_exp2f(o.x - top);
            ref[n] = top;
            sum[n] = sum[n] * wa + o.y * wb;
#pragma unroll
            for (int w = 0; w < W; w++) acc[n][w] = acc[n][w] * wa + *(const kv_f4 *)(at + (n * W + w) * 1024) * wb;
        }
    }

    // The columns' rows of o, or their part of a key range.
    __device__ __forceinline__ void store(const KvAttnArgs &a, const KvTask &k, int lane) const {
        const int col = lane & 15, ka = lane >> 4;
#pragma unroll
        for (int n = 0; n < NT; n++) {
            if (c0 + 16 * n + col >= k.ncols) continue;
            // (tok = q0 + c / G, head = kvh·G + c % G)
            const int64_t row = (int64_t)tok[n] * a.nh + k.kvh * k.G + (c0 + 16 * n + col - (tok[n] - k.q0) * k.G);
            if (a.nsplit > 1) {
                const int64_t at = (int64_t)k.split * a.n_tokens * a.nh + row;
                float *o = a.part_o + at * D + 4 * ka;
#pragma unroll
                for (int w = 0; w < W; w++) *(kv_f4 *)(o + 16 * w) = acc[n][w];
                if (ka == 0) *(float2 *)(a.part_ml + at * 2) = make_float2(ref[n], sum[n]);
                continue;
            }
            const float inv = sum[n] == 0.f ? 0.f : 1.0f / sum[n];  // no key at all: zeros
            if constexpr (F32) {
                float *o = (float *)a.o + row * D + 4 * ka;
#pragma unroll
                for (int w = 0; w < W; w++) *(kv_f4 *)(o + 16 * w) = acc[n][w] * inv;
            } else {
                _Float16 *o = (_Float16 *)a.o + row * D + 4 * ka;
#pragma unroll
                for (int w = 0; w < W; w++) {
                    const kv_f4 x = acc[n][w] * inv;
                    *(kv_h4 *)(o + 16 * w) = kv_h4{(_Float16)x[0], (_Float16)x[1], (_Float16)x[2], (_Float16)x[3]};
                }
            }
        }
    }
};

// ---- rings of chunks -----------------------------------------------------------
// A work-group takes NT · 16 columns against one range of keys; its four waves
// take chunks in turn and are joined in LDS.  Each wave keeps a ring of two
// chunks in LDS, loaded straight into it: while one is worked on the next is
// under way without holding registers, so that two to four work-groups share a
// CU (Q8_0 at head dim 256: one) and no wave waits for another before the end.
// One token of 64 sequences of up to 4096 keys (8 heads of 128, 32 query heads,
// Q4_0, 174 MB) takes 51 µs with the joining pass, 3.4 TB/s; one of 131 072 keys
// (151 MB) 41 µs, 3.7 TB/s.  Vector instructions, half of them the conversion of
// codes to fp16, are busy 55 % of the cycles there and wait on one another, on
// the longest range and on memory for the rest.  4 × 2048 causal queries over up
// to 2592 keys, 16 heads of 64: 109 µs, 318 TFLOP/s, of 64 that the 243 vector
// and matrix instructions of 32 keys and 32 columns take to issue.
constexpr int KV_STAGES = 2, KV_WAVES = 4;
// Waves a SIMD is to hold: at least two, so that no MFMA result takes the way
// through an accumulation register; more where the registers suffice.  (The rings
// of Q8_0 at head dim 256, 139 KB, leave room for one all the same, and 68 to 72
// accumulation registers are used there.)
constexpr int kv_waves(int Q, int NB, int NT) { return NT > 1 || NB == 8 || Q * NB == 32 ? 2 : (NB <= 2 ? 4 : 3); }
// The waves a SIMD that k_kv_attn, which holds both forms of fp16's P·d, is compiled
// for: the pairs' form would take two column tiles at head dim 64 past 128 registers
// and the prompts from 109 to 118 µs; it has 6 or 7 of them in memory instead.
constexpr int kv_bound(int Q, int NB, bool F32, int NT) { return !F32 && NT > 1 && NB == 2 ? 4 : kv_waves(Q, NB, NT); }

template <int Q, int NB, bool F32, int NT, bool PAIRS>
__device__ __forceinline__ void kv_rings(const KvAttnArgs &a, const KvTask &k, int s, uint8_t *smem) {
    using C = KvChunk<Q, NB>;
    using Cols = KvColumns<NB, F32, NT, false, PAIRS>;
    constexpr int W = Cols::W, WAVES = KV_WAVES;
    constexpr int LD = (C::BYTES + 1023) / 1024;  // 1 KB loads of a chunk

    const int tid = threadIdx.x, lane = tid & 63, ka = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const KvPlaces places(a, s, k.kvh, C::BYTES);

    const int g_end = (k.k_end + 31) >> 5;
    int g = (k.k_begin >> 5) + wave;
    uint8_t *const ring = smem + wave * (KV_STAGES * C::BYTES);
    // a chunk into a slot of the ring: LD loads, the last of fewer lanes
    auto fetch = [&](const uint8_t *p, int slot) {
#pragma unroll
        for (int i = 0; i < LD; i++)
            if (C::BYTES - i * 1024 >= 1024 || lane * 16 < C::BYTES - i * 1024)
                __builtin_amdgcn_global_load_lds((const void *)(p + i * 1024 + lane * 16),
                                                 (__attribute__((address_space(3))) void *)(ring + slot * C::BYTES + i * 1024), 16, 0, 0);
    };
    bool has[KV_STAGES];  // whether the cache has the page of the chunk in a slot
    const bool any = k.k_begin < k.k_end && g < g_end;
    if (any) {
#pragma unroll
        for (int i = 0; i < KV_STAGES; i++) {
            has[i] = true;
            if (g + WAVES * i < g_end) fetch(places.at(g + WAVES * i, has[i]), i);
        }
    }
    Cols cols;
    cols.start(a, k, k.c0, lane);
    if (any) {
        int slot = 0;
        while (true) {
            // this chunk has arrived when no more loads are under way than the next one's
            if (g + WAVES < g_end) __builtin_amdgcn_s_waitcnt(vm_wait(LD));
            else __builtin_amdgcn_s_waitcnt(vm_wait(0));
            __asm__ volatile("" ::: "memory");
            const kv_lds kh = (kv_lds)(ring + slot * C::BYTES), vh = kh + C::HALF;
            const bool have = has[0];
            const bool more = g + WAVES * KV_STAGES < g_end;
            bool have_n = true;
            const uint8_t *pn = places.at(more ? g + WAVES * KV_STAGES : g, have_n);
            KvHalf<Q, NB> K, V;
            K.load(kh, lane);
            cols.chunk(
                a, k, g, have, lane, [&](int i) { return K.word(i, cols.M); },
                [&](int b) { return scales_of<Q, NB>(kh, b, ka); },
                [&](int i) {
                    if (i == 0) V.load(vh, lane);
                    return V.word(i, cols.M);
                },
                [&](int b) { return scales_of<Q, NB>(vh, b, ka); },
                [&](int i) {
                    return *(__attribute__((address_space(3))) const uint32_t *)(vh + C::CODES + ((lane + 64 * i) % (NB * 16)) * 4);
                });
            if (g + WAVES >= g_end) break;
            // the slot's words are all in registers: the next chunk may come
            if (more) fetch(pn, slot);
#pragma unroll
            for (int i = 0; i + 1 < KV_STAGES; i++) has[i] = has[i + 1];
            has[KV_STAGES - 1] = have_n;
            g += WAVES;
            slot = slot + 1 < KV_STAGES ? slot + 1 : 0;
        }
    }
    cols.join_lanes();

    // the rings are done with: the memory joins the waves, 2 and 3 into 0 and 1, then 1 into 0
    constexpr int ONE = NT * (W * 1024 + 512);
    uint8_t *const at = smem + lane * 16;
    __syncthreads();
    if (wave >= 2) cols.give(at + (wave - 2) * ONE, lane);
    __syncthreads();
    if (wave < 2) cols.take(at + wave * ONE, lane);
    __syncthreads();
    if (wave == 1) cols.give(at, lane);
    __syncthreads();
    if (wave != 0) return;
    cols.take(at, lane);
    cols.store(a, k, lane);
}

template <int Q, int NB, bool F32, int NT>
__global__ __launch_bounds__(64 * KV_WAVES, kv_bound(Q, NB, F32, NT)) void k_kv_attn(KvAttnArgs a) {
    // the rings; at the end the accumulators of two waves
    constexpr int RING = KV_WAVES * KV_STAGES * KvChunk<Q, NB>::BYTES, JOIN = 2 * NT * (2 * NB * 1024 + 512);
    __shared__ __attribute__((aligned(16))) uint8_t smem[RING > JOIN ? RING : JOIN];
    int s;
    const KvTask k = kv_task<16 * NT>(a, s);
    if (!k.some) return;
    if (F32 || k.few) kv_rings<Q, NB, F32, NT, true>(a, k, s, smem);
    else if constexpr (!F32) kv_rings<Q, NB, F32, NT, false>(a, k, s, smem);
}

// ---- many columns at head dim 256: bound by vector instructions and LDS -------
// There a wave's registers hold no second column tile to share a chunk's
// conversion with, and the first kernel's rings leave a CU one or two
// work-groups.  Here the waves hold 16 columns each against the same chunks,
// whose words are converted to fp16 once for all of them: each converts some
// while chunks before are worked on, into one of four buffers of whole MFMA
// operands (16 bytes a lane and word, in the order of lanes, so neither side
// has bank conflicts).  One barrier every two chunks.  fp16 takes 12 waves in 168
// registers, fp32 8 in 256.  4096 queries over 28 736 keys of Q8_0: 228 µs and 12
// for the joining pass, 500 TFLOP/s.  A wave reads 32 KB of operands a chunk for
// its 16 columns, 96 µs at LDS's rate, beside 95 µs of vector instructions and
// 48 of MFMAs; the rest is three waves a SIMD waiting on LDS.  (8 waves: 273 µs; 8
// of two column tiles, half the LDS reads: 299, with 93 registers in memory.)
constexpr int KV_TILE_NB = 8;
constexpr int kv_tile_waves(bool F32) { return F32 ? 8 : 12; }
constexpr int kv_tile_cols(bool F32) { return 16 * kv_tile_waves(F32); }

// bytes of a buffer: K, V operands, K, V scales
template <int Q>
constexpr int KV_TILE_BUF = 2 * KvChunk<Q, KV_TILE_NB>::WORDS * 1024 + 2 * KvChunk<Q, KV_TILE_NB>::SCALES;

template <int Q, bool F32, bool PAIRS>
__device__ __forceinline__ void kv_tile(const KvAttnArgs &a, const KvTask &k, int s, uint8_t *smem) {
    constexpr int NB = KV_TILE_NB, WAVES = kv_tile_waves(F32);
    using C = KvChunk<Q, NB>;
    using Cols = KvColumns<NB, F32, 1, true, PAIRS>;
    constexpr int HALF = C::WORDS * 1024, BUF = KV_TILE_BUF<Q>;

    const int tid = threadIdx.x, lane = tid & 63, ka = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const KvPlaces places(a, s, k.kvh, C::BYTES);

    // pieces of K and V this wave converts; the scales are the last wave's (of fewer pieces)
    constexpr int P2 = 2 * C::PIECES, PW = (P2 + WAVES - 1) / WAVES;
    static_assert(8 * NB == 64 && C::WORDS % C::PER == 0, "16 bytes of scales a lane, whole pieces");
    uint4 raw[PW], rawd;
    auto fetch = [&](const uint8_t *p) {
#pragma unroll
        for (int i = 0; i < PW; i++) {
            const int u = wave + i * WAVES;
            if (u < P2) raw[i] = gload16(p + (u / C::PIECES) * C::HALF + u % C::PIECES * 1024 + lane * 16);
        }
        if (wave == WAVES - 1) rawd = gload16(p + C::CODES + (lane < 32 ? lane * 16 : C::HALF + (lane - 32) * 16));
    };
    const KvMagic M;
    auto convert = [&](uint8_t *buf) {
#pragma unroll
        for (int i = 0; i < PW; i++) {
            const int u = wave + i * WAVES;
            if (u >= P2) continue;
            uint8_t *o = buf + u * (C::PER * 1024) + lane * 16;
            const uint32_t x[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
#pragma unroll
            for (int w = 0; w < C::PER; w++) {
                kv_h8 h;
                if constexpr (Q == 4) h = word_h8_q4(x[w], M);
                else h = word_h8_q8(x[2 * w], x[2 * w + 1]);
                *(kv_h8 *)(o + w * 1024) = h;
            }
        }
        if (wave == WAVES - 1) *(uint4 *)(buf + 2 * HALF + lane * 16) = rawd;
    };

    const int g_end = (k.k_end + 31) >> 5;
    const int g0 = k.k_begin >> 5, n = k.k_begin < k.k_end ? g_end - g0 : 0;
    // the pages of chunks i, i + 1, i + 2
    bool have = true, have_1 = true, have_2 = true;
    if (n > 0) fetch(places.at(g0, have));
    Cols cols;
    cols.start(a, k, k.c0 + wave * 16, lane);
    // this wave's own columns see no key from here on
    const int i_last = (min(cols.c0 + 16, k.ncols) - 1) / k.G;
    const int see_any = cols.c0 >= k.ncols ? 0 : min(k.k_end, a.causal ? k.before + i_last + 1 : k.len);
    if (n > 0) {
        convert(smem);
        if (n > 1) {
            fetch(places.at(g0 + 1, have_1));
            convert(smem + BUF);
        }
        if (n > 2) fetch(places.at(g0 + 2, have_2));
        __syncthreads();
        for (int i = 0; i < n; i++) {
            const kv_lds kb = (kv_lds)(smem + (i & 3) * BUF), vb = kb + HALF, kd = kb + 2 * HALF, vd = kd + C::SCALES;
            bool have_3 = true;
            if (i + 2 < n) {
                convert(smem + (i + 2 & 3) * BUF);
                if (i + 3 < n) fetch(places.at(g0 + i + 3, have_3));
            }
            if (32 * (g0 + i) < see_any)
                cols.chunk(
                    a, k, g0 + i, have, lane, [&](int w) { return __builtin_bit_cast(kv_h8, lds16(kb + w * 1024 + lane * 16)); },
                    [&](int b) { return lds16(kd + b * 64 + ka * 16); },
                    [&](int w) { return __builtin_bit_cast(kv_h8, lds16(vb + w * 1024 + lane * 16)); },
                    [&](int b) { return lds16(vd + b * 64 + ka * 16); },
                    [&](int w) { return *(__attribute__((address_space(3))) const uint32_t *)(vd + (lane + 64 * w) * 4); });
            // chunk i + 2 takes the buffer of i − 2: apart by a barrier, as i + 2 and its conversion are
            if (i & 1) __syncthreads();
            have = have_1, have_1 = have_2, have_2 = have_3;
        }
    }
    cols.join_lanes();
    if (cols.c0 < k.ncols) cols.store(a, k, lane);
}

template <int Q, bool F32>
__global__ __launch_bounds__(64 * kv_tile_waves(F32), kv_tile_waves(F32) / 4) void k_kv_attn_tile(KvAttnArgs a) {
    __shared__ __attribute__((aligned(16))) uint8_t smem[4 * KV_TILE_BUF<Q>];
    int s;
    const KvTask k = kv_task<kv_tile_cols(F32)>(a, s);
    if (!k.some) return;
    if (F32 || k.few) kv_tile<Q, F32, true>(a, k, s, smem);
    else if constexpr (!F32) kv_tile<Q, F32, false>(a, k, s, smem);
}

// Column tiles a wave of the first kernel holds where there are more than 16 columns.
constexpr int kv_most_tiles(int NB) { return NB == 8 ? 1 : 2; }

template <int Q>
hipError_t launch_kv_attn(const KvAttnArgs &a, bool f32, hipStream_t st) {
    const int64_t grid = ((int64_t)a.c.heads * a.nsplit * (a.tiles ? a.tiles : (int64_t)a.n_seq * a.ctiles) + 7) / 8 * 8;
    if (grid > INT32_MAX) return hipErrorInvalidValue;
    auto go = [&](auto nb, auto f) {
        constexpr int NB = nb(), MOST = kv_most_tiles(NB);
        const dim3 g((unsigned)grid);
        if (a.tile) {
            if constexpr (NB == KV_TILE_NB) hipLaunchKernelGGL((k_kv_attn_tile<Q, f()>), g, dim3(64 * kv_tile_waves(f())), 0, st, a);
            else return hipErrorInvalidValue;
        } else if (a.nt == 1 || a.nt == MOST) {
            if (a.nt == 1) hipLaunchKernelGGL((k_kv_attn<Q, NB, f(), 1>), g, dim3(64 * KV_WAVES), 0, st, a);
            else hipLaunchKernelGGL((k_kv_attn<Q, NB, f(), MOST>), g, dim3(64 * KV_WAVES), 0, st, a);
        } else {
            return hipErrorInvalidValue;
        }
        return hipGetLastError();
    };
    auto by = [&](auto nb) { return f32 ? go(nb, std::true_type{}) : go(nb, std::false_type{}); };
    switch (a.c.D) {
        case 32: return by(std::integral_constant<int, 1>{});
        case 64: return by(std::integral_constant<int, 2>{});
        case 96: return by(std::integral_constant<int, 3>{});
        case 128: return by(std::integral_constant<int, 4>{});
        case 256: return by(std::integral_constant<int, 8>{});
        default: return hipErrorInvalidValue;
    }
}

}  // namespace
}  // namespace s3e
