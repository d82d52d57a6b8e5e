// k_kv_attn.h — attention over the quantized key/value cache (k_kv_attn_q4.hip
// and k_kv_attn_q8.hip instantiate it for their type).
//
// O = softmax(scale·Q·Kᵀ + mask)·V for the columns (query, head) of one
// sequence and key/value head, in one pass over the keys with a running
// reference and sum.  Both products run transposed on the 16 × 16 × 32 fp16
// MFMA: Sᵀ = K·Qᵀ, then Oᵀ = Vᵀ·Pᵀ, so that a lane's scores (column lane % 16,
// keys 8·(lane / 16) .. + 8 of a chunk of 32) are its operand of the second
// product as they stand, and the words of both tensors (k_kv.h) go from
// memory to the matrix core through registers alone.
//
// Codes are exact in fp16, and a block of 32 channels is the summed dimension
// of one MFMA, so K's scale multiplies each block sum in fp32: scores carry no
// rounding but q's own.  V's scale varies along the summed dimension and goes
// into the probabilities: P·d is rounded once, to fp16 (fp32 operands: kept as
// a pair hi + lo, as is q, scaled by its row's power of two).  So that P·d
// stays below fp16's largest and well above its smallest, a wave measures a
// column's exponents from a reference: the column's largest score so far plus
// the exponent of the largest scale of V so far; both are taken again, and the
// accumulators scaled, when a score exceeds its by 8 or a scale exceeds its
// own (P·d ≤ 2^15 in between).
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

// K's or V's half of a chunk as one wave holds it: its words, and the scales
// of keys 8a .. 8a + 8 of each block.
template <int Q, int NB>
struct KvHalf {
    using C = KvChunk<Q, NB>;
    uint32_t w[C::WORDS * Q / 4];
    kv_h8 d[NB];
    __device__ __forceinline__ void load(const uint8_t *p, int lane) {
#pragma unroll
        for (int i = 0; i < C::PIECES; i++) {
            const uint8_t *q = p + i * 1024 + lane * (C::width(i) * Q);
            const int n = C::width(i) * Q / 4, at = i * 4;
            if (n == 4) {
                const uint4 x = gload16(q);
                w[at] = x.x, w[at + 1] = x.y, w[at + 2] = x.z, w[at + 3] = x.w;
            } else {
                const uint2 x = gload8(q);
                w[at] = x.x, w[at + 1] = x.y;
            }
        }
#pragma unroll
        for (int b = 0; b < NB; b++) {
            const uint4 x = gload16(p + C::CODES + b * 64 + (lane >> 4) * 16);
            d[b] = __builtin_bit_cast(kv_h8, kv_u4{x.x, x.y, x.z, x.w});
        }
    }
    __device__ __forceinline__ kv_h8 word(int i, const KvMagic &M) const {
        if constexpr (Q == 4) return word_h8_q4(w[i], M);
        else return word_h8_q8(w[2 * i], w[2 * i + 1]);
    }
};

__device__ __forceinline__ float max_over_keys(float x) {
    x = fmaxf(x, __shfl_xor(x, 16, 64));
    return fmaxf(x, __shfl_xor(x, 32, 64));
}
__device__ __forceinline__ float sum_over_keys(float x) {
    x += __shfl_xor(x, 16, 64);
    return x + __shfl_xor(x, 32, 64);
}

// Waves a SIMD is to hold: at least two, so that no MFMA result takes the way
// through an accumulation register; more where the registers suffice.
constexpr int kv_waves(int Q, int NB, bool F32, int NT) {
    if (NT > 1 || NB == 8) return 2;
    return NB <= 2 ? 4 : 3;
}

// P·d of two neighbouring keys as an fp16 pair, each product rounded once.
__device__ __forceinline__ uint32_t scaled_pair(float p0, float p1, uint32_t d) {
    uint32_t r;
    __asm__("v_fma_mixlo_f16 %0, %1, %3, 0 op_sel_hi:[0,1,0]\n\tv_fma_mixhi_f16 %0, %2, %3, 0 op_sel:[0,1,0] op_sel_hi:[0,1,0]"
            : "=&v"(r) : "v"(p0), "v"(p1), "v"(d));
    return r;
}

// A mask over the fp16 pair of keys 2j, 2j + 1: zeros for those in `hidden`.
__device__ __forceinline__ uint32_t keep_pair(uint32_t hidden, int j) {
    return (hidden >> 2 * j & 1 ? 0u : 0xffffu) | (hidden >> 2 * j & 2 ? 0u : 0xffff0000u);
}

// One work-group: NT · 16 columns of a sequence and key/value head against one
// range of its keys; its four waves take chunks in turn and are joined in LDS.
// A chunk's K words for the wave's next turn are loaded as soon as the scores
// are done with these, its V words behind the second product.
template <int Q, int NB, bool F32, int NT>
__global__ __launch_bounds__(256, kv_waves(Q, NB, F32, NT)) void k_kv_attn(KvAttnArgs a) {
    using C = KvChunk<Q, NB>;
    constexpr int D = 32 * NB, W = 2 * NB;  // W: 16-channel tiles of V
    constexpr int PARTS = F32 ? 2 : 1;      // fp16 operands of an fp32 value
    __shared__ kv_f4 lds[2][NT * W][64];
    __shared__ float lds_ml[2][NT][2][64];

    const int tid = threadIdx.x, lane = tid & 63, col = lane & 15, ka = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    // work-group → (sequence, head, key range), column tile: those that read the
    // same keys on one XCD, and the later (under a causal mask longer) tiles first
    const int units = a.n_seq * a.c.heads * a.nsplit;
    int unit, ct;
    {
        const int id = blockIdx.x;
        if (units >= 8) {
            const int i = id >> 3;
            unit = (i / a.ctiles) * 8 + (id & 7);
            ct = a.ctiles - 1 - i % a.ctiles;
        } else {
            unit = id % units;
            ct = a.ctiles - 1 - id / units;
        }
    }
    if (unit >= units) return;
    const int split = unit % a.nsplit, sh = unit / a.nsplit;
    const int s = sh / a.c.heads, kvh = sh - s * a.c.heads;
    const int G = a.nh / a.c.heads;
    const int q0 = min(max(a.q_start[s], 0), a.n_tokens), q1 = min(max(a.q_start[s + 1], q0), a.n_tokens);
    const int nq = q1 - q0, ncols = min(nq, a.max_q) * G, c0 = ct * (16 * NT);
    if (c0 >= ncols) return;
    const int len = (int)min((int64_t)max(a.kv_len[s], 0), a.max_kv);
    // the keys that some column of the tile sees, and those that all of them see
    const int i_first = c0 / G, i_last = (min(c0 + 16 * NT, ncols) - 1) / G;
    const int see_all = a.causal ? min(len, len - nq + i_first + 1) : len;
    const int see_any = a.causal ? min(len, len - nq + i_last + 1) : len;
    const int64_t kb = split * a.chunk;
    if (kb >= len && split > 0) return;  // past the sequence: no range the joining pass reads
    const int k_begin = (int)kb, k_end = (int)min((int64_t)see_any, kb + a.chunk);

    // this lane's column of each tile: its query, head and limit (past the
    // last column: the last one's again, not stored)
    int lim[NT], tok[NT], head[NT];
    float cs[NT];
    kv_h8 qf[NT][NB][PARTS];
#pragma unroll
    for (int n = 0; n < NT; n++) {
        const int c = c0 + 16 * n + col, i = min(c, ncols - 1) / G;
        tok[n] = q0 + i;
        head[n] = kvh * G + (min(c, ncols - 1) - i * G);
        lim[n] = a.causal ? min(len, len - nq + i + 1) : len;
        cs[n] = a.scale;
        const int64_t at = tok[n] * a.q_st + head[n] * a.q_sh + 8 * ka;
        if constexpr (!F32) {
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
                qf[n][b][0] = a.neg ? -x : x;
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
            cs[n] = __builtin_amdgcn_ldexpf(a.scale, e);
#pragma unroll
            for (int b = 0; b < NB; b++)
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    float x = __builtin_amdgcn_ldexpf(v[b][j], -e);
                    if (a.neg) x = -x;
                    __asm__("" : "+v"(x));  // one value for hi and for lo
                    const _Float16 hi = (_Float16)x;
                    qf[n][b][0][j] = hi;
                    qf[n][b][PARTS - 1][j] = (_Float16)(x - (float)hi);
                }
        }
    }

    kv_f4 acc[NT][W];
    float ref[NT], sum[NT];  // reference (log2) and this lane's part of the sum
#pragma unroll
    for (int n = 0; n < NT; n++) {
        ref[n] = KV_NONE;
        sum[n] = 0.f;
#pragma unroll
        for (int w = 0; w < W; w++) acc[n][w] = kv_f4{0.f, 0.f, 0.f, 0.f};
    }
    int ed = -24;  // |scales of V so far| ≤ 2^ed

    const KvMagic M;
    const int gsh = a.c.page_shift - 5;
    const int64_t cpp = 1 << gsh;  // chunks of a page and head
    const int32_t *pages = a.pages + s * a.pages_ld;
    const int64_t n_pages = a.c.slots >> a.c.page_shift;
    // a page that the cache does not have is read as page 0 and masked
    auto place = [&](int g, bool &have) -> const uint8_t * {
        const int64_t p = pages[g >> gsh];
        have = p >= 0 && p < n_pages;
        return a.c.data + (((have ? p : 0) * a.c.heads + kvh) * cpp + (g & (cpp - 1))) * C::BYTES;
    };

    const int g_end = (k_end + 31) >> 5;
    int g = (k_begin >> 5) + wave;
    KvHalf<Q, NB> K, V;
    // V's scales once more, a dword a lane (each of the chunk's NB · 16 is some lane's)
    constexpr int VD = (NB * 16 + 63) / 64;
    uint32_t vds[VD];
    bool have = true;
    if (k_begin < k_end && g < g_end) {
        const uint8_t *p = place(g, have);
        K.load(p, lane);
        V.load(p + C::HALF, lane);
#pragma unroll
        for (int i = 0; i < VD; i++)
            vds[i] = *(const uint32_t *)(p + C::HALF + C::CODES + ((lane + 64 * i) % (NB * 16)) * 4);
        while (true) {
            const int gn = g + 4;
            const bool more = gn < g_end;
            bool have_n = have;
            const uint8_t *pn = place(more ? gn : g, have_n);

            // ---- Sᵀ = K·Qᵀ, times K's scales: a block's sums are scaled behind
            // the next block's MFMAs.  (The scheduling barriers keep the
            // compiler from converting every word, or loading the next chunk's,
            // before the first MFMA: it would spill.)
            float t[NT][8];
            kv_f4 m[2][NT][2];
#pragma unroll
            for (int b = 0; b <= NB; b++) {
                if (b < NB) {
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        const kv_h8 kw = K.word(h * NB + b, M);
#pragma unroll
                        for (int n = 0; n < NT; n++) {
                            kv_f4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                            for (int i = PARTS - 1; i >= 0; i--) x = __builtin_amdgcn_mfma_f32_16x16x32_f16(kw, qf[n][b][i], x, 0, 0, 0);
                            m[b & 1][n][h] = x;
                        }
                    }
                }
                if (b > 0) {
#pragma unroll
                    for (int n = 0; n < NT; n++)
#pragma unroll
                        for (int j = 0; j < 8; j++) {
                            const float x = m[(b - 1) & 1][n][j >> 2][j & 3], d = (float)K.d[b - 1][j];
                            t[n][j] = b == 1 ? d * x : __builtin_fmaf(d, x, t[n][j]);
                            __asm__ volatile("" : "+v"(t[n][j]));  // (here, not behind the next branch with every block's sums held)
                        }
                }
                __builtin_amdgcn_sched_barrier(0);
            }
            if (more) K.load(pn, lane);

            // ---- scores, in powers of two; masked ones −∞
            const int key0 = 32 * g + 8 * ka;
            const bool special = a.mask || !have || 32 * g + 32 > see_all;
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int j = 0; j < 8; j++) t[n][j] *= cs[n];
            uint32_t hidden[NT];  // bit j: key key0 + j is masked
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
                            for (int j = 0; j < 8; j++) mv[j] = key0 + j < len ? (float)mp[j] : 0.f;
                        }
#pragma unroll
                        for (int j = 0; j < 8; j++) t[n][j] = mv[j] == -INFINITY ? -INFINITY : __builtin_fmaf(mv[j], 1.4426950408889634f, t[n][j]);
                    }
                    hidden[n] = 0;
#pragma unroll
                    for (int j = 0; j < 8; j++) {
                        if (!have || key0 + j >= lim[n]) t[n][j] = -INFINITY;
                        hidden[n] |= t[n][j] == -INFINITY ? 1u << j : 0u;
                    }
                }
                // a masked key's probability is zero, but V's scale there may be
                // no number: zero where none of this lane's columns sees the key
                uint32_t all = hidden[0], any = hidden[0];
#pragma unroll
                for (int n = 1; n < NT; n++) all &= hidden[n], any |= hidden[n];
                uint32_t odd = 0;  // keys some column sees, with a scale that is no number
#pragma unroll
                for (int b = 0; b < NB; b++) {
                    kv_u4 d = __builtin_bit_cast(kv_u4, V.d[b]);
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        d[j] &= keep_pair(all, j);
                        odd |= ((d[j] & 0x7c00u) == 0x7c00u ? 1u << 2 * j : 0u) | ((d[j] & 0x7c000000u) == 0x7c000000u ? 2u << 2 * j : 0u);
                    }
                    V.d[b] = __builtin_bit_cast(kv_h8, d);
                }
                if constexpr (NT > 1) partly = __builtin_amdgcn_ballot_w64(odd & any) != 0;
            }

            // ---- the references, where a score or a scale outgrew them
            bool grow = false;
#pragma unroll
            for (int n = 0; n < NT; n++) {
                float mx = fmaxf(fmaxf(t[n][0], t[n][1]), t[n][2]);
                mx = fmaxf(fmaxf(mx, t[n][3]), t[n][4]);
                mx = fmaxf(fmaxf(mx, t[n][5]), fmaxf(t[n][6], t[n][7]));
                grow = grow || mx > ref[n] + (float)(15 - ed);
            }
            const uint32_t bound = (uint32_t)(ed >= -14 ? (ed + 15) << 10 : 1 << (ed + 24));  // fp16 bits of 2^ed
#pragma unroll
            for (int i = 0; i < VD; i++) grow = grow || (vds[i] & 0x7fffu) > bound || ((vds[i] >> 16) & 0x7fffu) > bound;
            if (__builtin_amdgcn_ballot_w64(grow)) {
                // V's largest scale among keys of the sequence; not those that are no numbers
                uint32_t dm = 0;
#pragma unroll
                for (int i = 0; i < VD; i++) {
                    const int k2 = 32 * g + 2 * ((lane + 64 * i) & 15);
                    const uint32_t lo = vds[i] & 0x7fffu, hi = (vds[i] >> 16) & 0x7fffu;
                    if (have && k2 < len && lo < 0x7c00u) dm = max(dm, lo);
                    if (have && k2 + 1 < len && hi < 0x7c00u) dm = max(dm, hi);
                }
#pragma unroll
                for (int x = 1; x < 64; x *= 2) dm = max(dm, (uint32_t)__shfl_xor((int)dm, x, 64));
                // 2^en ≥ every scale: one above the exponent, or of a subnormal its bit length − 24
                const int en = dm >= 0x400u ? (int)(dm >> 10) - 14 : 8 - (dm ? __builtin_clz(dm) : 32);
                const int ed_n = max(ed, __builtin_amdgcn_readfirstlane(en));
#pragma unroll
                for (int n = 0; n < NT; n++) {
                    float mx = fmaxf(fmaxf(t[n][0], t[n][1]), t[n][2]);
                    mx = fmaxf(fmaxf(mx, t[n][3]), t[n][4]);
                    mx = fmaxf(fmaxf(mx, t[n][5]), fmaxf(t[n][6], t[n][7]));
                    mx = max_over_keys(mx);
                    // the reference is the largest score + ed − 7
                    const float best = ref[n] == KV_NONE ? KV_NONE : ref[n] - (float)(ed - 7);
                    const float top = fmaxf(best, mx);
                    const float ref_n = top <= KV_NONE ? KV_NONE : top + (float)(ed_n - 7);
                    const float alpha = ref_n == ref[n] ? 1.f : __builtin_amdgcn_exp2f(ref[n] - ref_n);
                    ref[n] = ref_n;
                    sum[n] *= alpha;
#pragma unroll
                    for (int w = 0; w < W; w++) acc[n][w] *= alpha;
                }
                ed = ed_n;
            }

            // ---- probabilities, in units of the reference
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    t[n][j] = __builtin_amdgcn_exp2f(t[n][j] - ref[n]);
                    sum[n] += t[n][j];
                }

            // ---- Oᵀ += Vᵀ·(P·d)ᵀ, block by block of V's channels
#pragma unroll
            for (int b = 0; b < NB; b++) {
                kv_u4 p[NT][PARTS];
                const kv_u4 d = __builtin_bit_cast(kv_u4, V.d[b]);
#pragma unroll
                for (int n = 0; n < NT; n++)
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        if constexpr (!F32) {
                            p[n][0][j] = scaled_pair(t[n][2 * j], t[n][2 * j + 1], d[j]);
                        } else {
                            const kv_h2 dd = as_h2(d[j]);
                            float x = t[n][2 * j] * (float)dd[0], y = t[n][2 * j + 1] * (float)dd[1];
                            // one value for hi and for lo: folded into a mixed fma, hi alone would be rounded from the exact product
                            __asm__("" : "+v"(x), "+v"(y));
                            const kv_h2 hi = {(_Float16)x, (_Float16)y};
                            p[n][0][j] = __builtin_bit_cast(uint32_t, hi);
                            p[n][PARTS - 1][j] = __builtin_bit_cast(uint32_t, kv_h2{(_Float16)(x - (float)hi[0]), (_Float16)(y - (float)hi[1])});
                        }
                    }
                if (NT > 1 && partly) {
                    __asm__ volatile("");  // (a branch, not selects)
#pragma unroll
                    for (int n = 0; n < NT; n++)
#pragma unroll
                        for (int x = 0; x < PARTS; x++)
#pragma unroll
                            for (int j = 0; j < 4; j++) p[n][x][j] &= keep_pair(hidden[n], j);
                }
#pragma unroll
                for (int w = 2 * b; w < 2 * b + 2; w++) {
                    const kv_h8 vw = V.word(w, M);
#pragma unroll
                    for (int n = 0; n < NT; n++)
#pragma unroll
                        for (int x = 0; x < PARTS; x++)
                            acc[n][w] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vw, __builtin_bit_cast(kv_h8, p[n][x]), acc[n][w], 0, 0, 0);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
            if (!more) break;
            V.load(pn + C::HALF, lane);
#pragma unroll
            for (int i = 0; i < VD; i++)
                vds[i] = *(const uint32_t *)(pn + C::HALF + C::CODES + ((lane + 64 * i) % (NB * 16)) * 4);
            g = gn;
            have = have_n;
        }
    }

    // ---- the four waves joined: 2 and 3 into 0 and 1, then 1 into 0
#pragma unroll
    for (int n = 0; n < NT; n++) sum[n] = sum_over_keys(sum[n]);
    auto give = [&](int slot) {
#pragma unroll
        for (int n = 0; n < NT; n++) {
            lds_ml[slot][n][0][lane] = ref[n];
            lds_ml[slot][n][1][lane] = sum[n];
#pragma unroll
            for (int w = 0; w < W; w++) lds[slot][n * W + w][lane] = acc[n][w];
        }
    };
    auto take = [&](int slot) {
#pragma unroll
        for (int n = 0; n < NT; n++) {
            const float r = lds_ml[slot][n][0][lane], l = lds_ml[slot][n][1][lane];
            const float top = fmaxf(ref[n], r);
            const float wa = ref[n] == top ? 1.f : __builtin_amdgcn_exp2f(ref[n] - top);
            const float wb = r == top ? 1.f : __builtin_amdgcn_exp2f(r - top);
            ref[n] = top;
            sum[n] = sum[n] * wa + l * wb;
#pragma unroll
            for (int w = 0; w < W; w++) acc[n][w] = acc[n][w] * wa + lds[slot][n * W + w][lane] * wb;
        }
    };
    if (wave >= 2) give(wave - 2);
    __syncthreads();
    if (wave < 2) take(wave);
    __syncthreads();
    if (wave == 1) give(0);
    __syncthreads();
    if (wave != 0) return;
    take(0);

#pragma unroll
    for (int n = 0; n < NT; n++) {
        if (c0 + 16 * n + col >= ncols) continue;
        const int64_t row = (int64_t)tok[n] * a.nh + head[n];
        if (a.nsplit > 1) {
            const int64_t at = (int64_t)split * a.n_tokens * a.nh + row;
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

// Columns tiles a wave holds: as many as its registers leave room for (the
// accumulators are 8·NB of them a tile), one where there are no more columns.
template <int NB, bool F32>
constexpr int kv_most_tiles() { return NB <= 2 ? (F32 ? 2 : 4) : (NB == 8 ? 1 : 2); }

template <int Q>
hipError_t launch_kv_attn(const KvAttnArgs &a, bool f32, hipStream_t st) {
    const int64_t units = (int64_t)a.n_seq * a.c.heads * a.nsplit;
    const int64_t grid = (units >= 8 ? (units + 7) / 8 * 8 : units) * a.ctiles;
    if (grid > INT32_MAX) return hipErrorInvalidValue;
    auto go = [&](auto nb, auto f) {
        constexpr int NB = nb(), MOST = kv_most_tiles<NB, f()>();
        if (a.nt == 1) hipLaunchKernelGGL((k_kv_attn<Q, NB, f(), 1>), dim3((unsigned)grid), dim3(256), 0, st, a);
        else if (a.nt == MOST) hipLaunchKernelGGL((k_kv_attn<Q, NB, f(), MOST>), dim3((unsigned)grid), dim3(256), 0, st, a);
        else return hipErrorInvalidValue;
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
