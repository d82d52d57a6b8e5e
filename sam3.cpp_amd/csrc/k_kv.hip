// k_kv.hip — writing rows into the quantized key/value cache, reading them
// back, and joining attention's partial results over key ranges.
#include "k_kv.h"

namespace s3e {
namespace {

typedef _Float16 h8 __attribute__((ext_vector_type(8)));

// Maximum and minimum as the one instruction they are (the builtins put another
// before it that quiets a signalling NaN; whether there is a NaN is seen apart).
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ float max_of(float a, float b) { float r; __asm__("v_max_f32 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b)); return r; }
__device__ __forceinline__ float min_of(float a, float b) { float r; __asm__("v_min_f32 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b)); return r; }
__device__ __forceinline__ h2 max_of(h2 a, h2 b) { h2 r; __asm__("v_pk_max_f16 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b)); return r; }
__device__ __forceinline__ h2 min_of(h2 a, h2 b) { h2 r; __asm__("v_pk_min_f16 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b)); return r; }

// Before lane exchanges (DPP) of what inline asm has written: two wait states,
// which the compiler puts only behind instructions of its own.
__device__ __forceinline__ void settle(float &a, float &b) { __asm__("s_nop 1" : "+v"(a), "+v"(b)); }

// Eight consecutive values of a row, as they lie in memory until they are used.
template <typename T>
struct Raw8 {
    T x[8];
    __device__ __forceinline__ void load(const T *p, int vec) {
        if (vec) {
#pragma unroll
            for (int i = 0; i < (int)sizeof(T) / 2; i++) *(uint4 *)(x + i * (16 / sizeof(T))) = ((const uint4 *)p)[i];
        } else {
#pragma unroll
            for (int j = 0; j < 8; j++) x[j] = p[j];
        }
    }
    // largest and smallest value, and a number only if all of them are
    __device__ __forceinline__ void range(float &hi, float &lo, float &odd) const {
        if constexpr (sizeof(T) == 2) {
            h2 v[4], z = {(_Float16)0.f, (_Float16)0.f};
#pragma unroll
            for (int j = 0; j < 4; j++) {
                v[j] = h2{x[2 * j], x[2 * j + 1]};
                z = __builtin_elementwise_fma(v[j], h2{(_Float16)0.f, (_Float16)0.f}, z);
            }
            const h2 a = max_of(max_of(v[0], v[1]), max_of(v[2], v[3])), b = min_of(min_of(v[0], v[1]), min_of(v[2], v[3]));
            hi = max_of((float)a[0], (float)a[1]);
            lo = min_of((float)b[0], (float)b[1]);
            odd = (float)z[0] + (float)z[1];
        } else {
            hi = lo = x[0];
            odd = 0.f;
#pragma unroll
            for (int j = 0; j < 8; j++) {
                hi = max_of(hi, x[j]);
                lo = min_of(lo, x[j]);
                odd = __builtin_fmaf(x[j], 0.f, odd);
            }
        }
    }
    // the first value of magnitude top: its place, or 8
    __device__ __forceinline__ int place(float top) const {
        int at = 8;
#pragma unroll
        for (int j = 7; j >= 0; j--) at = fabsf((float)x[j]) == top ? j : at;
        return at;
    }
};

// The codes of one 32-channel block held as 8 values by each of 4 neighbouring
// lanes (in channel order), as ggml's quantize_row_q4_0 (d = max / −8, max the
// first value of largest magnitude; q = min(15, ⌊x/d + 8.5⌋)) and the engine's
// Q8_0 conversion (d = amax / 127, q = round-half-even(x·(127/amax))) choose
// them in fp32.  A block with an infinity or a NaN gets a NaN scale, so that
// all of it reads back as NaN, and the codes of zeros.  codes: 0..15, or int8
// in the low byte.
// (Lane exchanges within four lanes are DPP moves, folded into the instruction
// that uses them.)
template <int X>
__device__ __forceinline__ int quad_xor(int v) {
    static_assert(X == 1 || X == 2, "of four lanes");
    return __builtin_amdgcn_update_dpp(v, v, X == 1 ? 0xb1 : 0x4e, 0xf, 0xf, true);
}
template <int X>
__device__ __forceinline__ float quad_xor(float v) { return __int_as_float(quad_xor<X>(__float_as_int(v))); }

template <int Q, typename T>
__device__ __forceinline__ void quant_block(const Raw8<T> &raw, int lane, uint32_t *codes, uint16_t &scale) {
    float hi, lo, odd;
    raw.range(hi, lo, odd);
    settle(hi, lo);
    hi = max_of(hi, quad_xor<1>(hi)), lo = min_of(lo, quad_xor<1>(lo)), odd += quad_xor<1>(odd);
    settle(hi, lo);
    hi = max_of(hi, quad_xor<2>(hi)), lo = min_of(lo, quad_xor<2>(lo)), odd += quad_xor<2>(odd);
    const float top = max_of(hi, -lo);
    float d, id;
    if constexpr (Q == 4) {
        float lead = hi > -lo ? hi : lo;
        if (hi == -lo && top != 0.f) {
            // both signs reach it: the first in the block decides
            const int mine = raw.place(top), at = mine == 8 ? 32 : (lane & 3) * 8 + mine;
            int first = min(at, quad_xor<1>(at));
            first = min(first, quad_xor<2>(first));
            int sign = 0;  // of the lane that holds it: 1 where it is negative
#pragma unroll
            for (int j = 0; j < 8; j++) sign = first == (lane & 3) * 8 + j && raw.x[j] < (T)0.f ? 1 : sign;
            sign |= quad_xor<1>(sign);
            sign |= quad_xor<2>(sign);
            lead = sign ? -top : top;
        }
        d = (top == 0.f ? 0.f : lead) * -0.125f;
        id = d != 0.f ? 1.0f / d : 0.f;
    } else {
        d = top / 127.0f;
        id = top != 0.f ? 127.0f / top : 0.f;
    }
    // (a scale whose reciprocal overflows is far below fp16's smallest: zero)
    if (__builtin_isinf(id)) id = 0.f;
    scale = half_bits(d);
#pragma unroll
    for (int j = 0; j < 8; j++) {
        float x = __builtin_fmaf((float)raw.x[j], id, 0.f);  // the rounded product (of fp16 as it is)
        __asm__("" : "+v"(x));
        if constexpr (Q == 4) codes[j] = min(15u, (uint32_t)(x + 8.5f));
        else codes[j] = __float_as_uint(x + 12582912.0f);  // 1.5 · 2^23: rounded half to even into the low bits
    }
    if (!(odd == 0.f)) {
        scale = 0x7e00;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            codes[j] = Q == 4 ? 8 : 0;
            __asm__ volatile("" : "+v"(codes[j]));  // (a branch, not selects)
        }
    }
}

// Bytes 0 of four words as one.
__device__ __forceinline__ uint32_t pack4(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    return __builtin_amdgcn_perm(__builtin_amdgcn_perm(d, c, 0x0c0c0400u), __builtin_amdgcn_perm(b, a, 0x0c0c0400u), 0x05040100u);
}

template <int Q>
__device__ __forceinline__ uint64_t pack_word(const uint32_t *c) {
    if constexpr (Q == 4) {
        uint32_t x = c[0];
#pragma unroll
        for (int j = 1; j < 8; j++) x |= c[j] << (4 * ((j >> 1) + 4 * (j & 1)));
        return x;
    } else {
        return pack4(c[0], c[1], c[2], c[3]) | (uint64_t)pack4(c[4], c[5], c[6], c[7]) << 32;
    }
}

template <int Q>
__device__ __forceinline__ void store_word(uint8_t *p, uint64_t x) {
    if constexpr (Q == 4) *(uint32_t *)p = (uint32_t)x;
    else *(uint64_t *)p = x;
}

// A chunk's address: slot / 32 within the page, by head.
__device__ __forceinline__ uint8_t *chunk_of(const KvCache &c, int64_t slot, int head, int bytes) {
    const int64_t page = slot >> c.page_shift, in = (slot & ((1 << c.page_shift) - 1)) >> 5;
    return c.data + ((page * c.heads + head) * (1 << (c.page_shift - 5)) + in) * bytes;
}

constexpr int KV_ROWS = 64;  // rows of a work-group, four threads each

// One tensor (blockIdx.z) of 64 rows and one head.  Thread 4r + g takes
// channels 32b + 8g .. + 8 of row r for every block b: a K word each, and the
// four lanes agree on a block's scale.  A V word holds eight keys of one
// channel: where eight rows of the call fill one aligned run of eight slots
// their codes meet in LDS and the words are stored whole, by the work-group
// whose rows hold the run's first (it converts up to seven of the next one's
// rows again); a row outside any run replaces its own code in each word by a
// 64-bit atomic or a byte store, so that runs, lone rows and neighbouring
// work-groups never write each other's codes.
// Reads the rows and writes 9/16 (Q4_0) or 17/16 bytes a value once: 65 536
// tokens of 8 heads of 128, fp16 to Q4_0, take 81 µs write after write (344 MB,
// 4.3 TB/s; a copy of as many bytes 62), 92 in turn with reads of them, 28 736 of
// one head of 256 to Q8_0 16 µs.  Vector
// instructions keep 73 % of the SIMDs' cycles busy, the more so as memory waits
// on them: hence the packed range search, the row prefetched ahead of its slot,
// and the byte transposes that make V's words.  Scattered rows cost a 64-bit
// atomic for two words: 32 768 of those tokens 209-215 µs in Q4_0 (an and and an
// or a word: 1464), 115-123 µs in Q8_0; 512 of 16 heads of 64 8 µs.
template <int Q, int NB, typename T>
__global__ __launch_bounds__(256) void k_kv_write(KvWriteArgs a) {
    using C = KvChunk<Q, NB>;
    constexpr int D = 32 * NB;
    // rows −7 .. 64 + 13 of the call's slots around this work-group's
    __shared__ int32_t sl[KV_ROWS + 21];
    __shared__ __attribute__((aligned(16))) uint8_t codes_lds[(KV_ROWS + 7) * D];
    __shared__ int starts[KV_ROWS / 8 + 1], lones[KV_ROWS + 1];
    const int tid = threadIdx.x, lane = tid & 63, head = blockIdx.y;
    const bool is_v = blockIdx.z != 0;
    const int64_t r0 = (int64_t)blockIdx.x * KV_ROWS;
    const T *x = (const T *)(is_v ? a.x[1] : a.x[0]);
    const int64_t st = is_v ? a.st[1] : a.st[0], sh = is_v ? a.sh[1] : a.sh[0];
    const int vec = is_v ? a.vec[1] : a.vec[0];
    const int g = tid & 3;
    // own rows, on their way while the slots are looked at
    Raw8<T> own_row[NB];
    {
        const int64_t r = min(r0 + (tid >> 2), (int64_t)a.n - 1);
#pragma unroll
        for (int b = 0; b < NB; b++) own_row[b].load(x + r * st + head * sh + 32 * b + 8 * g, vec);
    }
    if (tid < KV_ROWS + 21) {
        const int64_t r = r0 + tid - 7;
        int32_t s = -1;
        if (r >= 0 && r < a.n) {
            s = a.slots[r];
            if (s < 0 || s >= a.c.slots) s = -1;
        }
        sl[tid] = s;
    }
    __syncthreads();
    // whether row r (relative) lies in a run of eight rows on eight aligned slots
    auto in_run = [&](int r) {
        const int s = sl[r + 7];
        if (s < 0) return false;
        const int j = s & 7;
        bool ok = true;
#pragma unroll
        for (int m = 0; m < 8; m++) {
            const int at = r + 7 - j + m;
            ok = ok && at >= 0 && at < KV_ROWS + 21 && sl[at] == s - j + m;
        }
        return ok;
    };
    if (!is_v) {
        const int r = tid >> 2, s = sl[r + 7];
        if (s < 0) return;  // (the four lanes of a row together)
        uint8_t *ck = chunk_of(a.c, s, head, C::BYTES);
        const int key = s & 31, t = (key >> 2) & 1, row = 4 * (key >> 3) + (key & 3);
        uint64_t w[NB];
#pragma unroll
        for (int b = 0; b < NB; b++) {
            uint32_t c[8];
            uint16_t d;
            quant_block<Q>(own_row[b], lane, c, d);
            w[b] = pack_word<Q>(c);
            if (g == (b & 3)) *(uint16_t *)(ck + C::CODES + (b * 32 + key) * 2) = d;
        }
        if constexpr (NB % C::PER == 0) {
            // a row's words of one lane are whole pieces
#pragma unroll
            for (int b = 0; b < NB; b += C::PER) {
                uint4 y;
                if constexpr (Q == 4) y = make_uint4((uint32_t)w[b], (uint32_t)w[b + 1], (uint32_t)w[b + 2], (uint32_t)w[b + 3]);
                else y = make_uint4((uint32_t)w[b], (uint32_t)(w[b] >> 32), (uint32_t)w[b + 1], (uint32_t)(w[b + 1] >> 32));
                *(uint4 *)(ck + C::word(t * NB + b, 16 * g + row)) = y;
            }
        } else {
#pragma unroll
            for (int b = 0; b < NB; b++) store_word<Q>(ck + C::word(t * NB + b, 16 * g + row), w[b]);
        }
        return;
    }

    // V: own rows' codes, then those of the next work-group that a run from here ends in
    auto convert = [&](int r, bool own, const Raw8<T> *raw) {
        const int s = sl[r + 7];
        uint8_t *cv = chunk_of(a.c, s, head, C::BYTES) + C::HALF;
#pragma unroll
        for (int b = 0; b < NB; b++) {
            uint32_t c[8];
            uint16_t d;
            quant_block<Q>(raw[b], lane, c, d);
            if (own && g == (b & 3)) *(uint16_t *)(cv + C::CODES + (b * 32 + (s & 31)) * 2) = d;
            *(uint2 *)(codes_lds + r * D + 32 * b + 8 * g) = make_uint2(pack4(c[0], c[1], c[2], c[3]), pack4(c[4], c[5], c[6], c[7]));
        }
    };
    if (sl[(tid >> 2) + 7] >= 0) convert(tid >> 2, true, own_row);
    if (tid < 28) {
        const int r = KV_ROWS + (tid >> 2), s = sl[r + 7];
        if (s >= 0 && in_run(r) && r - (s & 7) < KV_ROWS) {
            Raw8<T> next[NB];
#pragma unroll
            for (int b = 0; b < NB; b++) next[b].load(x + (r0 + r) * st + head * sh + 32 * b + 8 * g, vec);
            convert(r, false, next);
        }
    }
    if (tid < 64) {
        const bool run = in_run(tid), first = run && (sl[tid + 7] & 7) == 0, lone = !run && sl[tid + 7] >= 0;
        const uint64_t below = (1ull << tid) - 1, m = __ballot(first), o = __ballot(lone);
        if (first) starts[1 + __popcll(m & below)] = tid;
        if (lone) lones[1 + __popcll(o & below)] = tid;
        if (tid == 0) starts[0] = __popcll(m), lones[0] = __popcll(o);
    }
    __syncthreads();
    // lone rows: unit (row, piece, channel m of 16), the row's own code in each of
    // the lane's words.  Others of the call may share a word: a nibble is
    // exchanged by one xor with what it has to change (nobody else writes it, so
    // what is read of it stands), a byte is stored
    for (int u = tid; u < lones[0] * C::PIECES * 16; u += 256) {
        const int m = u & 15, pi = (u >> 4) % C::PIECES, r = lones[1 + (u >> 4) / C::PIECES];
        const int s = sl[r + 7], k8 = s & 7;
        uint8_t *o = chunk_of(a.c, s, head, C::BYTES) + C::HALF + C::word(pi * C::PER, 16 * ((s & 31) >> 3) + m);
        const uint8_t *c = codes_lds + r * D + 16 * pi * C::PER + m;
        if constexpr (Q == 4) {
            const int sft = 4 * ((k8 >> 1) + 4 * (k8 & 1));
            const bool whole = C::width(pi) == C::PER;
            const uint2 lo = *(const uint2 *)o, hi = whole ? *(const uint2 *)(o + 8) : make_uint2(0, 0);
            auto change = [&](uint32_t old, int w) { return (old ^ (uint32_t)c[16 * w] << sft) & 15u << sft; };
            atomicXor((unsigned long long *)o, change(lo.x, 0) | (unsigned long long)change(lo.y, 1) << 32);
            if (whole) atomicXor((unsigned long long *)(o + 8), change(hi.x, 2) | (unsigned long long)change(hi.y, 3) << 32);
        } else {
#pragma unroll
            for (int w = 0; w < C::PER; w++) o[8 * w + k8] = c[16 * w];
        }
    }
    // whole words: unit (run, piece, four channels 4q .. 4q + 4 of 16).  The bytes
    // of four channels come as one word a row; two rows' nibbles share its bytes,
    // and a 4 × 4 transpose of bytes turns four such words into a channel's each
    constexpr int ROWS = Q == 4 ? 2 : 1, WORDS4 = 8 / ROWS;  // rows in a byte, 4-byte words of eight rows
    const int units = starts[0] * C::PIECES * 4;
    for (int u = tid; u < units; u += 256) {
        const int q = u & 3, pi = (u >> 2) % C::PIECES, r = starts[1 + (u >> 2) / C::PIECES];
        const int s = sl[r + 7];
        uint8_t *cv = chunk_of(a.c, s, head, C::BYTES) + C::HALF;
        uint32_t out[4][4];  // channel, 4 bytes of its piece
#pragma unroll
        for (int i = 0; i < C::PER; i++) {
            const int w = min(pi * C::PER + i, C::WORDS - 1);  // (a short piece's missing words: any)
            uint32_t in[8];
#pragma unroll
            for (int j = 0; j < 8; j++) in[j] = *(const uint32_t *)(codes_lds + (r + j) * D + 16 * w + 4 * q);
            uint32_t m[WORDS4];
            if constexpr (Q == 4) m[0] = in[0] | in[2] << 4, m[1] = in[4] | in[6] << 4, m[2] = in[1] | in[3] << 4, m[3] = in[5] | in[7] << 4;
            else
#pragma unroll
                for (int j = 0; j < 8; j++) m[j % WORDS4] = in[j];
#pragma unroll
            for (int h = 0; h < WORDS4 / 4; h++) {
                const uint32_t a0 = __builtin_amdgcn_perm(m[4 * h + 1], m[4 * h], 0x05010400u), a1 = __builtin_amdgcn_perm(m[4 * h + 1], m[4 * h], 0x07030602u);
                const uint32_t b0 = __builtin_amdgcn_perm(m[4 * h + 3], m[4 * h + 2], 0x05010400u), b1 = __builtin_amdgcn_perm(m[4 * h + 3], m[4 * h + 2], 0x07030602u);
                const int at = i * (C::WB / 4) + h;
                out[0][at] = __builtin_amdgcn_perm(b0, a0, 0x05040100u);
                out[1][at] = __builtin_amdgcn_perm(b0, a0, 0x07060302u);
                out[2][at] = __builtin_amdgcn_perm(b1, a1, 0x05040100u);
                out[3][at] = __builtin_amdgcn_perm(b1, a1, 0x07060302u);
            }
        }
#pragma unroll
        for (int c = 0; c < 4; c++) {
            uint8_t *o = cv + C::word(pi * C::PER, 16 * ((s & 31) >> 3) + 4 * q + c);
            if (C::width(pi) == C::PER) *(uint4 *)o = make_uint4(out[c][0], out[c][1], out[c][2], out[c][3]);
            else *(uint2 *)o = make_uint2(out[c][0], out[c][1]);
        }
    }
}

// A code of a word as the byte of an int8.
template <int Q>
__device__ __forceinline__ uint32_t code_of(uint64_t w, int j) {
    if constexpr (Q == 4) return (((uint32_t)w >> (4 * ((j >> 1) + 4 * (j & 1)))) & 15u) - 8u;
    else return (uint32_t)(w >> (8 * j));
}

// A lane's words of one piece (16 bytes of them, or the 8 of a last one).
template <int Q, int NB>
__device__ __forceinline__ void load_piece(const uint8_t *half, int p, int lane, uint64_t *w) {
    using C = KvChunk<Q, NB>;
    const uint8_t *at = half + C::word(p * C::PER, lane);
    if (C::width(p) == C::PER) {
        const uint4 x = gload16(at);
        if constexpr (Q == 4) w[0] = x.x, w[1] = x.y, w[2] = x.z, w[3] = x.w;
        else w[0] = x.x | (uint64_t)x.y << 32, w[1] = x.z | (uint64_t)x.w << 32;
    } else {
        const uint2 x = gload8(at);
        w[0] = x.x, w[1] = x.y;
    }
}

// Eight values of a row, each scale · code rounded once.
template <typename T>
__device__ __forceinline__ void store8(T *o, const float *v) {
    if constexpr (sizeof(T) == 2) {
        h8 z;
#pragma unroll
        for (int j = 0; j < 8; j++) z[j] = (_Float16)v[j];
        *(h8 *)o = z;
    } else {
        *(float4 *)o = make_float4(v[0], v[1], v[2], v[3]);
        *(float4 *)(o + 4) = make_float4(v[4], v[5], v[6], v[7]);
    }
}

// One tensor (blockIdx.z) of 64 rows and one head.  K: thread 4r + g gives
// channels 32b + 8g .. + 8 of row r, its own words.  V's words hold eight keys
// of a channel: where eight rows are an aligned run of slots a thread takes
// whole pieces apart (four words of one lane, for all eight rows), else a row's
// own codes are picked out of them; the codes meet in LDS as bytes and leave
// row by row, so that both sides of memory see whole lines.  A slot outside the
// cache reads as zeros.  Bound by HBM: 65 536 tokens of 8 heads of 128 from Q4_0
// to fp16 take 85 µs (344 MB, 4.1 TB/s), 28 736 of one head of 256 from Q8_0
// 12 µs; a code at a time straight to memory took 154 and 15.
template <int Q, int NB, typename T>
__global__ __launch_bounds__(256) void k_kv_read(KvReadArgs a) {
    using C = KvChunk<Q, NB>;
    constexpr int D = 32 * NB;
    __shared__ int32_t sl[KV_ROWS];
    __shared__ __attribute__((aligned(16))) uint8_t codes_lds[KV_ROWS * D];
    __shared__ uint16_t scales_lds[KV_ROWS * NB];
    __shared__ uint64_t runs;
    const int tid = threadIdx.x, head = blockIdx.y;
    const bool is_v = blockIdx.z != 0;
    T *y = (T *)(is_v ? a.y[1] : a.y[0]);
    if (!y) return;
    const int64_t r0 = (int64_t)blockIdx.x * KV_ROWS;
    const int rows = (int)min((int64_t)KV_ROWS, a.n - r0);
    y += (r0 * a.c.heads + head) * D;
    const int64_t ld = (int64_t)a.c.heads * D;

    if (!is_v) {
        const int g = tid & 3, r = tid >> 2;
        if (r >= rows) return;
        const int64_t s = a.slots[r0 + r];
        const bool in = s >= 0 && s < a.c.slots;
        const uint8_t *ck = chunk_of(a.c, in ? s : 0, head, C::BYTES);
        const int key = (int)(s & 31), t = (key >> 2) & 1, row = 4 * (key >> 3) + (key & 3);
        uint64_t w[NB];
        if constexpr (NB % C::PER == 0) {
#pragma unroll
            for (int b = 0; b < NB; b += C::PER) load_piece<Q, NB>(ck, (t * NB + b) / C::PER, 16 * g + row, w + b);
        } else {
#pragma unroll
            for (int b = 0; b < NB; b++) {
                const uint8_t *at = ck + C::word(t * NB + b, 16 * g + row);
                if constexpr (Q == 4) w[b] = *(const uint32_t *)at;
                else w[b] = *(const uint64_t *)at;
            }
        }
        float d[NB];
#pragma unroll
        for (int b = 0; b < NB; b++) d[b] = (float)*(const _Float16 *)(ck + C::CODES + (b * 32 + key) * 2);
#pragma unroll
        for (int b = 0; b < NB; b++) {
            float v[8];
#pragma unroll
            for (int j = 0; j < 8; j++) v[j] = in ? (float)(int8_t)code_of<Q>(w[b], j) * d[b] : 0.f;
            store8(y + r * ld + 32 * b + 8 * g, v);
        }
        return;
    }

    if (tid < KV_ROWS) {
        int32_t s = tid < rows ? a.slots[r0 + tid] : -1;
        if (s < 0 || s >= a.c.slots) s = -1;
        sl[tid] = s;
        // (rows 0 .. 63 are one wave) bit r: rows r .. r + 8 are an aligned run
        bool run = s >= 0 && (s & 7) == 0 && tid + 8 <= KV_ROWS;
#pragma unroll
        for (int m = 1; m < 8; m++) run = run & (__shfl(s, min(tid + m, KV_ROWS - 1), 64) == s + m);
        const uint64_t b = __ballot(run);
        if (tid == 0) runs = b;
    }
    __syncthreads();
    const uint64_t starts = runs;
    // whole runs: unit (row, piece, channel m of 16) where a run starts
    for (int u = tid; u < KV_ROWS / 8 * C::PIECES * 16; u += 256) {
        const int m = u & 15, p = (u >> 4) % C::PIECES;
        uint64_t left = starts;
        for (int k = (u >> 4) / C::PIECES; k > 0; k--) left &= left - 1;  // the k-th start
        if (!left) continue;
        const int r = __ffsll((unsigned long long)left) - 1, s = sl[r];
        uint64_t w[C::PER];
        load_piece<Q, NB>(chunk_of(a.c, s, head, C::BYTES) + C::HALF, p, 16 * ((s & 31) >> 3) + m, w);
#pragma unroll
        for (int i = 0; i < C::PER; i++)
            if (i < C::width(p)) {
#pragma unroll
                for (int j = 0; j < 8; j++) codes_lds[(r + j) * D + 16 * (p * C::PER + i) + m] = (uint8_t)code_of<Q>(w[i], j);
            }
    }
    // lone rows: thread 16r + m, its channels 16w + m
    for (int u = tid; u < KV_ROWS * 16; u += 256) {
        const int m = u & 15, r = u >> 4, s = sl[r];
        const uint64_t before = starts & (r == 63 ? ~0ull : (2ull << r) - 1);  // runs that start at r or earlier
        const bool covered = before && r - (63 - __clzll((long long)before)) < 8;
        if (s < 0 || covered) continue;
        const uint8_t *cv = chunk_of(a.c, s, head, C::BYTES) + C::HALF;
#pragma unroll
        for (int p = 0; p < C::PIECES; p++) {
            uint64_t w[C::PER];
            load_piece<Q, NB>(cv, p, 16 * ((s & 31) >> 3) + m, w);
#pragma unroll
            for (int i = 0; i < C::PER; i++)
                if (i < C::width(p)) codes_lds[r * D + 16 * (p * C::PER + i) + m] = (uint8_t)code_of<Q>(w[i], s & 7);
        }
    }
    for (int u = tid; u < KV_ROWS * NB; u += 256) {
        const int r = u / NB, b = u % NB, s = sl[r];
        scales_lds[u] = s < 0 ? 0 : *(const uint16_t *)(chunk_of(a.c, s, head, C::BYTES) + C::HALF + C::CODES + (b * 32 + (s & 31)) * 2);
    }
    __syncthreads();
    for (int u = tid; u < rows * (D / 8); u += 256) {
        const int r = u / (D / 8), q = u % (D / 8);
        const uint2 c = *(const uint2 *)(codes_lds + r * D + 8 * q);
        const float d = (float)__builtin_bit_cast(_Float16, scales_lds[r * NB + (q >> 2)]);
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] = sl[r] < 0 ? 0.f : (float)(int8_t)((j < 4 ? c.x : c.y) >> (8 * (j & 3))) * d;
        store8(y + r * ld + 8 * q, v);
    }
}

// Output rows (query, head) from their key ranges: each range's unnormalised
// output and sum are in units of 2^reference.  D/4 threads hold a row.  Where a
// row has many ranges a work-group takes one row (SPREAD), its other threads
// further ranges, joined in LDS in a fixed order; where it has few, a row each
// (whole calls: 131 072 keys in 43 ranges 39 µs, a row each 52; 4096 in 16
// ranges 10.0 and 11.9; up to eight ranges alike).
// Bound by launch and two loads one behind the other where rows are few (32 rows
// of 128 from 43 ranges 5.2 µs), by memory where they are many (4096 rows of 256
// from 11 ranges, 47 MB: 12 µs).
template <int D, bool F32, bool SPREAD, bool FIND>
__global__ __launch_bounds__(256) void k_kv_combine(KvAttnArgs a) {
    constexpr int LANES = D / 4, GROUPS = 256 / LANES;
    __shared__ float4 acc_lds[SPREAD ? GROUPS : 1][LANES];
    __shared__ float sum_lds[GROUPS];
    const int tid = threadIdx.x, gr = tid / LANES, d4 = tid % LANES;
    const int r = SPREAD ? blockIdx.x : blockIdx.x * GROUPS + gr;
    int i = r / a.nh, s = blockIdx.y;
    const int h = r - i * a.nh;
    // (of a spread row all threads leave or none; GROUPS · LANES may be less than 256)
    if (!SPREAD && gr >= GROUPS) return;
    if (FIND) {
        // i is a row of all sequences': s the last that begins at or before it
        if (i >= a.n_tokens) return;
        int end = a.n_seq;
        while (end - s > 1) {
            const int mid = (s + end) >> 1;
            if (a.q_start[mid] <= i) s = mid;
            else end = mid;
        }
    }
    const int q0 = min(max(a.q_start[s], 0), a.n_tokens), q1 = min(max(a.q_start[s + 1], q0), a.n_tokens);
    if (FIND) i -= q0;
    if (i < 0 || i >= min(q1 - q0, a.max_q)) return;
    const int64_t len = min((int64_t)max(a.kv_len[s], 0), a.max_kv);
    const int n = (int)min((len + a.chunk - 1) / a.chunk, (int64_t)a.nsplit);
    const int64_t row = (int64_t)(q0 + i) * a.nh + h, rows = (int64_t)a.n_tokens * a.nh;
    const float2 *ml = (const float2 *)a.part_ml + row;
    const float *po = a.part_o + row * D + 4 * d4;
    // a range without a key for this row holds zeros at KV_NONE
    float top = KV_NONE;
    if constexpr (SPREAD) {
        for (int k = tid & 63; k < n; k += 64) top = fmaxf(top, ml[k * rows].x);
#pragma unroll
        for (int x = 1; x < 64; x *= 2) top = fmaxf(top, __shfl_xor(top, x, 64));
    } else {
#pragma unroll 4
        for (int k = 0; k < n; k++) top = fmaxf(top, ml[k * rows].x);
    }
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    float sum = 0.f;
    if (gr < GROUPS) {
#pragma unroll 4
        for (int k = SPREAD ? gr : 0; k < n; k += SPREAD ? GROUPS : 1) {
            const float2 m = ml[k * rows];
            const float4 o = *(const float4 *)(po + k * rows * D);
            const float w = m.x == KV_NONE ? 0.f : __builtin_amdgcn_exp2f(m.x - top);
            acc.x = __builtin_fmaf(w, o.x, acc.x);
            acc.y = __builtin_fmaf(w, o.y, acc.y);
            acc.z = __builtin_fmaf(w, o.z, acc.z);
            acc.w = __builtin_fmaf(w, o.w, acc.w);
            sum = __builtin_fmaf(w, m.y, sum);
        }
        if constexpr (SPREAD) {
            acc_lds[gr][d4] = acc;
            if (d4 == 0) sum_lds[gr] = sum;
        }
    }
    if constexpr (SPREAD) {
        __syncthreads();
        if (gr != 0) return;
#pragma unroll
        for (int k = 1; k < GROUPS; k++) {
            const float4 o = acc_lds[k][d4];
            acc.x += o.x, acc.y += o.y, acc.z += o.z, acc.w += o.w;
            sum += sum_lds[k];
        }
    }
    const float inv = sum == 0.f ? 0.f : 1.0f / sum;  // no key at all: zeros
    if constexpr (F32) {
        *(float4 *)((float *)a.o + row * D + 4 * d4) = make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
    } else {
        typedef _Float16 h4 __attribute__((ext_vector_type(4)));
        *(h4 *)((_Float16 *)a.o + row * D + 4 * d4) =
            h4{(_Float16)(acc.x * inv), (_Float16)(acc.y * inv), (_Float16)(acc.z * inv), (_Float16)(acc.w * inv)};
    }
}

// f<Q, NB>() for the cache's type and head dim
template <typename F>
hipError_t by_layout(const KvCache &c, F &&f) {
    auto nb = [&](auto q) {
        switch (c.D) {
            case 32: return f(q, std::integral_constant<int, 1>{});
            case 64: return f(q, std::integral_constant<int, 2>{});
            case 96: return f(q, std::integral_constant<int, 3>{});
            case 128: return f(q, std::integral_constant<int, 4>{});
            case 256: return f(q, std::integral_constant<int, 8>{});
            default: return hipErrorInvalidValue;
        }
    };
    if (c.type == S3E_TYPE_Q4_0) return nb(std::integral_constant<int, 4>{});
    if (c.type == S3E_TYPE_Q8_0) return nb(std::integral_constant<int, 8>{});
    return hipErrorInvalidValue;
}

}  // namespace

hipError_t launch_kv_write(const KvWriteArgs &a, bool f32, hipStream_t st) {
    const dim3 grid((a.n + KV_ROWS - 1) / KV_ROWS, a.c.heads, 2);
    return by_layout(a.c, [&](auto q, auto nb) {
        if (f32) hipLaunchKernelGGL((k_kv_write<q(), nb(), float>), grid, dim3(256), 0, st, a);
        else hipLaunchKernelGGL((k_kv_write<q(), nb(), _Float16>), grid, dim3(256), 0, st, a);
        return hipGetLastError();
    });
}

hipError_t launch_kv_read(const KvReadArgs &a, bool f32, hipStream_t st) {
    const dim3 grid((a.n + KV_ROWS - 1) / KV_ROWS, a.c.heads, 2);
    return by_layout(a.c, [&](auto q, auto nb) {
        if (f32) hipLaunchKernelGGL((k_kv_read<q(), nb(), float>), grid, dim3(256), 0, st, a);
        else hipLaunchKernelGGL((k_kv_read<q(), nb(), _Float16>), grid, dim3(256), 0, st, a);
        return hipGetLastError();
    });
}

hipError_t launch_kv_combine(const KvAttnArgs &a, bool f32, hipStream_t st) {
    auto go = [&](auto d, auto f) {
        constexpr int GROUPS = 256 / (d() / 4);
        // rows of each sequence up to max_q, or, where that is over twice as many as
        // there are, of all sequences, each of which is looked up
        const bool find = a.n_seq > 1 && (int64_t)a.n_seq * a.max_q > 2 * (int64_t)a.n_tokens;
        const int64_t rows = (int64_t)(find ? a.n_tokens : a.max_q) * a.nh;
        auto run = [&](auto spread, auto look) {
            const dim3 grid((unsigned)(spread() ? rows : (rows + GROUPS - 1) / GROUPS), find ? 1 : a.n_seq);
            hipLaunchKernelGGL((k_kv_combine<d(), f(), spread(), look()>), grid, dim3(256), 0, st, a);
        };
        auto by_find = [&](auto spread) { find ? run(spread, std::true_type{}) : run(spread, std::false_type{}); };
        a.nsplit > 8 ? by_find(std::true_type{}) : by_find(std::false_type{});
        return hipGetLastError();
    };
    auto by = [&](auto d) { return f32 ? go(d, std::true_type{}) : go(d, std::false_type{}); };
    switch (a.c.D) {
        case 32: return by(std::integral_constant<int, 32>{});
        case 64: return by(std::integral_constant<int, 64>{});
        case 96: return by(std::integral_constant<int, 96>{});
        case 128: return by(std::integral_constant<int, 128>{});
        case 256: return by(std::integral_constant<int, 256>{});
        default: return hipErrorInvalidValue;
    }
}

}  // namespace s3e
