// k_kv.hip — writing rows into the quantized key/value cache, reading them
// back, and joining attention's partial results over key ranges.
#include "k_kv.h"

namespace s3e {
namespace {

typedef _Float16 h8 __attribute__((ext_vector_type(8)));

// Eight consecutive values of a row.
template <typename T>
__device__ __forceinline__ void load8(const T *p, int vec, float *v) {
    if constexpr (sizeof(T) == 2) {
        if (vec) {
            const h8 x = *(const h8 *)p;
#pragma unroll
            for (int j = 0; j < 8; j++) v[j] = (float)x[j];
            return;
        }
    } else {
        if (vec) {
            const float4 x = *(const float4 *)p, y = *(const float4 *)(p + 4);
            v[0] = x.x, v[1] = x.y, v[2] = x.z, v[3] = x.w;
            v[4] = y.x, v[5] = y.y, v[6] = y.z, v[7] = y.w;
            return;
        }
    }
#pragma unroll
    for (int j = 0; j < 8; j++) v[j] = (float)p[j];
}

// The codes of one 32-channel block held as 8 values by each of 4 neighbouring
// lanes (in channel order), as ggml's quantize_row_q4_0 (d = max / −8, max the
// first value of largest magnitude; q = min(15, ⌊x/d + 8.5⌋)) and the engine's
// Q8_0 conversion (d = amax / 127, q = round-half-even(x·(127/amax))) choose
// them in fp32.  A block with an infinity or a NaN gets a NaN scale, so that
// all of it reads back as NaN.  codes: bytes 0..15, or int8 bits.
template <int Q>
__device__ __forceinline__ void quant_block(const float *v, int lane, uint32_t *codes, uint16_t &scale) {
    uint32_t top = 0;
    float lead = 0.f;
#pragma unroll
    for (int j = 0; j < 8; j++) {
        const uint32_t a = __float_as_uint(v[j]) & 0x7fffffffu;
        if (a > top) {
            top = a;
            lead = v[j];
        }
    }
#pragma unroll
    for (int x = 1; x <= 2; x *= 2) {
        const uint32_t ot = __shfl_xor(top, x, 64);
        const float ol = __shfl_xor(lead, x, 64);
        if (ot > top || (ot == top && (lane & x))) {
            top = ot;
            lead = ol;
        }
    }
    const bool finite = top < 0x7f800000u;
    float d, id;
    if constexpr (Q == 4) {
        d = lead / -8.0f;
        id = d != 0.f ? 1.0f / d : 0.f;
    } else {
        const float amax = __uint_as_float(top);
        d = amax / 127.0f;
        id = top ? 127.0f / amax : 0.f;
    }
    // (a scale whose reciprocal overflows is far below fp16's smallest: zero)
    if (!finite || __builtin_isinf(id)) id = 0.f;
    scale = finite ? half_bits(d) : (uint16_t)0x7e00;
#pragma unroll
    for (int j = 0; j < 8; j++) {
        const float x = finite ? v[j] * id : 0.f;
        if constexpr (Q == 4) codes[j] = (uint32_t)min(15, (int)(x + 8.5f));
        else codes[j] = (uint32_t)(int)__builtin_rintf(x) & 0xffu;
    }
}

template <int Q>
__device__ __forceinline__ uint64_t pack_word(const uint32_t *c) {
    uint64_t x = 0;
#pragma unroll
    for (int j = 0; j < 8; j++)
        x |= (uint64_t)c[j] << (Q == 4 ? 4 * ((j >> 1) + 4 * (j & 1)) : 8 * j);
    return x;
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
// rows again); a row outside any run replaces its own code in each word, a
// nibble by an atomic and and or, a byte by a byte store, so that runs, lone
// rows and neighbouring work-groups never write each other's codes.
// Bound by HBM: the rows are read once and the words written once.
template <int Q, int NB, typename T>
__global__ __launch_bounds__(256) void k_kv_write(KvWriteArgs a) {
    using C = KvChunk<Q, NB>;
    constexpr int D = 32 * NB;
    // rows −7 .. 64 + 13 of the call's slots around this work-group's
    __shared__ int32_t sl[KV_ROWS + 21];
    __shared__ uint8_t codes_lds[(KV_ROWS + 7) * D];
    __shared__ int starts[KV_ROWS / 8 + 1];
    const int tid = threadIdx.x, lane = tid & 63, head = blockIdx.y;
    const bool is_v = blockIdx.z != 0;
    const int64_t r0 = (int64_t)blockIdx.x * KV_ROWS;
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
    const T *x = (const T *)(is_v ? a.x[1] : a.x[0]);
    const int64_t st = is_v ? a.st[1] : a.st[0], sh = is_v ? a.sh[1] : a.sh[0];
    const int vec = is_v ? a.vec[1] : a.vec[0];
    const int g = tid & 3;

    if (!is_v) {
        const int r = tid >> 2, s = sl[r + 7];
        if (s < 0) return;  // (the four lanes of a row together)
        float v[NB][8];
#pragma unroll
        for (int b = 0; b < NB; b++) load8<T>(x + (r0 + r) * st + head * sh + 32 * b + 8 * g, vec, v[b]);
        uint8_t *ck = chunk_of(a.c, s, head, C::BYTES);
        const int key = s & 31, t = (key >> 2) & 1, row = 4 * (key >> 3) + (key & 3);
        uint64_t w[NB];
#pragma unroll
        for (int b = 0; b < NB; b++) {
            uint32_t c[8];
            uint16_t d;
            quant_block<Q>(v[b], lane, c, d);
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

    // V: own rows, then those of the next work-group that a run from here ends in
    auto convert = [&](int r, bool own) {
        const int s = sl[r + 7];
        if (s < 0) return;
        const bool run = in_run(r);
        if (!own && !(run && r - (s & 7) < KV_ROWS)) return;
        float v[NB][8];
#pragma unroll
        for (int b = 0; b < NB; b++) load8<T>(x + (r0 + r) * st + head * sh + 32 * b + 8 * g, vec, v[b]);
        uint8_t *cv = chunk_of(a.c, s, head, C::BYTES) + C::HALF;
        const int key = s & 31;
#pragma unroll
        for (int b = 0; b < NB; b++) {
            uint32_t c[8];
            uint16_t d;
            quant_block<Q>(v[b], lane, c, d);
            if (own && g == (b & 3)) *(uint16_t *)(cv + C::CODES + (b * 32 + key) * 2) = d;
            if (run) {
                uint2 y = make_uint2(0, 0);
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    y.x |= c[j] << (8 * j);
                    y.y |= c[4 + j] << (8 * j);
                }
                *(uint2 *)(codes_lds + r * D + 32 * b + 8 * g) = y;
            } else {
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const int ch = 32 * b + 8 * g + j, k8 = key & 7;
                    uint8_t *p = cv + C::word(ch >> 4, 16 * (key >> 3) + (ch & 15));
                    if constexpr (Q == 4) {
                        const int sft = 4 * ((k8 >> 1) + 4 * (k8 & 1));
                        atomicAnd((uint32_t *)p, ~(15u << sft));
                        atomicOr((uint32_t *)p, c[j] << sft);
                    } else {
                        p[k8] = (uint8_t)c[j];
                    }
                }
            }
        }
    };
    convert(tid >> 2, true);
    if (tid < 28) convert(KV_ROWS + (tid >> 2), false);
    if (tid < 64) {
        const bool first = (sl[tid + 7] & 7) == 0 && in_run(tid);
        const uint64_t m = __ballot(first);
        if (first) starts[1 + __popcll(m & ((1ull << tid) - 1))] = tid;
        if (tid == 0) starts[0] = __popcll(m);
    }
    __syncthreads();
    // whole words: unit (run, piece, channel m of 16)
    const int units = starts[0] * C::PIECES * 16;
    for (int u = tid; u < units; u += 256) {
        const int m = u & 15, pi = (u >> 4) % C::PIECES, r = starts[1 + (u >> 4) / C::PIECES];
        const int s = sl[r + 7];
        uint8_t *cv = chunk_of(a.c, s, head, C::BYTES) + C::HALF;
        const int lane16 = 16 * ((s & 31) >> 3) + m;
        uint64_t w[C::PER];
#pragma unroll
        for (int i = 0; i < C::PER; i++) {
            const int ww = pi * C::PER + i;
            uint32_t c[8];
#pragma unroll
            for (int j = 0; j < 8; j++) c[j] = ww < C::WORDS ? codes_lds[(r + j) * D + 16 * ww + m] : 0;
            w[i] = pack_word<Q>(c);
        }
        if (C::width(pi) == C::PER) {
            uint4 y;
            if constexpr (Q == 4) y = make_uint4((uint32_t)w[0], (uint32_t)w[1], (uint32_t)w[2], (uint32_t)w[3]);
            else y = make_uint4((uint32_t)w[0], (uint32_t)(w[0] >> 32), (uint32_t)w[1], (uint32_t)(w[1] >> 32));
            *(uint4 *)(cv + C::word(pi * C::PER, lane16)) = y;
        } else {
#pragma unroll
            for (int i = 0; i < C::PER; i++)
                if (i < C::width(pi)) store_word<Q>(cv + C::word(pi * C::PER + i, lane16), w[i]);
        }
    }
}

template <int Q>
__device__ __forceinline__ int code_of(uint64_t w, int j) {
    if constexpr (Q == 4) return (int)((w >> (4 * ((j >> 1) + 4 * (j & 1)))) & 15) - 8;
    else return (int)(int8_t)(w >> (8 * j));
}
template <int Q>
__device__ __forceinline__ uint64_t load_word(const uint8_t *p) {
    if constexpr (Q == 4) return *(const uint32_t *)p;
    else return *(const uint64_t *)p;
}

// One tensor (blockIdx.z) of 64 rows and one head: thread 4r + g gives K's
// channels 32b + 8g .. + 8 of row r (its words), or V's channels 16w + 4g .. + 4
// (a code of each of their words; the eight rows of a run read the same words,
// from L1).  A slot outside the cache reads as zeros.  Bound by HBM.
template <int Q, int NB, typename T>
__global__ __launch_bounds__(256) void k_kv_read(KvReadArgs a) {
    using C = KvChunk<Q, NB>;
    constexpr int D = 32 * NB;
    const int tid = threadIdx.x, head = blockIdx.y, g = tid & 3;
    const bool is_v = blockIdx.z != 0;
    T *y = (T *)(is_v ? a.y[1] : a.y[0]);
    const int64_t r = (int64_t)blockIdx.x * KV_ROWS + (tid >> 2);
    if (!y || r >= a.n) return;
    const int64_t s = a.slots[r];
    const bool in = s >= 0 && s < a.c.slots;
    const uint8_t *ck = chunk_of(a.c, in ? s : 0, head, C::BYTES) + (is_v ? C::HALF : 0);
    const int key = (int)(s & 31);
    y += (r * a.c.heads + head) * D;
    // each value once: code · scale in fp32 (exact), rounded to the row's type
    auto value = [&](int code, uint16_t d) { return in ? (float)code * (float)__builtin_bit_cast(_Float16, d) : 0.f; };
    if (!is_v) {
        const int t = (key >> 2) & 1, row = 4 * (key >> 3) + (key & 3);
#pragma unroll
        for (int b = 0; b < NB; b++) {
            const uint64_t w = load_word<Q>(ck + C::word(t * NB + b, 16 * g + row));
            const uint16_t d = *(const uint16_t *)(ck + C::CODES + (b * 32 + key) * 2);
            float v[8];
#pragma unroll
            for (int j = 0; j < 8; j++) v[j] = value(code_of<Q>(w, j), d);
            T *o = y + 32 * b + 8 * g;
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
        return;
    }
#pragma unroll
    for (int w = 0; w < C::WORDS; w++) {
        const uint16_t d = *(const uint16_t *)(ck + C::CODES + ((w >> 1) * 32 + key) * 2);
        float v[4];
#pragma unroll
        for (int i = 0; i < 4; i++)
            v[i] = value(code_of<Q>(load_word<Q>(ck + C::word(w, 16 * (key >> 3) + 4 * g + i)), key & 7), d);
        T *o = y + 16 * w + 4 * g;
        if constexpr (sizeof(T) == 2) {
            typedef _Float16 h4 __attribute__((ext_vector_type(4)));
            *(h4 *)o = h4{(_Float16)v[0], (_Float16)v[1], (_Float16)v[2], (_Float16)v[3]};
        } else {
            *(float4 *)o = make_float4(v[0], v[1], v[2], v[3]);
        }
    }
}

// Output rows (query, head) from their key ranges: each range's unnormalised
// output and sum are in units of 2^reference.  D/4 threads hold a row.  Where a
// row has many ranges a work-group takes one row (SPREAD), its other threads
// further ranges, joined in LDS in a fixed order; where it has few, a row each.
template <int D, bool F32, bool SPREAD>
__global__ __launch_bounds__(256) void k_kv_combine(KvAttnArgs a) {
    constexpr int LANES = D / 4, GROUPS = 256 / LANES;
    __shared__ float4 acc_lds[SPREAD ? GROUPS : 1][LANES];
    __shared__ float sum_lds[GROUPS];
    const int tid = threadIdx.x, s = blockIdx.y;
    const int q0 = min(max(a.q_start[s], 0), a.n_tokens), q1 = min(max(a.q_start[s + 1], q0), a.n_tokens);
    const int gr = tid / LANES, d4 = tid % LANES;
    const int r = SPREAD ? blockIdx.x : blockIdx.x * GROUPS + gr;
    const int i = r / a.nh, h = r - i * a.nh;
    // (of a spread row all threads leave or none; GROUPS · LANES may be less than 256)
    if (i >= min(q1 - q0, a.max_q) || (!SPREAD && gr >= GROUPS)) return;
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
        const int64_t rows = (int64_t)a.max_q * a.nh;
        if (a.nsplit > 8)
            hipLaunchKernelGGL((k_kv_combine<d(), f(), true>), dim3((unsigned)rows, a.n_seq), dim3(256), 0, st, a);
        else
            hipLaunchKernelGGL((k_kv_combine<d(), f(), false>), dim3((unsigned)((rows + GROUPS - 1) / GROUPS), a.n_seq), dim3(256), 0, st, a);
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
