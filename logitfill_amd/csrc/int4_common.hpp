// The 4-bit row cache's record layout and code words (lf_int4_layer), shared by its kernels.
#pragma once

#include "decode_common.hpp"

namespace lf {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int kBlock = 32;  // tokens of a record

// Byte offsets of a record's parts.
template <int D, int GROUP>
struct Int4Rec {
    static constexpr int G = D / GROUP;         // groups per row
    static constexpr int chunks = D / 32;       // words of a Key row that one lane of a product takes
    static constexpr int v = 16 * D;            // Key codes: 32 rows of D / 2 bytes
    static constexpr int ksm = 32 * D;
    static constexpr int vsm = ksm + 128 * G;   // G times 32 rows' (scale, min) pairs
    static constexpr int bytes = vsm + 128 * G;
    static_assert(bytes == LF_INT4_BLOCK_BYTES(D, GROUP), "record size");
};

// Nibble e of a Key word is in bits 4 e + 3 .. of it, of a Value word in bits 4 e + 6 .., the last one's upper bits
// wrapping to the lowest: with the word turned by 4 e bits, nibbles e and e + 4 are the upper four mantissa bits of the
// bf16 halves 0x4180 | code << 3 or the fp16 halves 0x4C00 | code << 6, 16 + code, without a shift of their own.
constexpr int kKeyTurn = 3, kValueTurn = 6;
__device__ __forceinline__ uint32_t turn(uint32_t w, int bits) { return __builtin_amdgcn_alignbit(w, w, bits); }
template <int Turn>
__device__ __forceinline__ uint32_t code_at(uint32_t w, int e) { return turn(w, (4 * e + Turn) & 31) & 15u; }

// A constant in a vector register: the and-or of a code's pair takes one literal-free scalar and vector operands (with
// both as literals it is an and, then an or).
__device__ __forceinline__ uint32_t in_vgpr(uint32_t x) {
    asm volatile("" : "+v"(x));
    return x;
}

// A Key word's eight codes as bf16, a Value word's as fp16 16 + code; element 2 i is nibble i, element 2 i + 1 nibble
// i + 4.  ``base``: kKeyBase or kValueBase in a vector register.
constexpr float kCodeBias = 16.f;
constexpr uint32_t kKeyBase = 0x41804180u, kValueBase = 0x4C004C00u, kKeyBaseHalf = 0x58005800u, kKeyMask = 0x00780078u, kValueMask = 0x03C003C0u;
template <uint32_t Mask>
__device__ __forceinline__ u32x4 codes8(uint32_t w, uint32_t base) {
    return u32x4{(w & Mask) | base, (turn(w, 4) & Mask) | base, (turn(w, 8) & Mask) | base, (turn(w, 12) & Mask) | base};
}

// Where a Key row's word w (channels 8 w .. 8 w + 7) stands in it.
__host__ __device__ constexpr int key_word(int D, int w) { return (w & 3) * (D / 32) + (w >> 2); }

// Four consecutive Value words belong to lane (quad, c): of channels 64 s + 4 c + t, or with groups of 32, where a
// product's sixteen channels have to be of one group, 64 s + 32 (t / 2) + 2 c + t % 2.  A row r of tile t of the
// transposed output is then channel value_channel(r, t).
template <int GROUP>
__host__ __device__ constexpr int value_channel(int c, int t) {
    return GROUP == 32 ? 64 * (t >> 2) + 32 * ((t >> 1) & 1) + 2 * c + (t & 1) : 64 * (t >> 2) + 4 * c + (t & 3);
}

constexpr int kInlineSeqs = 64;  // sequences whose numbers travel in one launch's arguments

__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{a, b}, bf16x2));
}
__device__ __forceinline__ uint32_t pack_f16(float a, float b) {
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{a, b}, f16x2));
}

// N (2, 4 or 8) floats to consecutive elements, rounded to nearest.
template <int Dt, int N>
__device__ __forceinline__ void store_row(void* p, int64_t at, const float (&x)[N]) {
    if constexpr (Dt == LF_FP32 && N == 2) {
        *reinterpret_cast<u32x2*>(static_cast<float*>(p) + at) = u32x2{__float_as_uint(x[0]), __float_as_uint(x[1])};
    } else if constexpr (Dt == LF_FP32) {
#pragma unroll
        for (int e = 0; e < N; e += 4) *reinterpret_cast<f32x4*>(static_cast<float*>(p) + at + e) = f32x4{x[e], x[e + 1], x[e + 2], x[e + 3]};
    } else {
        uint32_t w[N / 2];
#pragma unroll
        for (int e = 0; e < N / 2; ++e) w[e] = Dt == LF_BF16 ? pack_bf16(x[2 * e], x[2 * e + 1]) : pack_f16(x[2 * e], x[2 * e + 1]);
        uint16_t* dst = static_cast<uint16_t*>(p) + at;
        if constexpr (N == 8) *reinterpret_cast<u32x4*>(dst) = u32x4{w[0], w[1], w[2], w[3]};
        else if constexpr (N == 2) *reinterpret_cast<uint32_t*>(dst) = w[0];
        else *reinterpret_cast<u32x2*>(dst) = u32x2{w[0], w[1]};
    }
}

// Record ``block`` of (sequence b, kv head h).
__device__ __forceinline__ uint8_t* int4_block(const lf_int4_layer& L, int b, int h, int block, int bytes) {
    return L.blocks + ((static_cast<int64_t>(b) * L.n_kv + h) * (L.cap_tokens / kBlock) + block) * bytes;
}

__device__ __forceinline__ uint16_t* int4_top(const lf_int4_layer& L, int b, int h, int block) {
    return L.tops + (static_cast<int64_t>(b) * L.n_kv + h) * (L.cap_tokens / kBlock) + block;
}

__device__ __forceinline__ int int4_len(const lf_int4_layer& L, int b) {
    return min(max(L.lens[b], 0), L.cap_tokens);
}

__device__ __forceinline__ float pair_scale(uint32_t sm) { return f16_to_f32(static_cast<uint16_t>(sm)); }
__device__ __forceinline__ float pair_min(uint32_t sm) { return f16_to_f32(static_cast<uint16_t>(sm >> 16)); }

// An attention call, as its kernels take it.
struct Int4Attention {
    lf_int4_layer L;
    const void* q;
    int64_t qb, qh, qt;
    int vec;  // query rows start on 16 bytes
    const int32_t* q_lens;
    void* out;
    int n_q, g, q_len;
    float qscale;  // scaling * log2(e)
    const int32_t* pages;
    int n_pages;
    int splits, split_tokens;  // with pages: split_tokens is in records of the page list
    int prefix;                // splits of the many-row kernel in front of them
    int parts;                 // of every output row
    int part0;                 // the first one of this launch
    float* part_o;             // [batch * n_q * q_len][parts][D]
    float* part_ml;            // [batch * n_q * q_len][parts][2]
};

// The same of shared prefixes (the kernels' Shared forms): L holds the prefixes, one for ``each`` sequences in turn, and own the
// sequences.  The general kernel's launch holds shared_blocks workgroups of the prefixes, shared_tiles row tiles each, and
// behind them those of the sequences' own rows.
struct Int4Shared : Int4Attention {
    lf_int4_layer own;
    int each;
    int shared_blocks, shared_tiles, own_tiles, own_splits, own_split_tokens;
};

// Query row ``r`` of a prefix's (sequence, head of the group, token), tokens fastest.
struct SharedRow {
    int b, i, j;   // sequence of the whole batch
    bool real;
};
__device__ __forceinline__ SharedRow shared_row(const Int4Shared& a, int prefix, int r) {
    const int per = a.g * a.q_len, s = r / per, rest = r - s * per, i = rest / a.q_len;
    return {prefix * a.each + s, i, rest - i * a.q_len, s < a.each};
}
// Rows of a prefix of ``len`` that the row's query sees: all of them, unless its sequence is shorter than its queries.
__device__ __forceinline__ int shared_limit(const Int4Shared& a, const SharedRow& row, int len) {
    if (!row.real) return 0;
    const int n = a.q_lens ? min(max(a.q_lens[row.b], 0), a.q_len) : a.q_len;
    const int own = int4_len(a.own, row.b);
    return row.j < n ? min(max(len + own - n + row.j + 1, 0), len) : 0;
}

template <bool Shared> struct Int4Call { using Args = Int4Attention; };
template <> struct Int4Call<true> { using Args = Int4Shared; };

constexpr int kManyRows = 128;  // query rows of a many-row workgroup

// The records in front of everything that some query of many-row tile ``tile`` does not see: rows are (head of the
// group, token), tokens fastest, and a tile of one head starts at its first token.
__device__ __forceinline__ int prefix_records(const Int4Attention& a, int len, int n, int tile) {
    const int r0 = tile * kManyRows, r1 = min(r0 + kManyRows, a.g * a.q_len) - 1;
    const int j = r0 / a.q_len == r1 / a.q_len ? r0 % a.q_len : 0;
    return j < n ? max(len - n + j + 1, 0) / kBlock : 0;
}

// Eight elements of a query row as float32.
template <int Dt>
__device__ __forceinline__ void query8(const Int4Attention& a, int64_t at, float (&x)[8]) {
    if (a.vec) {
        if constexpr (Dt == LF_FP32) {
            const f32x4* p = reinterpret_cast<const f32x4*>(static_cast<const float*>(a.q) + at);
            const f32x4 u = p[0], v = p[1];
#pragma unroll
            for (int e = 0; e < 4; ++e) { x[e] = u[e]; x[4 + e] = v[e]; }
        } else {
            const u32x4 u = *reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(a.q) + at);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const uint16_t h = static_cast<uint16_t>(u[e >> 1] >> (16 * (e & 1)));
                x[e] = Dt == LF_BF16 ? bf16_to_f32(h) : f16_to_f32(h);
            }
        }
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = load_as_f32(a.q, at + e, Dt);
    }
}

// fn(channel, values) for every four consecutive channels that a lane of the transposed output holds.
template <int D, int GROUP, class Fn>
__device__ __forceinline__ void each_run(const f32x4 (&o)[D / 16], int quad, Fn&& fn) {
    constexpr int N = GROUP == 32 ? 2 : 4;  // tiles whose rows' channels are neighbours
#pragma unroll
    for (int t = 0; t < D / 16; t += N)
#pragma unroll
        for (int k = 0; k < N; ++k) {
            float x[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = o[t + e % N][(4 * k + e) / N];
            fn(value_channel<GROUP>(4 * quad + 4 * k / N, t), x);
        }
}

// Calls fn(Int4Shape<D, GROUP>) for a layer's shape; LF_E_UNSUPPORTED for any other.
template <int D, int GROUP>
struct Int4Shape {
    static constexpr int d = D, group = GROUP;
};
template <class Fn>
int int4_dispatch(const lf_int4_layer& L, Fn&& fn) {
    switch (L.head_dim * 1000 + L.group) {
        case 64032: return fn(Int4Shape<64, 32>());
        case 64064: return fn(Int4Shape<64, 64>());
        case 128032: return fn(Int4Shape<128, 32>());
        case 128064: return fn(Int4Shape<128, 64>());
        case 128128: return fn(Int4Shape<128, 128>());
        case 256032: return fn(Int4Shape<256, 32>());
        case 256064: return fn(Int4Shape<256, 64>());
        case 256128: return fn(Int4Shape<256, 128>());
        default: return LF_E_UNSUPPORTED;
    }
}

}  // namespace lf
