// The 4-bit row cache's record layout and code words (lf_int4_layer), shared by its kernels.
#pragma once

#include "decode_common.hpp"

namespace lf {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
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

// Nibble e of a code word is in bits 4 e + 3 .. 4 e + 6, the last one wrapping to bits 31, 0, 1, 2: with the
// word turned by 4 e bits, nibbles e and e + 4 are the upper four mantissa bits of the bf16 halves
// 0x4180 | code << 3 = 16 + code, without a shift of their own.
__device__ __forceinline__ uint32_t turn(uint32_t w, int bits) { return __builtin_amdgcn_alignbit(w, w, bits); }
__device__ __forceinline__ uint32_t code_at(uint32_t w, int e) { return turn(w, (4 * e + 3) & 31) & 15u; }

// Bits of nibble e of a word.
__device__ __forceinline__ uint32_t nibble_bits(uint32_t code, int e) { return turn(code, (32 - (4 * e + 3)) & 31); }

// A word's eight codes as bf16 16 + code; element 2 i is nibble i, element 2 i + 1 nibble i + 4.
constexpr float kCodeBias = 16.f;
__device__ __forceinline__ bf16x8 codes8(uint32_t w) {
    constexpr uint32_t mask = 0x00780078u, base = 0x41804180u;
    return __builtin_bit_cast(bf16x8, u32x4{(w & mask) | base, (turn(w, 4) & mask) | base, (turn(w, 8) & mask) | base,
                                            (turn(w, 12) & mask) | base});
}

// A Key row's word w (channels 8 w .. 8 w + 7) and a Value block's word of (token, channel), in words.
__host__ __device__ constexpr int key_word(int D, int w) { return (w & 3) * (D / 32) + (w >> 2); }
__host__ __device__ constexpr int value_word(int tok, int c) {
    return (((c >> 6) * 64 + ((tok & 15) >> 2) * 16 + (c & 15)) << 2) + ((c >> 4) & 3);
}
__host__ __device__ constexpr int value_nibble(int tok) { return (tok & 3) + 4 * (tok >> 4); }

// Record ``block`` of (sequence b, kv head h).
__device__ __forceinline__ uint8_t* int4_block(const lf_int4_layer& L, int b, int h, int block, int bytes) {
    return L.blocks + ((static_cast<int64_t>(b) * L.n_kv + h) * (L.cap_tokens / kBlock) + block) * bytes;
}

__device__ __forceinline__ int int4_len(const lf_int4_layer& L, int b) {
    return min(max(L.lens[b], 0), L.cap_tokens);
}

__device__ __forceinline__ float pair_scale(uint32_t sm) { return f16_to_f32(static_cast<uint16_t>(sm)); }
__device__ __forceinline__ float pair_min(uint32_t sm) { return f16_to_f32(static_cast<uint16_t>(sm >> 16)); }

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
