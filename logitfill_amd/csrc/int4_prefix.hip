// Attention of many query rows over the 4-bit row cache: the records that every query of a 128-row tile sees (a
// prompt's chunk over what is in front of it).
//
// Per record the general kernel's waves unpack the codes and form scale and minimum terms for 16 rows each.  Here the
// workgroup unpacks a record once, by packed fp16 arithmetic, into LDS, in the order in which the products' lanes read it, and
// its four waves take it for 32 rows each, on v_mfma_f32_16x16x32_f16:
//     S_t = sum_g scale_t,g (code_t,g . q_g) + min_t,g sum(q_g),  p = 2^(S c - ref),  O^T = V^T . P^T,  l = sum p.
// Keys enter as their codes, which fp16 holds, and scale and minimum in fp32 as in the general kernel: as fp16 s * code + m a
// Key was off by 2^-12 of itself, which beside a channel that is large in every token (a bias of 400) moved weights by a
// hundredth and more.  (In two exact fp16 parts, scale * code, Keys take twice the LDS reads and products: 263 us in
// place of 222 below.)  With several groups, the minima's terms are a product of their own, sixteen deep, of the fp16 factors as
// they stand and the queries' sums in two fp16 parts (2^-22 of them); with one group of 128 they are a sum per score, for
// the product's registers spill (223 us against 238).
// A query row is scaled by a power of two so that its largest element lies in [1, 2); the factor goes into c.  Values enter as
// fp16 s * code + m, times a power of two of the split's, off by 2^-12 of their size, and so does a weight p; against bf16's
// rounding of the output that is little (rel. error 1.66e-3 to 1.69e-3, its own 1.64e-3 to 1.66e-3), against fp16's it is not,
// so bf16 rows alone come here.
//
// 512 queries of 28 / 4 heads of 128 over 16 384 tokens, groups of 128 / 64 / 32: calls of 222 / 237 / 266 us where the general
// kernel alone takes 273 / 324 / 417; 14 / 2 heads of 64, groups of 64 / 32: 85 / 91 and 105 / 136.
//
// Double-buffered: a record's codes are loaded into registers two records ahead (a lane's sixteen bytes are exactly
// what it turns into operands), dequantised one ahead, one barrier per record.
#include "int4_common.hpp"

namespace lf {
namespace {

// A weight is formed as up to 2^15: 2^7 where the reference point is, 2^8 before that moves.  fp16 keeps it down to 2^-24,
// 2^-31 of a row's largest, and it takes 2^22 smaller ones to show in bf16.  (With 1 where the reference point is, 131 071
// tokens of 2^-26 each, 2^-9 of their row, were lost.)
constexpr float kHeadroom = 7.f;

constexpr int kWaves = 4, kTile = 16, MT = kManyRows / (kWaves * kTile);  // row tiles of a wave

__device__ __forceinline__ f32x4 mfma(f16x8 a, f16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ uint32_t lower_pair(uint32_t a, uint32_t b) { return __builtin_amdgcn_perm(b, a, 0x05040100u); }
__device__ __forceinline__ uint32_t upper_pair(uint32_t a, uint32_t b) { return __builtin_amdgcn_perm(b, a, 0x07060302u); }

// A word's eight codes in fp16, element pairs (nibble i, nibble i + 4).  The fp16 bits of a Key word's, 0x5800 | code << 3,
// are 128 + code; of a Value word's, 0x4C00 | code << 6, 16 + code.
template <uint32_t Mask>
__device__ __forceinline__ f16x2 code_pair(const u32x4& bits, int i) {
    constexpr _Float16 bias = static_cast<_Float16>(Mask == kKeyMask ? 128 : 16);
    const uint32_t pair = bits[i];
    return __builtin_bit_cast(f16x2, pair) - f16x2{bias, bias};
}
// A Key word's codes.
__device__ __forceinline__ u32x4 keys8(uint32_t w, uint32_t base) {
    const u32x4 bits = codes8<kKeyMask>(w, base);
    u32x4 r;
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = __builtin_bit_cast(uint32_t, code_pair<kKeyMask>(bits, i));
    return r;
}
// A Value word's codes times s[i] plus m[i].
__device__ __forceinline__ u32x4 values8(uint32_t w, const f16x2 (&s)[4], const f16x2 (&m)[4], uint32_t base) {
    const u32x4 bits = codes8<kValueMask>(w, base);
    u32x4 r;
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(code_pair<kValueMask>(bits, i), s[i], m[i]));
    return r;
}
// LDS reads stay behind this point: hoisted to a record's start they take more registers than three waves a SIMD leave.
__device__ __forceinline__ void phase() { asm volatile("" ::: "memory"); }
__device__ __forceinline__ f16x2 halves(uint32_t x) { return __builtin_bit_cast(f16x2, x); }

template <int D, int GROUP>
__global__ __launch_bounds__(kWaves * kWave, D == 128 && GROUP < 128 ? 2 : 3) void int4_prefix_kernel(Int4Attention a) {
    using R = Int4Rec<D, GROUP>;
    constexpr int G = R::G, CH = R::chunks, VT = D / 16;
    constexpr bool kOne = D == 128 && G == 1;  // the minima's terms by sums
    constexpr int kK = 2 * CH * kWave, kV = VT * kWave;  // 16-byte pieces of a record's Keys and Values
    __shared__ u32x4 lds[2][kK + kV];
    __shared__ __attribute__((aligned(16))) uint32_t key_pairs[2][G * kBlock];  // Keys' scales and minima
    __shared__ float widest[kWaves];
    const int h = blockIdx.x % a.L.n_kv, tile = blockIdx.x / a.L.n_kv, b = blockIdx.y, part = blockIdx.z;
    const int lane = threadIdx.x % kWave, wave = in_sgpr(static_cast<int>(threadIdx.x / kWave));
    const int col = lane & 15, quad = lane >> 4;
    const uint8_t* base = int4_block(a.L, b, h, 0, R::bytes);
    const int len = int4_len(a.L, b);
    const int n = a.q_lens ? min(max(a.q_lens[b], 0), a.q_len) : a.q_len;
    const int records = prefix_records(a, len, n, tile);
    const int per = (records + a.prefix - 1) / a.prefix, first = min(part * per, records), last = min(first + per, records);

    // 2^up takes the split's largest Value to 2^14 .. 2^15: read back a Value reaches 16 * 65 504, fp16's infinity, and 2^-14 is
    // where fp16 begins to lose bits.  (One that is not finite takes no part.)  The scales and minima are read twice for it: 3, 5
    // and 9 us of the calls above with groups of 128, 64 and 32.
    float most_value = 0.f;
    for (int k = threadIdx.x; k < (last - first) * 8 * G; k += kWaves * kWave) {
        const u32x4 pair = reinterpret_cast<const u32x4*>(base + static_cast<int64_t>(first + k / (8 * G)) * R::bytes + R::vsm)[k % (8 * G)];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float m = pair_min(pair[i]), v = fmaxf(fabsf(m), fabsf(fmaf(15.f, pair_scale(pair[i]), m)));
            most_value = fmaxf(most_value, v < 4e6f ? v : 0.f);
        }
    }
    most_value = wave_max(most_value);
    if (lane == 0) widest[wave] = most_value;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWaves; ++w) most_value = fmaxf(most_value, widest[w]);
    const int up = in_sgpr(min(max(141 - static_cast<int>(__float_as_uint(most_value) >> 23), -14), 15));
    const f16x2 raise = halves(static_cast<uint32_t>(15 + up) * 0x04000400u);

    // This wave's share of a record: 0, 1: sixteen Key rows; 2, 3: half of a lane's Value words.
    constexpr int VW = VT / 2;                          // a lane's Value words
    constexpr int VG = GROUP == 32 ? VW / 2 : 1;        // and the groups they lie in
    const uint32_t code_base = in_vgpr(wave < 2 ? kKeyBaseHalf : kValueBase);  // (a wave stages Keys or Values)
    constexpr int NP = 2 * VG > G ? 2 * VG : G;
    // Every wave loads the same pieces, whichever it stages: with a branch around the loads, what it joins waited for them.
    struct Raw {
        uint32_t w[4];
        u32x4 pair[NP];  // scale and minimum: [g][0] a Key row's, or a Value word's of tokens 4 quad .. and 16 + 4 quad ..
    };
    const int half = wave & 1;
    const uint32_t word_at = wave < 2 ? (16 * half + col) * (D / 2) + CH * 4 * quad
                                      : R::v + 16 * lane + (VW == 4 ? 1024 * half : 8 * half);
    const uint32_t key_at = R::ksm + 4 * (16 * half + col);
    // (head_dim 64: words 2 half, 2 half + 1 are of group half with groups of 32)
    const uint32_t value_at = R::vsm + 16 * quad + 4 * kBlock * (GROUP == 32 ? VG * half : 64 * half * (VW / 4) / GROUP);
    const auto load = [&](int record, Raw& r) {
        const uint8_t* rec = base + static_cast<int64_t>(record) * R::bytes;
        if constexpr (CH == 4) {
            const u32x4 x = *reinterpret_cast<const u32x4*>(rec + word_at);
#pragma unroll
            for (int c = 0; c < 4; ++c) r.w[c] = x[c];
        } else {
            const u32x2 x = *reinterpret_cast<const u32x2*>(rec + word_at);
            r.w[0] = x[0];
            r.w[1] = x[1];
        }
#pragma unroll
        for (int k = 0; k < NP; ++k) {
            const uint32_t at = wave < 2 ? key_at + 4 * kBlock * min(k, G - 1) : value_at + 4 * kBlock * (k >> 1) + 64 * (k & 1);
            __builtin_memcpy(&r.pair[k], __builtin_assume_aligned(rec + at, 4), 16);
        }
    };
    const auto stage = [&](const Raw& r, u32x4* to, uint32_t* pairs) {
        if (wave < 2) {
#pragma unroll
            for (int c = 0; c < CH; ++c) to[(half * CH + c) * kWave + lane] = keys8(r.w[c], code_base);
            if (quad == 0)
#pragma unroll
                for (int g = 0; g < G; ++g) pairs[g * kBlock + 16 * half + col] = r.pair[g][0];
        } else {
#pragma unroll
            for (int k = 0; k < VG; ++k) {
                f16x2 s[4], m[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    s[i] = halves(lower_pair(r.pair[2 * k][i], r.pair[2 * k + 1][i])) * raise;
                    m[i] = halves(upper_pair(r.pair[2 * k][i], r.pair[2 * k + 1][i])) * raise;
                }
#pragma unroll
                for (int c = k * (VW / VG); c < (k + 1) * (VW / VG); ++c)
                    to[kK + (half * VW + c) * kWave + lane] = values8(r.w[c], s, m, code_base);
            }
        }
    };

    // rows (head of the group, token), tokens fastest: this lane's, one of each row tile
    f16x8 q[MT][CH];
    f16x4 qsum[MT];  // the query's sum over lane quad's group: 0 (for the scale), upper part, 0, lower part
    float qall[MT];  // or over the one group
    float scale[MT], ref[MT], limit[MT];  // limit: how far a score may pass ref; -inf until one is seen
    const bool flip = a.qscale < 0.f;
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        const int r = tile * kManyRows + (wave * MT + t) * kTile + col, i = r / a.q_len, j = r % a.q_len;
        float x[CH][8] = {}, most = 0.f;
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            if (i < a.g) query8<LF_BF16>(a, b * a.qb + static_cast<int64_t>(h * a.g + i) * a.qh + j * a.qt + 32 * c + 8 * quad, x[c]);
#pragma unroll
            for (int e = 0; e < 8; ++e) most = fmaxf(most, fabsf(x[c][e]));
        }
        most = rows_max(most);
        // 2^-exponent of the largest element (an all-zero or subnormal row: 2^126)
        const int exponent = static_cast<int>(__float_as_uint(most) >> 23);
        const float down = __uint_as_float(static_cast<uint32_t>(min(max(254 - exponent, 1), 253)) << 23);
        scale[t] = fmaxf(fabsf(a.qscale) / down, 1e-37f);
        float sums[G] = {}, mine = 0.f;
#pragma unroll
        for (int c = 0; c < CH; ++c)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                // operand element 2 i is channel i of the word, element 2 i + 1 channel 4 + i
                const float v = x[c][(e >> 1) + 4 * (e & 1)] * down;
                q[t][c][e] = static_cast<_Float16>(flip ? -v : v);
                sums[c / (CH / G)] += flip ? -v : v;
            }
#pragma unroll
        for (int g = 0; g < G; ++g) {
            const float sum = rows_sum(sums[g]);  // (in every quad)
            mine = kOne || quad == g ? sum : mine;
        }
        qall[t] = mine;
        const _Float16 upper = static_cast<_Float16>(mine);
        qsum[t] = f16x4{0, upper, 0, static_cast<_Float16>(mine - static_cast<float>(upper))};
        ref[t] = 0.f;
        limit[t] = -__builtin_inff();
    }
    f32x4 o[MT][VT];
    float l[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        l[t] = 0.f;
#pragma unroll
        for (int v = 0; v < VT; ++v) o[t][v] = f32x4{0.f, 0.f, 0.f, 0.f};
    }

    Raw raw;
    if (first < last) {
        load(first, raw);
        stage(raw, lds[0], key_pairs[0]);
        load(min(first + 1, last - 1), raw);
    }
    __syncthreads();
    for (int k = first; k < last; ++k) {
        const u32x4* rec = lds[(k - first) & 1];
        const uint32_t* pairs = key_pairs[(k - first) & 1];
        if (k + 1 < last) {
            stage(raw, lds[(k + 1 - first) & 1], key_pairs[(k + 1 - first) & 1]);
            load(min(k + 2, last - 1), raw);
        }
        f32x4 y[MT][2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            if constexpr (!kOne) {
                const uint32_t pair = pairs[min(quad, G - 1) * kBlock + 16 * u + col];  // (a quad past the groups: times zero)
                const f16x4 factors = __builtin_bit_cast(f16x4, u32x2{pair, pair});
#pragma unroll
                for (int t = 0; t < MT; ++t) y[t][u] = __builtin_amdgcn_mfma_f32_16x16x16f16(factors, qsum[t], f32x4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
            }
#pragma unroll
            for (int g = 0; g < G; ++g) {
                f32x4 acc[MT];
#pragma unroll
                for (int t = 0; t < MT; ++t) acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int c = g * (CH / G); c < (g + 1) * (CH / G); ++c) {
                    const f16x8 key = __builtin_bit_cast(f16x8, rec[(u * CH + c) * kWave + lane]);
#pragma unroll
                    for (int t = 0; t < MT; ++t) acc[t] = mfma(key, q[t][c], acc[t]);
                }
                const u32x4 pair = *reinterpret_cast<const u32x4*>(pairs + g * kBlock + 16 * u + 4 * quad);
#pragma unroll
                for (int t = 0; t < MT; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        // (a sum with zero where it is a product: it takes the fp16 factor as it is)
                        const float low = kOne ? fmaf(pair_min(pair[i]), qall[t], 0.f) : y[t][u][i];
                        y[t][u][i] = fmaf(pair_scale(pair[i]), acc[t][i], low);
                    }
                phase();
            }
        }
        f16x8 p[MT];
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            // (scaled before they are compared: the comparisons take a product's sums as they are)
            float z[2][4];
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int i = 0; i < 4; ++i) z[u][i] = fmaf(y[t][u][i], scale[t], -ref[t]);
            float most = fmaxf(fmaxf(fmaxf(z[0][0], z[0][1]), fmaxf(z[0][2], z[0][3])),
                               fmaxf(fmaxf(z[1][0], z[1][1]), fmaxf(z[1][2], z[1][3])));
            if (__any(most > limit[t])) {
                most = rows_max(most);
                const bool moves = most > limit[t];
                const float by = moves ? most - kHeadroom : 0.f;
                const float down = limit[t] < 0.f && moves ? 0.f : __builtin_amdgcn_exp2f(-by);
                ref[t] += by;
                limit[t] = moves ? kHeadroom + 8.f : limit[t];
                l[t] *= down;
#pragma unroll
                for (int v = 0; v < VT; ++v) o[t][v] *= down;
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int i = 0; i < 4; ++i) z[u][i] -= by;
            }
            // element 2 i is token i of the lower sixteen, element 2 i + 1 of the upper
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const float e = __builtin_amdgcn_exp2f(z[u][i]);
                    l[t] += e;
                    p[t][2 * i + u] = static_cast<_Float16>(e);
                }
        }
#pragma unroll
        for (int v = 0; v < VT; ++v) {
            const f16x8 value = __builtin_bit_cast(f16x8, rec[kK + v * kWave + lane]);
#pragma unroll
            for (int t = 0; t < MT; ++t) o[t][v] = mfma(value, p[t], o[t][v]);
        }
        __syncthreads();
    }
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        l[t] = rows_sum(l[t]);
        const int r = tile * kManyRows + (wave * MT + t) * kTile + col;  // head of the group * q_len + token
        if (r >= a.g * a.q_len) continue;
        const int64_t at = ((static_cast<int64_t>(b) * a.n_q + h * a.g) * a.q_len + r) * a.parts + part;
        // (a sum of NaN counts as seen; rows behind the sequence's last token are zeros whatever they saw)
        const bool token = r % a.q_len < n;
        if (quad == 0) {
            a.part_ml[2 * at] = token && l[t] != 0.f ? ref[t] : -__builtin_inff();
            a.part_ml[2 * at + 1] = token ? l[t] : 0.f;
        }
        if (!token)
#pragma unroll
            for (int v = 0; v < VT; ++v) o[t][v] = f32x4{0.f, 0.f, 0.f, 0.f};
        const float down = __uint_as_float(static_cast<uint32_t>(127 - up) << 23);
#pragma unroll
        for (int v = 0; v < VT; ++v) o[t][v] *= down;
        each_run<D, GROUP>(o[t], quad, [&](int c, const float (&x)[4]) { store_row<LF_FP32>(a.part_o, at * D + c, x); });
    }
}

}  // namespace

int launch_int4_prefix(const Int4Attention& a, hipStream_t stream) {
    const int tiles = (a.g * a.q_len + kManyRows - 1) / kManyRows;
    const dim3 grid(a.L.n_kv * tiles, a.L.batch, a.prefix);
    const auto launch = [&](auto shape) {
        constexpr int D = decltype(shape)::d, GROUP = decltype(shape)::group;
        hipLaunchKernelGGL((int4_prefix_kernel<D, GROUP>), grid, dim3(kWaves * kWave), 0, stream, a);
        const hipError_t err = hipGetLastError();
        return err == hipSuccess ? LF_OK : static_cast<int>(err);
    };
    switch (a.L.head_dim * 1000 + a.L.group) {
        case 64032: return launch(Int4Shape<64, 32>());
        case 64064: return launch(Int4Shape<64, 64>());
        case 128032: return launch(Int4Shape<128, 32>());
        case 128064: return launch(Int4Shape<128, 64>());
        case 128128: return launch(Int4Shape<128, 128>());
        default: return LF_E_UNSUPPORTED;
    }
}

}  // namespace lf
