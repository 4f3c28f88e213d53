// Attention of many query rows over the 4-bit row cache: the records that every query of a 128-row tile sees (a
// prompt's chunk over what is in front of it).
//
// Per record the general kernel's waves unpack the codes and form scale and minimum terms for 16 rows each.  Here the
// workgroup dequantises a record once -- Keys and Values as fp16 s * code + m, by packed fp16 arithmetic -- into LDS,
// in the order in which the products' lanes read it, and its four waves take it for 32 rows each:
//     S^T = K . Q^T,  p = 2^(S c - ref),  O^T = V^T . P^T,  l = 1 . P^T   on v_mfma_f32_16x16x32_f16.
// A query row is scaled by a power of two so that its largest element lies in [1, 2); the factor goes into c.  The
// fp16 steps: a Key and a Value element are off by 2^-12 of their size (a Key's error in a score is that of a sum of
// head_dim independent ones), a weight p by 2^-12; l is the sum of the rounded weights.  Against bf16's rounding of the
// output that is little (rel. error 1.7e-3 to 1.8e-3, at head_dim 64 2.2e-3, its own 1.65e-3); against fp16's it is not
// (4e-4 to 1.5e-3 against 2.1e-4), so bf16 rows alone come here.
//
// 512 queries of 28 / 4 heads of 128 over 16 384 tokens, groups of 128: 150 us of the call's 175, 0.8 PFLOP/s; matrix cores 34 %, VALU
// 47 % and LDS 41 % busy: the operands' LDS reads and the softmax beside the products, two workgroups a CU.
//
// Double-buffered: a record's codes are loaded into registers two records ahead (a lane's sixteen bytes are exactly
// what it turns into operands), dequantised one ahead, one barrier per record.
#include "int4_common.hpp"

namespace lf {
namespace {

constexpr int kWaves = 4, kTile = 16, MT = kManyRows / (kWaves * kTile);  // row tiles of a wave

__device__ __forceinline__ f32x4 mfma(f16x8 a, f16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ uint32_t lower_pair(uint32_t a, uint32_t b) { return __builtin_amdgcn_perm(b, a, 0x05040100u); }
__device__ __forceinline__ uint32_t upper_pair(uint32_t a, uint32_t b) { return __builtin_amdgcn_perm(b, a, 0x07060302u); }

// A word's eight codes times s[i] plus m[i], element pairs (nibble i, nibble i + 4).  The fp16 bits of a Key word's,
// 0x5800 | code << 3, are 128 + code; of a Value word's, 0x4C00 | code << 6, 16 + code.
template <uint32_t Mask>
__device__ __forceinline__ u32x4 dequant8(uint32_t w, const uint32_t (&s)[4], const uint32_t (&m)[4], uint32_t base) {
    constexpr _Float16 bias = static_cast<_Float16>(Mask == kKeyMask ? 128 : 16);
    const u32x4 bits = codes8<Mask>(w, base);
    u32x4 r;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t pair = bits[i];
        const f16x2 code = __builtin_bit_cast(f16x2, pair) - f16x2{bias, bias};
        r[i] = __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(code, __builtin_bit_cast(f16x2, s[i]), __builtin_bit_cast(f16x2, m[i])));
    }
    return r;
}

template <int D, int GROUP>
__global__ __launch_bounds__(kWaves * kWave, 3) void int4_prefix_kernel(Int4Attention a) {
    using R = Int4Rec<D, GROUP>;
    constexpr int G = R::G, CH = R::chunks, VT = D / 16;
    constexpr int kK = 2 * CH * kWave, kV = VT * kWave;  // 16-byte pieces of a record's Keys and Values
    __shared__ u32x4 lds[2][kK + kV];
    const int h = blockIdx.x % a.L.n_kv, tile = blockIdx.x / a.L.n_kv, b = blockIdx.y, part = blockIdx.z;
    const int lane = threadIdx.x % kWave, wave = in_sgpr(static_cast<int>(threadIdx.x / kWave));
    const int col = lane & 15, quad = lane >> 4;
    const int len = int4_len(a.L, b);
    const int n = a.q_lens ? min(max(a.q_lens[b], 0), a.q_len) : a.q_len;
    const int records = prefix_records(a, len, n, tile);
    const int per = (records + a.prefix - 1) / a.prefix, first = min(part * per, records), last = min(first + per, records);

    // This wave's share of a record: 0, 1: sixteen Key rows; 2, 3: half of a lane's Value words.
    const uint8_t* base = int4_block(a.L, b, h, 0, R::bytes);
    constexpr int VW = VT / 2;                          // a lane's Value words
    constexpr int VG = GROUP == 32 ? VW / 2 : 1;        // and the groups they lie in
    const uint32_t code_base = in_vgpr(wave < 2 ? kKeyBaseHalf : kValueBase);  // (a wave stages Keys or Values)
    // Every wave loads the same pieces, whichever it stages: with a branch around the loads, what it joins waited for them.
    struct Raw {
        uint32_t w[4];
        uint32_t key[G];        // scale and minimum of a Key row's groups
        u32x4 value[2 * VG];    // of tokens 4 quad .. and 16 + 4 quad .. of a Value word's groups
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
        for (int g = 0; g < G; ++g) r.key[g] = *reinterpret_cast<const uint32_t*>(rec + key_at + 4 * kBlock * g);
#pragma unroll
        for (int k = 0; k < 2 * VG; ++k)
            r.value[k] = *reinterpret_cast<const u32x4*>(rec + value_at + 4 * kBlock * (k >> 1) + 64 * (k & 1));
    };
    const auto stage = [&](const Raw& r, u32x4* to) {
        if (wave < 2) {
#pragma unroll
            for (int c = 0; c < CH; ++c) {
                const uint32_t pair = r.key[c / (CH / G)], s = lower_pair(pair, pair), m = upper_pair(pair, pair);
                const uint32_t ss[4] = {s, s, s, s}, mm[4] = {m, m, m, m};
                to[(half * CH + c) * kWave + lane] = dequant8<kKeyMask>(r.w[c], ss, mm, code_base);
            }
        } else {
#pragma unroll
            for (int k = 0; k < VG; ++k) {
                uint32_t s[4], m[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    s[i] = lower_pair(r.value[2 * k][i], r.value[2 * k + 1][i]);
                    m[i] = upper_pair(r.value[2 * k][i], r.value[2 * k + 1][i]);
                }
#pragma unroll
                for (int c = k * (VW / VG); c < (k + 1) * (VW / VG); ++c)
                    to[kK + (half * VW + c) * kWave + lane] = dequant8<kValueMask>(r.w[c], s, m, code_base);
            }
        }
    };

    // rows (head of the group, token), tokens fastest: this lane's, one of each row tile
    f16x8 q[MT][CH];
    float scale[MT], ref[MT], limit[MT];  // limit: how far a score may pass ref; -inf until one is seen
    int row[MT];  // head of the group * q_len + token, or -1
    const bool flip = a.qscale < 0.f;
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        const int r = tile * kManyRows + (wave * MT + t) * kTile + col, i = r / a.q_len, j = r % a.q_len;
        row[t] = i < a.g ? r : -1;
        float x[CH][8] = {}, most = 0.f;
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            if (row[t] >= 0) query8<LF_BF16>(a, b * a.qb + static_cast<int64_t>(h * a.g + i) * a.qh + j * a.qt + 32 * c + 8 * quad, x[c]);
#pragma unroll
            for (int e = 0; e < 8; ++e) most = fmaxf(most, fabsf(x[c][e]));
        }
        most = rows_max(most);
        // 2^-exponent of the largest element (an all-zero or subnormal row: 2^126)
        const int exponent = static_cast<int>(__float_as_uint(most) >> 23);
        const float down = __uint_as_float(static_cast<uint32_t>(min(max(254 - exponent, 1), 253)) << 23);
        scale[t] = fmaxf(fabsf(a.qscale) / down, 1e-37f);
#pragma unroll
        for (int c = 0; c < CH; ++c)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                // operand element 2 i is channel i of the word, element 2 i + 1 channel 4 + i
                const float v = x[c][(e >> 1) + 4 * (e & 1)] * down;
                q[t][c][e] = static_cast<_Float16>(flip ? -v : v);
            }
        ref[t] = 0.f;
        limit[t] = -__builtin_inff();
    }
    f32x4 o[MT][VT], l[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        l[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int v = 0; v < VT; ++v) o[t][v] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    const f16x8 ones = {1, 1, 1, 1, 1, 1, 1, 1};

    Raw raw;
    if (first < last) {
        load(first, raw);
        stage(raw, lds[0]);
        load(min(first + 1, last - 1), raw);
    }
    __syncthreads();
    for (int k = first; k < last; ++k) {
        const u32x4* rec = lds[(k - first) & 1];
        if (k + 1 < last) {
            stage(raw, lds[(k + 1 - first) & 1]);
            load(min(k + 2, last - 1), raw);
        }
        f32x4 y[MT][2];
#pragma unroll
        for (int t = 0; t < MT; ++t) y[t][0] = y[t][1] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < CH; ++c)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const f16x8 key = __builtin_bit_cast(f16x8, rec[(u * CH + c) * kWave + lane]);
#pragma unroll
                for (int t = 0; t < MT; ++t) y[t][u] = mfma(key, q[t][c], y[t][u]);
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
                const float by = moves ? most : 0.f;
                const float down = limit[t] < 0.f && moves ? 0.f : __builtin_amdgcn_exp2f(-by);
                ref[t] += by;
                limit[t] = moves ? 8.f : limit[t];
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
                for (int u = 0; u < 2; ++u) p[t][2 * i + u] = static_cast<_Float16>(__builtin_amdgcn_exp2f(z[u][i]));
            l[t] = mfma(ones, p[t], l[t]);
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
        if (row[t] < 0) continue;
        const int64_t at = ((static_cast<int64_t>(b) * a.n_q + h * a.g) * a.q_len + row[t]) * a.parts + part;
        // (a sum of NaN counts as seen; rows behind the sequence's last token are zeros whatever they saw)
        const bool token = row[t] % a.q_len < n;
        if (quad == 0) {
            a.part_ml[2 * at] = token && l[t][0] != 0.f ? ref[t] : -__builtin_inff();
            a.part_ml[2 * at + 1] = token ? l[t][0] : 0.f;
        }
        if (!token)
#pragma unroll
            for (int v = 0; v < VT; ++v) o[t][v] = f32x4{0.f, 0.f, 0.f, 0.f};
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
