// Rows of the 4-bit cache: quantised as they are written, and read back.
//
// Per row and group of channels: lo = min x, hi = max x, s = clamp((hi - lo) / 15, 1e-5, 1e5),
// code = clamp(rint((x - lo) / s), 0, 15), every step IEEE float32; read back, code * fp16(s) + fp16(lo)
// with one rounding (the product of an 11- and a 4-bit number is exact).
//
// A wave owns a record of 32 tokens: D / 8 lanes take a row, eight channels each, which is one Key code word;
// the groups' minima and maxima are exchanged within GROUP / 8 lanes.  A Value word holds eight tokens of one
// channel (the attention's operand), so Value codes turn around through LDS and, where the write covers only
// some of a record's tokens, join the nibbles that are there: no other wave touches the record.  The sequences'
// lengths are read and advanced on the device.
#include "int4_common.hpp"

namespace lf {
namespace {

struct RowsArgs {
    lf_int4_layer L;
    const void* src[2];
    int64_t sb[2], sh[2], st[2];
    const int32_t* counts;
    int tokens;
    int vec;  // every source row starts on 16 bytes
};

// Eight consecutive elements of a row as float32.
template <int Dt>
__device__ __forceinline__ void load8(const void* p, int64_t at, int vec, float (&x)[8]) {
    if (vec) {
        if constexpr (Dt == LF_FP32) {
            const f32x4* q = reinterpret_cast<const f32x4*>(static_cast<const float*>(p) + at);
            const f32x4 a = q[0], b = q[1];
#pragma unroll
            for (int e = 0; e < 4; ++e) { x[e] = a[e]; x[4 + e] = b[e]; }
        } else {
            const u32x4 a = *reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(p) + at);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const uint16_t u = static_cast<uint16_t>(a[e >> 1] >> (16 * (e & 1)));
                x[e] = Dt == LF_BF16 ? bf16_to_f32(u) : f16_to_f32(u);
            }
        }
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = load_as_f32(p, at + e, Dt);
    }
}

// Codes of a lane's eight channels; scale and minimum of their group in every lane.
template <int GROUP>
__device__ __forceinline__ void quantise8(const float (&x)[8], uint32_t (&code)[8], float& s, float& lo) {
    lo = x[0];
    float hi = x[0];
#pragma unroll
    for (int e = 1; e < 8; ++e) { lo = fminf(lo, x[e]); hi = fmaxf(hi, x[e]); }
#pragma unroll
    for (int m = 1; m < GROUP / 8; m <<= 1) {
        lo = fminf(lo, __shfl_xor(lo, m, kWave));
        hi = fmaxf(hi, __shfl_xor(hi, m, kWave));
    }
    s = fminf(fmaxf((hi - lo) / 15.f, 1e-5f), 1e5f);
#pragma unroll
    for (int e = 0; e < 8; ++e) code[e] = static_cast<uint32_t>(fminf(fmaxf(rintf((x[e] - lo) / s), 0.f), 15.f));
}

// Tokens t0 .. t1 - 1 of a record, from source rows src0 .. of (b, h); one wave.  ``codes``: its 32 x D bytes of LDS.
template <int D, int GROUP, int Dt>
__device__ void write_block(const RowsArgs& a, uint8_t* rec, int b, int h, int src0, int t0, int t1, uint8_t* codes) {
    using R = Int4Rec<D, GROUP>;
    constexpr int LR = D / 8, RP = kWave / LR;  // lanes per row, rows per pass
    const int lane = threadIdx.x & (kWave - 1), w = lane % LR;
    uint32_t* words = reinterpret_cast<uint32_t*>(rec);
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
        const int64_t base = b * a.sb[kv] + h * a.sh[kv] + 8 * w;
        uint32_t* sm = reinterpret_cast<uint32_t*>(rec + (kv ? R::vsm : R::ksm));
        for (int r0 = t0; r0 < t1; r0 += RP) {
            const int row = r0 + lane / LR;
            const int from = src0 + min(row, t1 - 1) - t0;
            float x[8], s, lo;
            load8<Dt>(a.src[kv], base + from * a.st[kv], a.vec, x);
            uint32_t code[8];
            quantise8<GROUP>(x, code, s, lo);
            if (row >= t1) continue;
            if (w % (GROUP / 8) == 0)
                sm[w / (GROUP / 8) * kBlock + row] = f32_to_f16(s) | static_cast<uint32_t>(f32_to_f16(lo)) << 16;
            if (kv == 0) {
                uint32_t word = 0;
#pragma unroll
                for (int e = 0; e < 8; ++e) word |= nibble_bits(code[e], e);
                words[row * LR + key_word(D, w)] = word;
            } else {
                u32x2 packed = {0, 0};
#pragma unroll
                for (int e = 0; e < 8; ++e) packed[e >> 2] |= code[e] << (8 * (e & 3));
                *reinterpret_cast<u32x2*>(codes + row * D + 8 * w) = packed;
            }
        }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    const bool whole = t0 == 0 && t1 == kBlock;
    const int quad = lane >> 4, c0 = lane & 15;
    uint32_t fresh = 0;  // the nibbles this write replaces
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const int tok = 4 * quad + (e & 3) + 16 * (e >> 2);
        if (tok >= t0 && tok < t1) fresh |= nibble_bits(15u, e);
    }
    u32x4* vw = reinterpret_cast<u32x4*>(rec + R::v) + lane;
#pragma unroll
    for (int u = 0; u < D / 64; ++u) {
        u32x4 word = {0, 0, 0, 0};
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int e = 0; e < 8; ++e)
                word[t] |= nibble_bits(codes[(4 * quad + (e & 3) + 16 * (e >> 2)) * D + 64 * u + 16 * t + c0] & 15u, e);
        if (whole) vw[u * kWave] = word;
        else if (fresh) vw[u * kWave] = (vw[u * kWave] & ~fresh) | (word & fresh);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// float32 rounded outward to bf16 (the pair's lower bound down, its upper bound up).
__device__ __forceinline__ uint16_t bf16_up(float x) {
    const uint32_t u = __float_as_uint(x);
    return static_cast<uint16_t>((u >> 31 ? u : u + 0xffffu) >> 16);
}
__device__ __forceinline__ uint16_t bf16_down(float x) { return static_cast<uint16_t>(bf16_up(-x) ^ 0x8000u); }

// Per-channel bounds of full page ``page``'s Keys, from the records: ``n`` threads (whole waves) of index tid.
// One wave alone (n == 64), or all of a workgroup's with ``red`` [n / 64][2][D] and barriers.
template <int D, int GROUP>
__device__ void page_bounds(const lf_int4_layer& L, int b, int h, int page, int tid, int n, float* red) {
    using R = Int4Rec<D, GROUP>;
    constexpr int LR = D / 8;
    const int P = L.page_size, w = tid % LR, wave = tid / kWave, lane = tid % kWave;
    const uint8_t* rec0 = int4_block(L, b, h, page * (P / kBlock), R::bytes);
    float lo[8], hi[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) { lo[e] = __builtin_inff(); hi[e] = -__builtin_inff(); }
    for (int t = tid / LR; t < P; t += n / LR) {
        const uint8_t* rec = rec0 + (t / kBlock) * R::bytes;
        const int row = t % kBlock;
        const uint32_t word = reinterpret_cast<const uint32_t*>(rec)[row * LR + key_word(D, w)];
        const uint32_t sm = reinterpret_cast<const uint32_t*>(rec + R::ksm)[w / (GROUP / 8) * kBlock + row];
        const float s = pair_scale(sm), m = pair_min(sm);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float x = fmaf(static_cast<float>(code_at(word, e)), s, m);
            lo[e] = fminf(lo[e], x);
            hi[e] = fmaxf(hi[e], x);
        }
    }
#pragma unroll
    for (int m = LR; m < kWave; m <<= 1)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            lo[e] = fminf(lo[e], __shfl_xor(lo[e], m, kWave));
            hi[e] = fmaxf(hi[e], __shfl_xor(hi[e], m, kWave));
        }
    uint16_t* out = L.bounds + ((static_cast<int64_t>(b) * L.n_kv + h) * (L.cap_tokens / P) + page) * 2 * D;
    if (n == kWave) {
        if (lane < LR)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                out[8 * w + e] = bf16_down(lo[e]);
                out[D + 8 * w + e] = bf16_up(hi[e]);
            }
        return;
    }
    if (lane < LR)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            red[wave * 2 * D + 8 * w + e] = lo[e];
            red[wave * 2 * D + D + 8 * w + e] = hi[e];
        }
    __syncthreads();
    for (int c = tid; c < 2 * D; c += n) {
        float x = red[c];
        for (int k = 1; k < n / kWave; ++k) x = c < D ? fminf(x, red[k * 2 * D + c]) : fmaxf(x, red[k * 2 * D + c]);
        out[c] = c < D ? bf16_down(x) : bf16_up(x);
    }
}

__device__ __forceinline__ int append_count(const RowsArgs& a, int b) {
    return a.counts ? min(max(a.counts[b], 0), a.tokens) : a.tokens;
}

// Many tokens: a workgroup per (page, kv head, sequence), a wave per record.
template <int D, int GROUP, int Dt>
__global__ __launch_bounds__(256) void int4_append_pages_kernel(RowsArgs a) {
    __shared__ __attribute__((aligned(16))) uint8_t lds[4 * kBlock * D];
    const int b = blockIdx.z, h = blockIdx.y, P = a.L.page_size;
    const int start = int4_len(a.L, b);
    const int end = static_cast<int>(min(static_cast<int64_t>(start) + append_count(a, b), static_cast<int64_t>(a.L.cap_tokens)));
    const int page = start / P + blockIdx.x;
    if (static_cast<int64_t>(page) * P >= end) return;
    const int p0 = page * P, lo = max(start, p0), hi = min(end, p0 + P);
    const int wave = threadIdx.x / kWave;
    for (int k = wave; k < P / kBlock; k += blockDim.x / kWave) {
        const int k0 = p0 + k * kBlock;
        const int t0 = max(lo - k0, 0), t1 = min(hi - k0, kBlock);
        if (t0 < t1)
            write_block<D, GROUP, Dt>(a, int4_block(a.L, b, h, k0 / kBlock, Int4Rec<D, GROUP>::bytes), b, h,
                                      k0 + t0 - start, t0, t1, lds + wave * kBlock * D);
    }
    if (hi < p0 + P) return;
    __threadfence_block();
    __syncthreads();
    page_bounds<D, GROUP>(a.L, b, h, page, threadIdx.x, blockDim.x, reinterpret_cast<float*>(lds));
}

__global__ void int4_advance_kernel(RowsArgs a) {
    const int b = blockIdx.x * blockDim.x + threadIdx.x;
    if (b < a.L.batch)
        a.L.lens[b] = static_cast<int>(min(static_cast<int64_t>(int4_len(a.L, b)) + append_count(a, b), static_cast<int64_t>(a.L.cap_tokens)));
}

// A few tokens (at most a record's): a workgroup per sequence, a wave per kv head; the workgroup advances the length.
constexpr int kFewTokens = 8;
template <int D, int GROUP, int Dt>
__global__ __launch_bounds__(512) void int4_append_few_kernel(RowsArgs a) {
    constexpr int kWaves = D > 128 ? 4 : 8;
    __shared__ __attribute__((aligned(16))) uint8_t lds[kWaves * kBlock * D];
    const int b = blockIdx.x, P = a.L.page_size, wave = threadIdx.x / kWave;
    const int start = int4_len(a.L, b);
    const int end = static_cast<int>(min(static_cast<int64_t>(start) + append_count(a, b), static_cast<int64_t>(a.L.cap_tokens)));
    for (int h = wave; h < a.L.n_kv && start < end; h += blockDim.x / kWave) {
        for (int k = start / kBlock; k * kBlock < end; ++k) {
            const int t0 = max(start - k * kBlock, 0), t1 = min(end - k * kBlock, kBlock);
            write_block<D, GROUP, Dt>(a, int4_block(a.L, b, h, k, Int4Rec<D, GROUP>::bytes), b, h, k * kBlock + t0 - start,
                                      t0, t1, lds + wave * kBlock * D);
        }
        for (int page = start / P; page < end / P; ++page) {
            __threadfence_block();
            page_bounds<D, GROUP>(a.L, b, h, page, threadIdx.x % kWave, kWave, nullptr);
        }
    }
    __syncthreads();  // every wave has read the length
    if (threadIdx.x == 0) a.L.lens[b] = end;
}

struct ReadArgs {
    lf_int4_layer L;
    const int32_t* starts;
    int tokens;
    void* out[2];
    int dtype;
};

// A thread per (token, eight channels): one Key word, and one nibble of eight Value words.
template <int D, int GROUP>
__global__ __launch_bounds__(256) void int4_read_kernel(ReadArgs a) {
    using R = Int4Rec<D, GROUP>;
    constexpr int LR = D / 8;
    const int b = blockIdx.z, h = blockIdx.y;
    const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    const int t = static_cast<int>(i / LR), w = static_cast<int>(i % LR);
    if (t >= a.tokens) return;
    const int64_t pos = static_cast<int64_t>(a.starts ? a.starts[b] : 0) + t;
    const bool there = pos >= 0 && pos < int4_len(a.L, b);
    const int64_t dst = ((static_cast<int64_t>(b) * a.L.n_kv + h) * a.tokens + t) * D + 8 * w;
    const uint8_t* rec = int4_block(a.L, b, h, there ? static_cast<int>(pos / kBlock) : 0, R::bytes);
    const int row = there ? static_cast<int>(pos % kBlock) : 0, g = w / (GROUP / 8);
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
        if (!a.out[kv]) continue;
        uint32_t code[8] = {};
        float s = 0.f, m = 0.f;
        if (there) {
            const uint32_t sm = reinterpret_cast<const uint32_t*>(rec + (kv ? R::vsm : R::ksm))[g * kBlock + row];
            s = pair_scale(sm);
            m = pair_min(sm);
            if (kv == 0) {
                const uint32_t word = reinterpret_cast<const uint32_t*>(rec)[row * LR + key_word(D, w)];
#pragma unroll
                for (int e = 0; e < 8; ++e) code[e] = code_at(word, e);
            } else {
                const uint32_t* v = reinterpret_cast<const uint32_t*>(rec + R::v);
                const int e = value_nibble(row);
#pragma unroll
                for (int c = 0; c < 8; ++c) code[c] = turn(v[value_word(row, 8 * w + c)], (4 * e + 3) & 31) & 15u;
            }
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) store_from_f32(a.out[kv], dst + e, a.dtype, fmaf(static_cast<float>(code[e]), s, m));
    }
}

template <int D, int GROUP, int Dt>
int append_typed(const RowsArgs& a, hipStream_t stream) {
    const lf_int4_layer& L = a.L;
    if (a.tokens <= kFewTokens) {
        const int waves = min(L.n_kv, D > 128 ? 4 : 8);
        hipLaunchKernelGGL((int4_append_few_kernel<D, GROUP, Dt>), dim3(L.batch), dim3(waves * kWave), 0, stream, a);
    } else {
        const int P = L.page_size, waves = min(4, P / kBlock);
        const int64_t pages = (static_cast<int64_t>(a.tokens) + 2 * P - 2) / P;  // that a run of tokens can touch
        const int64_t here = min(pages, static_cast<int64_t>(L.cap_tokens / P) + 1);
        hipLaunchKernelGGL((int4_append_pages_kernel<D, GROUP, Dt>), dim3(static_cast<uint32_t>(here), L.n_kv, L.batch),
                           dim3(waves * kWave), 0, stream, a);
        hipLaunchKernelGGL(int4_advance_kernel, dim3((L.batch + 255) / 256), dim3(256), 0, stream, a);
    }
    const hipError_t err = hipGetLastError();
    return err == hipSuccess ? LF_OK : static_cast<int>(err);
}

}  // namespace

int launch_int4_append(const lf_int4_layer& L, const void* k_src, const void* v_src, int dtype, const int64_t* k_strides,
                       const int64_t* v_strides, const int32_t* counts, int tokens, hipStream_t stream) {
    RowsArgs a{};
    a.L = L;
    a.src[0] = k_src; a.src[1] = v_src;
    a.counts = counts;
    a.tokens = tokens;
    const int esize = dtype == LF_FP32 ? 4 : 2;
    bool vec = true;
    for (int kv = 0; kv < 2; ++kv) {
        const int64_t* s = kv ? v_strides : k_strides;
        a.sb[kv] = s[0]; a.sh[kv] = s[1]; a.st[kv] = s[2];
        vec = vec && reinterpret_cast<uintptr_t>(a.src[kv]) % 16 == 0;
        for (int i = 0; i < 3; ++i) vec = vec && s[i] * esize % 16 == 0;
    }
    a.vec = vec;
    return int4_dispatch(L, [&](auto shape) {
        constexpr int D = decltype(shape)::d, GROUP = decltype(shape)::group;
        return dtype == LF_BF16 ? append_typed<D, GROUP, LF_BF16>(a, stream)
               : dtype == LF_FP16 ? append_typed<D, GROUP, LF_FP16>(a, stream) : append_typed<D, GROUP, LF_FP32>(a, stream);
    });
}

int launch_int4_read(const lf_int4_layer& L, const int32_t* starts, int tokens, void* k_out, void* v_out, int dtype,
                     hipStream_t stream) {
    ReadArgs a{L, starts, tokens, {k_out, v_out}, dtype};
    return int4_dispatch(L, [&](auto shape) {
        constexpr int D = decltype(shape)::d, GROUP = decltype(shape)::group;
        const int64_t threads = static_cast<int64_t>(tokens) * (D / 8);
        hipLaunchKernelGGL((int4_read_kernel<D, GROUP>), dim3(static_cast<uint32_t>((threads + 255) / 256), L.n_kv, L.batch),
                           dim3(256), 0, stream, a);
        const hipError_t err = hipGetLastError();
        return err == hipSuccess ? LF_OK : static_cast<int>(err);
    });
}

}  // namespace lf
