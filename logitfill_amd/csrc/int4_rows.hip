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
    int tokens;
    int vec;       // every source row starts on 16 bytes
    int b0;        // the launch's first sequence
    int counted;   // 1: counts holds the tokens of sequences b0 ..
    int started;   // 1: starts holds their lengths
    int32_t counts[kInlineSeqs], starts[kInlineSeqs];
};

// Eight consecutive elements of a row, as they are and as float32.
template <int Dt>
struct Raw8 {
    u32x4 w[Dt == LF_FP32 ? 2 : 1];
};
template <int Dt>
__device__ __forceinline__ Raw8<Dt> load8(const void* p, int64_t at, int vec) {
    Raw8<Dt> r;
    if constexpr (Dt == LF_FP32) {
        const uint32_t* q = static_cast<const uint32_t*>(p) + at;
        if (vec) {
            r.w[0] = *reinterpret_cast<const u32x4*>(q);
            r.w[1] = *reinterpret_cast<const u32x4*>(q + 4);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) r.w[e >> 2][e & 3] = q[e];
        }
    } else {
        const uint16_t* q = static_cast<const uint16_t*>(p) + at;
        if (vec) {
            r.w[0] = *reinterpret_cast<const u32x4*>(q);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) r.w[0][e] = q[2 * e] | static_cast<uint32_t>(q[2 * e + 1]) << 16;
        }
    }
    return r;
}
template <int Dt>
__device__ __forceinline__ void widen8(const Raw8<Dt>& r, float (&x)[8]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        if constexpr (Dt == LF_FP32) x[e] = __uint_as_float(r.w[e >> 2][e & 3]);
        else if constexpr (Dt == LF_BF16) x[e] = __uint_as_float(e & 1 ? r.w[0][e >> 1] & 0xffff0000u : r.w[0][e >> 1] << 16);
        else x[e] = f16_to_f32(static_cast<uint16_t>(r.w[0][e >> 1] >> (16 * (e & 1))));
    }
}

// The smallest x of 4, 8 or 16 neighbouring lanes, in every one of them: exchanges within a row of 16 lanes that ride on
// the comparison (lanes i and i ^ 1, i ^ 2, then 7 - i and 15 - i, whose fours and eights hold one value by then).
template <int Ctrl>
__device__ __forceinline__ float row_other(float x) {
    const int i = __builtin_bit_cast(int, x);
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(i, i, Ctrl, 0xf, 0xf, true));
}
template <int N>
__device__ __forceinline__ float lanes_min(float x) {
    x = fminf(x, row_other<0xB1>(x));                       // quad_perm 1, 0, 3, 2
    x = fminf(x, row_other<0x4E>(x));                       // quad_perm 2, 3, 0, 1
    if constexpr (N > 4) x = fminf(x, row_other<0x141>(x)); // row_half_mirror
    if constexpr (N > 8) x = fminf(x, row_other<0x140>(x)); // row_mirror
    return x;
}

// a / b, rounded to nearest, from y = RN(1 / b) and one correction by the exact residual (Markstein): the correctly
// rounded quotient, as the division gives it, where no step overflows.
__device__ __forceinline__ float quotient(float a, float b, float y) {
    const float q = a * y;
    return fmaf(fmaf(-q, b, a), y, q);
}

// Codes of a lane's eight channels, each with kCodeCarry; scale and minimum of their group in every lane.  The codes of
// a group share the reciprocal of the scale.  A range beyond float32's is cut to its largest number, whose quotient
// clamps to 15 as the infinite one does.  Adding 2^23 rounds to an integer, half to even, in the lower bits.
constexpr uint32_t kCodeCarry = 0x4B000000u;
template <int GROUP, int Dt>
__device__ __forceinline__ void quantise8(const float (&x)[8], uint32_t (&code)[8], float& s, float& lo) {
    lo = x[0];
    float hi = x[0];
#pragma unroll
    for (int e = 1; e < 8; ++e) { lo = fminf(lo, x[e]); hi = fmaxf(hi, x[e]); }
    lo = lanes_min<GROUP / 8>(lo);
    hi = -lanes_min<GROUP / 8>(-hi);
    constexpr float kMost = 3.40282347e38f;
    s = __builtin_amdgcn_fmed3f(quotient(fminf(hi - lo, kMost), 15.f, 1.f / 15.f), 1e-5f, 1e5f);
    const float y = 1.f / s;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const float d = Dt == LF_FP16 ? x[e] - lo : fminf(x[e] - lo, kMost);
        code[e] = __float_as_uint(__builtin_amdgcn_fmed3f(quotient(d, s, y), 0.f, 15.f) + 8388608.f);
    }
}
// The sum of kCodeCarry << (step e), e = 0 .. n - 1: what a word of n codes added up in their places carries too much.
constexpr uint32_t carried(int n, int step) {
    uint32_t c = 0;
    for (int e = 0; e < n; ++e) c += kCodeCarry << (step * e);
    return c;
}

// Four Value words from eight tokens' codes of four channels, a byte each: word c's nibble e is byte c of tok[e].
__device__ __forceinline__ u32x4 value_words(const uint32_t (&tok)[8]) {
    uint32_t x[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) x[k] = tok[2 * k] | tok[2 * k + 1] << 4;
    const uint32_t a = __builtin_amdgcn_perm(x[1], x[0], 0x05010400u), b = __builtin_amdgcn_perm(x[3], x[2], 0x05010400u);
    const uint32_t c = __builtin_amdgcn_perm(x[1], x[0], 0x07030602u), d = __builtin_amdgcn_perm(x[3], x[2], 0x07030602u);
    const u32x4 w = {__builtin_amdgcn_perm(b, a, 0x05040100u), __builtin_amdgcn_perm(b, a, 0x07060302u),
                     __builtin_amdgcn_perm(d, c, 0x05040100u), __builtin_amdgcn_perm(d, c, 0x07060302u)};
    constexpr int left = 32 - kValueTurn;
    return u32x4{turn(w[0], left), turn(w[1], left), turn(w[2], left), turn(w[3], left)};
}

// Tokens t0 .. t1 - 1 of a record, from source rows src0 .. of (b, h); one wave.  ``codes``: its 32 x D bytes of LDS;
// ``most``: the record's largest Value scale.  Whole: all 32, of rows that start on 16 bytes, every row's load on its way
// before the first is used (a branch around each load, for rows that do not, made each wait for the one before).
// Four prompts of up to 16 300 tokens, 4 heads of 128, groups of 64: 47 us for 117 MB of rows and 33 MB of codes (3.2
// TB/s); the VALU is 63 % busy with the quantisation (a reciprocal per group, a corrected quotient per element).
template <int D, int GROUP, int Dt, bool Whole>
__device__ __forceinline__ void write_block(const RowsArgs& a, uint8_t* rec, int b, int h, int src0, int t0, int t1, uint8_t* codes, uint16_t* most) {
    using R = Int4Rec<D, GROUP>;
    constexpr int LR = D / 8, RP = kWave / LR, Passes = kBlock / RP;  // lanes per row, rows per pass
    const int lane = threadIdx.x & (kWave - 1), w = lane % LR;
    uint32_t* words = reinterpret_cast<uint32_t*>(rec);
    const int quad = lane >> 4, c0 = lane & 15;
    u32x4* vw = reinterpret_cast<u32x4*>(rec + R::v) + lane;
    u32x4 old[Whole ? 1 : D / 64];  // the Value words that a part of the record's tokens joins
    if constexpr (!Whole)
#pragma unroll
        for (int u = 0; u < D / 64; ++u) old[u] = vw[u * kWave];
    const auto load = [&](int kv, int row) {
        return load8<Dt>(a.src[kv], b * a.sb[kv] + h * a.sh[kv] + 8 * w + (src0 + static_cast<int64_t>(row) - t0) * a.st[kv], Whole || a.vec);
    };
    uint32_t top = Whole || t0 == 0 ? 0 : *most;  // (fp16 numbers above zero are ordered as their bits)
    const auto take = [&](int kv, int row, const Raw8<Dt>& raw, bool real) {
        float x[8], s, lo;
        widen8<Dt>(raw, x);
        uint32_t code[8];
        quantise8<GROUP, Dt>(x, code, s, lo);
        if (!real) return;
        uint32_t* sm = reinterpret_cast<uint32_t*>(rec + (kv ? R::vsm : R::ksm));
        if (w % (GROUP / 8) == 0)
            sm[w / (GROUP / 8) * kBlock + row] = f32_to_f16(s) | static_cast<uint32_t>(f32_to_f16(lo)) << 16;
        if (kv) top = max(top, static_cast<uint32_t>(f32_to_f16(s)));
        if (kv == 0) {
            uint32_t word = -carried(8, 4);
#pragma unroll
            for (int e = 0; e < 8; ++e) word += code[e] << (4 * e);
            words[row * LR + key_word(D, w)] = turn(word, 32 - kKeyTurn);
        } else {
            u32x2 packed = {-carried(4, 8), -carried(4, 8)};
#pragma unroll
            for (int e = 0; e < 8; ++e) packed[e >> 2] += code[e] << (8 * (e & 3));
            *reinterpret_cast<u32x2*>(codes + row * D + 8 * w) = packed;
        }
    };
    if constexpr (Whole && Dt != LF_FP32 && Passes <= 8) {
        Raw8<Dt> raw[2][Passes];
#pragma unroll
        for (int kv = 0; kv < 2; ++kv)
#pragma unroll
            for (int p = 0; p < Passes; ++p) raw[kv][p] = load(kv, p * RP + lane / LR);
#pragma unroll
        for (int kv = 0; kv < 2; ++kv)
#pragma unroll
            for (int p = 0; p < Passes; ++p) take(kv, p * RP + lane / LR, raw[kv][p], true);
    } else if constexpr (Whole) {
        constexpr int Ahead = Dt == LF_FP32 || Passes > 8 ? 4 : 8;  // rows on their way
#pragma unroll
        for (int kv = 0; kv < 2; ++kv)
#pragma unroll
            for (int p0 = 0; p0 < Passes; p0 += Ahead) {
                Raw8<Dt> raw[Ahead];
#pragma unroll
                for (int p = 0; p < Ahead && p0 + p < Passes; ++p) raw[p] = load(kv, (p0 + p) * RP + lane / LR);
#pragma unroll
                for (int p = 0; p < Ahead && p0 + p < Passes; ++p) take(kv, (p0 + p) * RP + lane / LR, raw[p], true);
            }
    } else {
        for (int r0 = t0; r0 < t1; r0 += RP) {
            const int row = r0 + lane / LR, from = min(row, t1 - 1);
            const Raw8<Dt> k = load(0, from), v = load(1, from);
            take(0, row, k, row < t1);
            take(1, row, v, row < t1);
        }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    top = min(top, 0x7bffu);  // (an infinite scale counts as the largest)
#pragma unroll
    for (int m = 1; m < kWave; m <<= 1) top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), m, kWave)));
    if (lane == 0) *most = static_cast<uint16_t>(top);
    uint32_t fresh = 0;  // the nibbles this write replaces
    if constexpr (!Whole)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int tok = 4 * quad + (e & 3) + 16 * (e >> 2);
            if (tok >= t0 && tok < t1) fresh |= turn(15u << (4 * e), 32 - kValueTurn);
        }
#pragma unroll
    for (int u = 0; u < D / 64; ++u) {
        uint32_t tok[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            // (rows this write does not bring: whatever the LDS holds, and replaced below)
            const uint8_t* at = codes + (4 * quad + (e & 3) + 16 * (e >> 2)) * D + 64 * u;
            if constexpr (GROUP == 32) {
                tok[e] = *reinterpret_cast<const uint16_t*>(at + 2 * c0) | static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(at + 32 + 2 * c0)) << 16;
            } else {
                tok[e] = *reinterpret_cast<const uint32_t*>(at + 4 * c0);
            }
            if constexpr (!Whole) tok[e] &= 0x0f0f0f0fu;
        }
        const u32x4 word = value_words(tok);
        if constexpr (Whole) vw[u * kWave] = word;
        else if (fresh) vw[u * kWave] = (old[u] & ~fresh) | (word & fresh);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// float32 rounded outward to bf16 (the pair's lower bound down, its upper bound up), infinities to the largest number
// (a selection multiplies bounds by zeros).
__device__ __forceinline__ uint16_t bf16_up(float x) {
    const uint32_t u = __float_as_uint(__builtin_amdgcn_fmed3f(x, -3.3895314e38f, 3.3895314e38f));
    return static_cast<uint16_t>((u >> 31 ? u : u + 0xffffu) >> 16);
}
__device__ __forceinline__ uint16_t bf16_down(float x) { return static_cast<uint16_t>(bf16_up(-x) ^ 0x8000u); }

// Per-channel bounds of full page ``page``'s Keys, from the records, by the whole workgroup (``n`` threads, barriers);
// ``red`` [n / 64][2][D].
template <int D, int GROUP>
__device__ void page_bounds(const lf_int4_layer& L, int b, int h, int page, int tid, int n, float* red) {
    using R = Int4Rec<D, GROUP>;
    constexpr int LR = D / 8;
    const int P = L.page_size, w = tid % LR, wave = tid / kWave, lane = tid % kWave;
    const uint8_t* rec0 = int4_block(L, b, h, page * (P / kBlock), R::bytes);
    float lo[8], hi[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) { lo[e] = __builtin_inff(); hi[e] = -__builtin_inff(); }
#pragma unroll 4
    for (int t = tid / LR; t < P; t += n / LR) {
        const uint8_t* rec = rec0 + (t / kBlock) * R::bytes;
        const int row = t % kBlock;
        const uint32_t word = reinterpret_cast<const uint32_t*>(rec)[row * LR + key_word(D, w)];
        const uint32_t sm = reinterpret_cast<const uint32_t*>(rec + R::ksm)[w / (GROUP / 8) * kBlock + row];
        const float s = pair_scale(sm), m = pair_min(sm);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float x = fmaf(static_cast<float>(code_at<kKeyTurn>(word, e)), s, m);
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

__device__ __forceinline__ int append_count(const RowsArgs& a, int i) { return a.counted ? a.counts[i] : a.tokens; }
__device__ __forceinline__ int append_start(const RowsArgs& a, int i) { return a.started ? a.starts[i] : int4_len(a.L, a.b0 + i); }
__device__ __forceinline__ int append_end(const RowsArgs& a, int i, int start) {
    return static_cast<int>(min(static_cast<int64_t>(start) + append_count(a, i), static_cast<int64_t>(a.L.cap_tokens)));
}

// Many tokens: a workgroup per (page, kv head, sequence), a wave per record.
template <int D, int GROUP, int Dt>
__global__ __launch_bounds__(256) void int4_append_pages_kernel(RowsArgs a) {
    __shared__ __attribute__((aligned(16))) uint8_t lds[4 * kBlock * D];
    const int b = a.b0 + blockIdx.z, h = blockIdx.y, P = a.L.page_size;
    const int start = append_start(a, blockIdx.z), end = append_end(a, blockIdx.z, start);
    // (with the lengths in the arguments nobody reads lens)
    if (a.started && blockIdx.x == 0 && h == 0 && threadIdx.x == 0) a.L.lens[b] = end;
    const int page = start / P + blockIdx.x;
    if (static_cast<int64_t>(page) * P >= end) return;
    const int p0 = page * P, lo = max(start, p0), hi = min(end, p0 + P);
    const int wave = in_sgpr(static_cast<int>(threadIdx.x / kWave));
    for (int k = wave; k < P / kBlock; k += blockDim.x / kWave) {
        const int k0 = p0 + k * kBlock;
        const int t0 = max(lo - k0, 0), t1 = min(hi - k0, kBlock);
        if (t0 >= t1) continue;
        uint8_t* rec = int4_block(a.L, b, h, k0 / kBlock, Int4Rec<D, GROUP>::bytes);
        if (t1 - t0 == kBlock && a.vec) write_block<D, GROUP, Dt, true>(a, rec, b, h, k0 - start, 0, kBlock, lds + wave * kBlock * D, int4_top(a.L, b, h, k0 / kBlock));
        else write_block<D, GROUP, Dt, false>(a, rec, b, h, k0 + t0 - start, t0, t1, lds + wave * kBlock * D, int4_top(a.L, b, h, k0 / kBlock));
    }
    if (hi == p0 + P) {
        __threadfence_block();
        __syncthreads();
        page_bounds<D, GROUP>(a.L, b, h, page, threadIdx.x, blockDim.x, reinterpret_cast<float*>(lds));
    }
}

__global__ void int4_advance_kernel(RowsArgs a) {
    const int i = threadIdx.x, b = a.b0 + i;
    if (i < kInlineSeqs && b < a.L.batch) a.L.lens[b] = append_end(a, i, int4_len(a.L, b));
}

// A few tokens behind lengths that only the device knows: a workgroup per sequence, a wave per kv head; the workgroup
// advances the length, which with a workgroup per page and head takes a launch of its own.  Captured appends of 1, 4 and
// 8 tokens, 16 sequences of 4 heads of 128: 4.2, 4.5 and 5.5 us; 9 tokens, by pages, 6.6.  (A page that is completed gets
// its bounds head after head: not measured with more than 4.)  With the lengths in the
// arguments pages are the faster way for any count (one token to 8 sequences that fill a page 6.4 us against 8.1).
constexpr int kFewTokens = 8;
template <int D, int GROUP, int Dt>
__global__ __launch_bounds__(512) void int4_append_few_kernel(RowsArgs a) {
    constexpr int kWaves = D > 128 ? 4 : 8;
    __shared__ __attribute__((aligned(16))) uint8_t lds[kWaves * kBlock * D];
    const int b = a.b0 + blockIdx.x, P = a.L.page_size, wave = in_sgpr(static_cast<int>(threadIdx.x / kWave));
    const int start = append_start(a, blockIdx.x), end = append_end(a, blockIdx.x, start);
    for (int h = wave; h < a.L.n_kv && start < end; h += kWaves)
        for (int k = start / kBlock; k * kBlock < end; ++k) {
            const int t0 = max(start - k * kBlock, 0), t1 = min(end - k * kBlock, kBlock);
            write_block<D, GROUP, Dt, false>(a, int4_block(a.L, b, h, k, Int4Rec<D, GROUP>::bytes), b, h,
                                             k * kBlock + t0 - start, t0, t1, lds + wave * kBlock * D, int4_top(a.L, b, h, k));
        }
    __threadfence_block();
    __syncthreads();  // every wave has read the length, and its rows are there
    if (threadIdx.x == 0) a.L.lens[b] = end;
    for (int page = start / P; page < end / P; ++page)
        for (int h = 0; h < a.L.n_kv; ++h) {
            page_bounds<D, GROUP>(a.L, b, h, page, threadIdx.x, kWaves * kWave, reinterpret_cast<float*>(lds));
            __syncthreads();
        }
}

constexpr int kInlineLens = 512;  // 2 of a launch's 4 KB of arguments
struct LensArgs {
    int32_t* lens;
    int b0, n;
    int32_t value[kInlineLens];
};
__global__ void int4_set_lens_kernel(LensArgs a) {
    if (static_cast<int>(threadIdx.x) < a.n) a.lens[a.b0 + threadIdx.x] = a.value[threadIdx.x];
}

struct ReadArgs {
    lf_int4_layer L;
    int tokens;
    int b0;
    void* out[2];
    int32_t starts[kInlineSeqs];
};

// Rows from .. to - 1 of a record, zeros from row ``seen`` on: a Key word and row segment of eight channels per lane, and
// Values of four (two and two) channels and eight tokens.
template <int D, int GROUP, int Dt, bool Whole>
__device__ __forceinline__ void read_record(const ReadArgs& a, const uint8_t* rec, int64_t dst, int from, int to, int seen, int lane) {
    using R = Int4Rec<D, GROUP>;
    constexpr int LR = D / 8, RP = kWave / LR, Passes = kBlock / RP, U = D / 64;
    const int w = lane % LR, quad = lane >> 4, c0 = lane & 15;
    uint32_t word[Passes], key[Passes];
    u32x4 values[U], pairs[U][2][2];
#pragma unroll
    for (int p = 0; p < Passes; ++p) {
        if (!Whole && (p * RP + RP <= from || p * RP >= to)) continue;
        const int row = p * RP + lane / LR;
        word[p] = reinterpret_cast<const uint32_t*>(rec)[row * LR + key_word(D, w)];
        key[p] = reinterpret_cast<const uint32_t*>(rec + R::ksm)[w / (GROUP / 8) * kBlock + row];
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        values[u] = reinterpret_cast<const u32x4*>(rec + R::v)[u * kWave + lane];
#pragma unroll
        for (int v = 0; v < 2; ++v)
#pragma unroll
            for (int k = 0; k < 2; ++k)  // of the four channels, or of the lower and the upper two
                pairs[u][v][k] = reinterpret_cast<const u32x4*>(rec + R::vsm)[(GROUP == 32 ? 2 * u + k : 64 * u / GROUP) * (kBlock / 4) + 4 * v + quad];
    }
    if (a.out[0])
#pragma unroll
        for (int p = 0; p < Passes; ++p) {
            if (!Whole && (p * RP + RP <= from || p * RP >= to)) continue;
            const int row = p * RP + lane / LR;
            float x[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = Whole || row < seen ? fmaf(static_cast<float>(code_at<kKeyTurn>(word[p], e)), pair_scale(key[p]), pair_min(key[p])) : 0.f;
            if (Whole || (row >= from && row < to)) store_row<Dt>(a.out[0], dst + row * D + 8 * w, x);
        }
    if (a.out[1])
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int row = 16 * (e >> 2) + 4 * quad + (e & 3);
                if (!Whole && (row < from || row >= to)) continue;
                float x[4];
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    const uint32_t pair = pairs[u][e >> 2][t >> 1][e & 3];
                    x[t] = Whole || row < seen ? fmaf(static_cast<float>(code_at<kValueTurn>(values[u][t], e)), pair_scale(pair), pair_min(pair)) : 0.f;
                }
                if constexpr (GROUP == 32) {
                    const float a0[2] = {x[0], x[1]}, a1[2] = {x[2], x[3]};
                    store_row<Dt>(a.out[1], dst + row * D + 64 * u + 2 * c0, a0);
                    store_row<Dt>(a.out[1], dst + row * D + 64 * u + 32 + 2 * c0, a1);
                } else {
                    store_row<Dt>(a.out[1], dst + row * D + 64 * u + 4 * c0, x);
                }
            }
}

// A wave per record.  The same four prompts back: 25 us for 33 MB of codes and 134 MB of rows (6.5 TB/s), the stores' bandwidth.
template <int D, int GROUP, int Dt>
__global__ __launch_bounds__(256) void int4_read_kernel(ReadArgs a) {
    using R = Int4Rec<D, GROUP>;
    const int b = a.b0 + blockIdx.z, h = blockIdx.y, lane = threadIdx.x % kWave;
    const int start = a.starts[blockIdx.z], len = int4_len(a.L, b);
    const int block = start / kBlock + static_cast<int>(blockIdx.x) * 4 + in_sgpr(static_cast<int>(threadIdx.x / kWave));
    const int64_t pos0 = static_cast<int64_t>(block) * kBlock, end = static_cast<int64_t>(start) + a.tokens;
    if (pos0 >= end) return;
    const bool there = pos0 < len;
    const uint8_t* rec = int4_block(a.L, b, h, there ? block : 0, R::bytes);
    // element 0 of the row of the record's token 0, which may lie in front of the first
    const int64_t dst = ((static_cast<int64_t>(b) * a.L.n_kv + h) * a.tokens + (pos0 - start)) * D;
    const int from = static_cast<int>(max(start - pos0, static_cast<int64_t>(0))), to = static_cast<int>(min(end - pos0, static_cast<int64_t>(kBlock)));
    const int seen = static_cast<int>(min(max(len - pos0, static_cast<int64_t>(0)), static_cast<int64_t>(kBlock)));
    // (a whole record: all of its loads on their way before the first store)
    if (from == 0 && to == kBlock && seen == kBlock) read_record<D, GROUP, Dt, true>(a, rec, dst, 0, kBlock, kBlock, lane);
    else read_record<D, GROUP, Dt, false>(a, rec, dst, from, to, seen, lane);
}

template <int D, int GROUP, int Dt>
void append_typed(const RowsArgs& a, int batch, hipStream_t stream) {
    const lf_int4_layer& L = a.L;
    if (a.tokens <= kFewTokens && !a.started) {
        hipLaunchKernelGGL((int4_append_few_kernel<D, GROUP, Dt>), dim3(batch), dim3((D > 128 ? 4 : 8) * kWave), 0, stream, a);
        return;
    }
    const int P = L.page_size, waves = min(4, P / kBlock);
    const int64_t pages = (static_cast<int64_t>(a.tokens) + 2 * P - 2) / P;  // that a run of tokens can touch
    const int64_t here = min(pages, static_cast<int64_t>(L.cap_tokens / P) + 1);
    hipLaunchKernelGGL((int4_append_pages_kernel<D, GROUP, Dt>), dim3(static_cast<uint32_t>(here), L.n_kv, batch),
                       dim3(waves * kWave), 0, stream, a);
    if (!a.started) hipLaunchKernelGGL(int4_advance_kernel, dim3(1), dim3(kInlineSeqs), 0, stream, a);
}

int last_error() {
    const hipError_t err = hipGetLastError();
    return err == hipSuccess ? LF_OK : static_cast<int>(err);
}

}  // namespace

int launch_int4_set_lens(const lf_int4_layer& L, const int32_t* lens, hipStream_t stream) {
    for (int b0 = 0; b0 < L.batch; b0 += kInlineLens) {
        LensArgs a{L.lens, b0, min(kInlineLens, L.batch - b0), {}};
        for (int i = 0; i < a.n; ++i) a.value[i] = lens[b0 + i];
        hipLaunchKernelGGL(int4_set_lens_kernel, dim3(1), dim3(kInlineLens), 0, stream, a);
    }
    return last_error();
}

int launch_int4_append(const lf_int4_layer& L, const void* k_src, const void* v_src, int dtype, const int64_t* k_strides,
                       const int64_t* v_strides, const int32_t* starts, const int32_t* counts, int tokens,
                       hipStream_t stream) {
    RowsArgs a{};
    a.L = L;
    a.src[0] = k_src; a.src[1] = v_src;
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
    a.counted = counts != nullptr;
    a.started = starts != nullptr;
    return int4_dispatch(L, [&](auto shape) {
        constexpr int D = decltype(shape)::d, GROUP = decltype(shape)::group;
        for (a.b0 = 0; a.b0 < L.batch; a.b0 += kInlineSeqs) {
            const int n = min(kInlineSeqs, L.batch - a.b0);
            for (int i = 0; i < n && counts; ++i) a.counts[i] = counts[a.b0 + i];
            for (int i = 0; i < n && starts; ++i) a.starts[i] = starts[a.b0 + i];
            if (dtype == LF_BF16) append_typed<D, GROUP, LF_BF16>(a, n, stream);
            else if (dtype == LF_FP16) append_typed<D, GROUP, LF_FP16>(a, n, stream);
            else append_typed<D, GROUP, LF_FP32>(a, n, stream);
        }
        return last_error();
    });
}

int launch_int4_read(const lf_int4_layer& L, const int32_t* starts, int tokens, void* k_out, void* v_out, int dtype,
                     hipStream_t stream) {
    ReadArgs a{};
    a.L = L;
    a.tokens = tokens;
    a.out[0] = k_out; a.out[1] = v_out;
    return int4_dispatch(L, [&](auto shape) {
        constexpr int D = decltype(shape)::d, GROUP = decltype(shape)::group;
        const int64_t records = (static_cast<int64_t>(tokens) + 2 * kBlock - 2) / kBlock;  // that a run of tokens can touch
        for (a.b0 = 0; a.b0 < L.batch; a.b0 += kInlineSeqs) {
            const int n = min(kInlineSeqs, L.batch - a.b0);
            for (int i = 0; i < n; ++i) a.starts[i] = starts ? starts[a.b0 + i] : 0;
            const dim3 grid(static_cast<uint32_t>((records + 3) / 4), L.n_kv, n);
            if (dtype == LF_BF16) hipLaunchKernelGGL((int4_read_kernel<D, GROUP, LF_BF16>), grid, dim3(256), 0, stream, a);
            else if (dtype == LF_FP16) hipLaunchKernelGGL((int4_read_kernel<D, GROUP, LF_FP16>), grid, dim3(256), 0, stream, a);
            else hipLaunchKernelGGL((int4_read_kernel<D, GROUP, LF_FP32>), grid, dim3(256), 0, stream, a);
        }
        return last_error();
    });
}

}  // namespace lf
