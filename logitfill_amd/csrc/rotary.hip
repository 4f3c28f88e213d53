// Rotary positions: pairs of a row's channels are turned by an angle that grows with the token's position,
//     (x, y) -> factor (x cos t - y sin t, y cos t + x sin t),   t = position * frequency of the pair.
//
// The angle is formed in 64 bits as turns (position * frequency / 2 pi), of which the whole ones are dropped before
// sine and cosine: a float32 angle of position 2^20 is off by 0.03.  A workgroup forms the sines and cosines of its tokens
// once, in LDS, for all their query and Key heads; rows pass through in 16-byte pieces, two a lane (both halves of its
// pairs), Query and Key in one launch.  The rotation itself is in fp32, rounded once.
//
// Bound by HBM: four prompts of up to 16 300 tokens, 28 + 4 heads of 128, bf16: 582 MB read and written in 110 us, 5.3 TB/s (a
// 1 GiB copy: 4.8 to 5.1), VALU 63 % busy.  One token of eight sequences: 3.9 us on the GPU, 7.6 a call.
#include "lf_common.hpp"

namespace lf {
namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
constexpr int kThreads = 256, kMaxTokens = 16;

struct RotaryLaunch {
    lf_rotary_args A;
    int tokens_per;      // tokens of a workgroup
    uint32_t heads_inv;  // ceil(2^32 / (n_q + n_kv)): exact for rows below 2^32 / heads
    int per_head;        // lanes of a row: pieces of Vec pairs, rotated ones first
    int rotated;         // of them
};

template <int Dt, int Vec>
__device__ __forceinline__ void load_piece(const void* p, int64_t at, float (&x)[Vec]) {
    if constexpr (Vec == 1) {
        x[0] = load_as_f32(p, at, Dt);
    } else if constexpr (Dt == LF_FP32) {
        const u32x4 w = *reinterpret_cast<const u32x4*>(static_cast<const float*>(p) + at);
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = __uint_as_float(w[e]);
    } else {
        const u32x4 w = *reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(p) + at);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const uint16_t h = static_cast<uint16_t>(w[e >> 1] >> (16 * (e & 1)));
            x[e] = Dt == LF_BF16 ? bf16_to_f32(h) : f16_to_f32(h);
        }
    }
}

template <int Dt, int Vec>
__device__ __forceinline__ void store_piece(void* p, int64_t at, const float (&x)[Vec]) {
    if constexpr (Vec == 1) {
        store_from_f32(p, at, Dt, x[0]);
    } else if constexpr (Dt == LF_FP32) {
        *reinterpret_cast<u32x4*>(static_cast<float*>(p) + at) =
            u32x4{__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3])};
    } else {
        u32x4 w;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const uint32_t lo = Dt == LF_BF16 ? f32_to_bf16(x[2 * e]) : f32_to_f16(x[2 * e]);
            const uint32_t hi = Dt == LF_BF16 ? f32_to_bf16(x[2 * e + 1]) : f32_to_f16(x[2 * e + 1]);
            w[e] = lo | hi << 16;
        }
        *reinterpret_cast<u32x4*>(static_cast<uint16_t*>(p) + at) = w;
    }
}

// Vec pairs a lane: 8 of 16-bit rows and 4 of float32 (16 bytes of each half), or 1 where sizes, strides or
// addresses do not allow it.
template <int Dt, int Vec, bool Interleaved>
__global__ __launch_bounds__(kThreads) void rotary_kernel(RotaryLaunch a) {
    extern __shared__ float2 turned[];  // [tokens_per][rotary_dim / 2] cosines and sines
    __shared__ int2 where[kMaxTokens];  // (sequence, token) of the workgroup's tokens
    const lf_rotary_args& A = a.A;
    const int pairs = A.rotary_dim / 2, heads = A.n_q + A.n_kv;
    const uint32_t first = blockIdx.x * static_cast<uint32_t>(a.tokens_per);  // (all tokens are fewer than 2^27)
    const int tokens = static_cast<int>(min(static_cast<uint32_t>(a.tokens_per), static_cast<uint32_t>(A.batch) * A.tokens - first));
    if (threadIdx.x < tokens) {
        const uint32_t at = first + threadIdx.x, b = at / A.tokens;
        where[threadIdx.x] = int2{static_cast<int>(b), static_cast<int>(at - b * A.tokens)};
    }
    __syncthreads();
    for (int i = threadIdx.x; i < tokens * pairs; i += kThreads) {
        const int t = i / pairs, j = i - t * pairs;
        const int64_t place = where[t].x * A.position_strides[0] + where[t].y * A.position_strides[1];
        const double position = !A.positions ? static_cast<double>(A.start + where[t].y)
                                : A.wide ? static_cast<double>(static_cast<const int64_t*>(A.positions)[place])
                                         : static_cast<double>(static_cast<const int32_t*>(A.positions)[place]);
        const double turns = position * A.turns[j];
        double sine, cosine;
        sincospi(2.0 * (turns - rint(turns)), &sine, &cosine);
        turned[i] = float2{static_cast<float>(cosine * A.factor), static_cast<float>(sine * A.factor)};
    }
    __syncthreads();
    const int rows = tokens * heads;
    const int step = kThreads / a.per_head;  // rows that the workgroup takes at once
    const int piece = threadIdx.x % a.per_head;
    const bool turn = piece < a.rotated;
    int c0, c1;  // first channels of the lane's two pieces
    if (!turn) {
        c0 = A.rotary_dim + (piece - a.rotated) * 2 * Vec;
        c1 = c0 + Vec;
    } else if (Interleaved) {
        c0 = piece * 2 * Vec;
        c1 = c0 + Vec;
    } else {
        c0 = piece * Vec;
        c1 = pairs + c0;
    }
    if (static_cast<int>(threadIdx.x) >= step * a.per_head) return;
    for (int row = threadIdx.x / a.per_head; row < rows; row += step) {
        const int t = heads == 1 ? row : static_cast<int>(__umulhi(static_cast<uint32_t>(row), a.heads_inv));
        const int h = row - t * heads;
        const int64_t b = where[t].x, s = where[t].y;
        const bool key = h >= A.n_q;
        const int64_t hh = key ? h - A.n_q : h;
        const void* src = key ? A.key : A.query;
        void* dst = key ? A.key_out : A.query_out;
        const int64_t from = key ? b * A.k_strides[0] + hh * A.k_strides[1] + s * A.k_strides[2]
                                 : b * A.q_strides[0] + hh * A.q_strides[1] + s * A.q_strides[2];
        const int64_t to = key ? b * A.ko_strides[0] + hh * A.ko_strides[1] + s * A.ko_strides[2]
                               : b * A.qo_strides[0] + hh * A.qo_strides[1] + s * A.qo_strides[2];
        float x[Vec], y[Vec];
        load_piece<Dt, Vec>(src, from + c0, x);
        load_piece<Dt, Vec>(src, from + c1, y);
        if (turn) {
            const float2* cs = turned + t * pairs + piece * Vec;
#pragma unroll
            for (int e = 0; e < Vec; ++e) {
                const float2 w = cs[e];
                // interleaved: elements 2 e, 2 e + 1 of the 2 Vec channels are a pair
                float& u = Interleaved && Vec > 1 ? (2 * e < Vec ? x[(2 * e) % Vec] : y[(2 * e) % Vec]) : x[e];
                float& v = Interleaved && Vec > 1 ? (2 * e < Vec ? x[(2 * e + 1) % Vec] : y[(2 * e + 1) % Vec]) : y[e];
                const float p = u, q = v;
                u = fmaf(p, w.x, -(q * w.y));
                v = fmaf(q, w.x, p * w.y);
            }
        }
        store_piece<Dt, Vec>(dst, to + c0, x);
        store_piece<Dt, Vec>(dst, to + c1, y);
    }
}

template <int Dt, int Vec>
void launch_typed(const RotaryLaunch& a, uint32_t groups, size_t lds, hipStream_t stream) {
    if (a.A.interleaved) hipLaunchKernelGGL((rotary_kernel<Dt, Vec, true>), dim3(groups), dim3(kThreads), lds, stream, a);
    else hipLaunchKernelGGL((rotary_kernel<Dt, Vec, false>), dim3(groups), dim3(kThreads), lds, stream, a);
}

bool aligned(const void* p, const int64_t (&strides)[3], int esize) {
    bool ok = reinterpret_cast<uintptr_t>(p) % 16 == 0;
    for (const int64_t s : strides) ok = ok && s * esize % 16 == 0;
    return ok;
}

}  // namespace

int launch_rotary(const lf_rotary_args& A, hipStream_t stream) {
    RotaryLaunch a{};
    a.A = A;
    const int esize = A.dtype == LF_FP32 ? 4 : 2, vec = 16 / esize, heads = A.n_q + A.n_kv;
    bool wide = A.rotary_dim / 2 % vec == 0 && (A.head_dim - A.rotary_dim) % (2 * vec) == 0;
    if (A.n_q) wide = wide && aligned(A.query, A.q_strides, esize) && aligned(A.query_out, A.qo_strides, esize);
    if (A.n_kv) wide = wide && aligned(A.key, A.k_strides, esize) && aligned(A.key_out, A.ko_strides, esize);
    const int pairs = wide ? vec : 1;
    a.per_head = A.head_dim / 2 / pairs;
    a.rotated = A.rotary_dim / 2 / pairs;
    a.heads_inv = static_cast<uint32_t>(((1ull << 32) + heads - 1) / heads);  // (of one head: unused)
    // A sine and cosine per thread or so, unless that leaves compute units without a workgroup.
    const int64_t tokens = static_cast<int64_t>(A.batch) * A.tokens;
    int64_t per = 2 * kThreads / A.rotary_dim;
    per = per < tokens / 1024 ? per : tokens / 1024;
    const int64_t least = (tokens + (1 << 23) - 1) >> 23;  // (2^32 threads in a grid)
    per = per < least ? least : per;
    a.tokens_per = static_cast<int>(per < 1 ? 1 : per > kMaxTokens ? kMaxTokens : per);
    const uint32_t groups = static_cast<uint32_t>((tokens + a.tokens_per - 1) / a.tokens_per);
    const size_t lds = static_cast<size_t>(a.tokens_per) * (A.rotary_dim / 2) * sizeof(float2);
    switch (A.dtype * 2 + wide) {
        case LF_BF16 * 2: launch_typed<LF_BF16, 1>(a, groups, lds, stream); break;
        case LF_BF16 * 2 + 1: launch_typed<LF_BF16, 8>(a, groups, lds, stream); break;
        case LF_FP16 * 2: launch_typed<LF_FP16, 1>(a, groups, lds, stream); break;
        case LF_FP16 * 2 + 1: launch_typed<LF_FP16, 8>(a, groups, lds, stream); break;
        case LF_FP32 * 2: launch_typed<LF_FP32, 1>(a, groups, lds, stream); break;
        default: launch_typed<LF_FP32, 4>(a, groups, lds, stream);
    }
    const hipError_t err = hipGetLastError();
    return err == hipSuccess ? LF_OK : static_cast<int>(err);
}

}  // namespace lf
