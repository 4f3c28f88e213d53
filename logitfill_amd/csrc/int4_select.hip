// Page selection of the 4-bit row cache: a score per page from its Keys' bounds, and the pages of highest score.
//
// score(page) = max over the kv head's query heads of sum_c max(q_c lo_c, q_c hi_c): no Key of the page has a larger
// q . k.  Products of a bf16 bound and a query element are exact in float64: 16 bits of a bf16 query's, 19 of fp16's, 32
// of float32's.  So is their sum, and the choice then does not hang on its order, where the product's bits, the spans of the
// query's elements and of the page's bounds and log2(head_dim) come to 53 together: at head_dim 128 spans of 2^30, 2^27 and 2^14
// in all.  Beyond that a sum is off by 2^-53 of sum |q bound| a step, and of pages closer than that any may be chosen.
#include "int4_common.hpp"

namespace lf {
namespace {

struct SelectArgs {
    lf_int4_layer L;
    const void* q;
    int64_t qb, qh, qt;
    const int32_t* q_lens;
    int g, q_len, dtype;
    int vec;  // 2-byte query rows that start on 16 bytes
    int n_pages;
    int32_t* pages;
    uint64_t* keys;  // [batch][n_kv][q_len][cap_tokens / page_size]
};

// The pages in front of query token j's own one (0 where it has none, or is no token of the sequence).
__device__ __forceinline__ int candidates(const SelectArgs& a, int b, int j) {
    const int len = int4_len(a.L, b);
    const int n = a.q_lens ? min(max(a.q_lens[b], 0), a.q_len) : a.q_len;
    const int at = len - n + j;
    return j < n && at > 0 ? at / a.L.page_size : 0;
}

// Larger scores have larger keys; NaN the smallest.
__device__ __forceinline__ uint64_t score_key(double x) {
    if (x != x) return 0;
    const uint64_t u = __builtin_bit_cast(uint64_t, x + 0.0);  // (-0 and 0 are one score)
    return u >> 63 ? ~u : u | 0x8000000000000000ull;
}


// D / 8 lanes take a page, eight channels each, and eight heads at a time: the heads' elements stay in registers, the
// bounds are widened once for all heads, and the heads' sums are exchanged so that each step of the butterfly halves the
// heads a lane still adds up.  11 us for 16 384 pages of 128 channels and 7 heads, 8.4 MB, and neither of them bounds it: a
// wave issues some 970 vector instructions around 64 float64 sums a lane (both operands widened, a select per product, the
// exchanges of doubles), one after the other's result, the VALU 32 % busy.  Measured beside it: four pages a lane with the queries kept in
// float64, 21 us (256 registers, one wave a SIMD); products of float64 matrix instructions, max(q, 0) hi + min(q, 0) lo
// over tiles of sixteen heads, 9 us, and 22 in one launch with the choice below (they do four times the products).
constexpr int kHeads = 8;
constexpr int score_pages(int D) { return 256 / (D / 8); }  // of a workgroup

__device__ __forceinline__ double other(double x, int mask) { return __shfl_xor(x, mask, kWave); }

template <int D>
__global__ __launch_bounds__(256) void int4_score_kernel(SelectArgs a) {
    constexpr int LR = D / 8;
    static_assert(LR >= kHeads, "a lane per head");
    const int b = blockIdx.z, h = blockIdx.y / a.q_len, j = blockIdx.y % a.q_len;
    const int count = candidates(a, b, j);
    const int p0 = blockIdx.x * score_pages(D);
    if (p0 >= count || count <= a.n_pages) return;
    const int w = threadIdx.x % LR, page = p0 + threadIdx.x / LR;
    const int pages = a.L.cap_tokens / a.L.page_size;
    const uint16_t* bounds = a.L.bounds + ((static_cast<int64_t>(b) * a.L.n_kv + h) * pages + min(page, count - 1)) * 2 * D + 8 * w;
    const u32x4 lo = *reinterpret_cast<const u32x4*>(bounds), hi = *reinterpret_cast<const u32x4*>(bounds + D);
    double best = -__builtin_inf();
    int nan = 0;
    for (int i0 = 0; i0 < a.g; i0 += kHeads) {
        double sum[kHeads];
#pragma unroll
        for (int k = 0; k < kHeads; ++k) {
            // (heads past the group repeat its last one)
            const int64_t at = b * a.qb + static_cast<int64_t>(h * a.g + min(i0 + k, a.g - 1)) * a.qh + j * a.qt + 8 * w;
            float q[8];
            if (a.vec) {
                const u32x4 x = *reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(a.q) + at);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const uint16_t u = static_cast<uint16_t>(x[e >> 1] >> (16 * (e & 1)));
                    q[e] = a.dtype == LF_BF16 ? bf16_to_f32(u) : f16_to_f32(u);
                }
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) q[e] = load_as_f32(a.q, at + e, a.dtype);
            }
            sum[k] = 0.;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const double l = __uint_as_float(e & 1 ? lo[e >> 1] & 0xffff0000u : lo[e >> 1] << 16);
                const double u = __uint_as_float(e & 1 ? hi[e >> 1] & 0xffff0000u : hi[e >> 1] << 16);
                sum[k] = fma(static_cast<double>(q[e]), q[e] < 0.f ? l : u, sum[k]);
            }
        }
        // lanes w and w ^ m split the heads that are left, then the lanes of one head add up
#pragma unroll
        for (int m = 1, left = kHeads / 2; left > 0; m <<= 1, left >>= 1)
#pragma unroll
            for (int k = 0; k < left; ++k) {
                const bool upper = w & m;
                const double keep = upper ? sum[k + left] : sum[k], give = upper ? sum[k] : sum[k + left];
                sum[k] = keep + other(give, m);
            }
#pragma unroll
        for (int m = kHeads; m < LR; m <<= 1) sum[0] += other(sum[0], m);
        nan |= sum[0] != sum[0];
        best = sum[0] > best ? sum[0] : best;
    }
#pragma unroll
    for (int m = 1; m < kHeads; m <<= 1) {
        const double o = other(best, m);
        best = o > best ? o : best;
        nan |= __shfl_xor(nan, m, kWave);
    }
    if (page < count && w == 0) a.keys[((static_cast<int64_t>(b) * a.L.n_kv + h) * a.q_len + j) * pages + page] = nan ? 0 : score_key(best);
}

// A workgroup per (query token, kv head): the n_pages-th largest key, eight bits at a time (as far as the pages at
// the prefix are more than are needed), then the pages above it and the first of those at it, in order.  Thread t
// holds keys t, t + T, .. in registers (``Hold`` of them, 0: any number, read anew).  4.5 us for 128 pages, 11.5 for 4 096:
// bound by the rounds' barriers, some five of eight bits each, not by the keys.
template <int T, int Hold>
__global__ __launch_bounds__(T) void int4_top_kernel(SelectArgs a) {
    constexpr int W = T / kWave;
    __shared__ int hist[256];
    __shared__ int found[3];  // bucket, keys above it, keys in it
    __shared__ int sums[2][2][W];
    const int b = blockIdx.z, h = blockIdx.y / a.q_len, j = blockIdx.y % a.q_len, tid = threadIdx.x;
    const int lane = tid % kWave, wave = tid / kWave;
    const int count = candidates(a, b, j), top = a.n_pages;
    const int pages = a.L.cap_tokens / a.L.page_size;
    const int64_t slot = (static_cast<int64_t>(b) * a.L.n_kv + h) * a.q_len + j;
    int32_t* out = a.pages + slot * top;
    if (count <= top) {
        for (int k = tid; k < top; k += T) out[k] = k < count ? k : -1;
        return;
    }
    const uint64_t* keys = a.keys + slot * pages;
    uint64_t held[Hold ? Hold : 1];
    if constexpr (Hold > 0)
#pragma unroll
        for (int s = 0; s < Hold; ++s) held[s] = s * T + tid < count ? keys[s * T + tid] : 0;
    const auto each = [&](auto&& fn) {
        if constexpr (Hold > 0) {
#pragma unroll
            for (int s = 0; s < Hold; ++s)
                if (s * T < count) fn(s * T + tid, held[s]);
        } else {
            for (int k0 = 0; k0 < count; k0 += T) fn(k0 + tid, k0 + tid < count ? keys[k0 + tid] : 0);
        }
    };
    uint64_t prefix = 0;
    int need = top, shift = 56;  // keys still to find among those whose upper bits are the prefix
    for (;; shift -= 8) {
        if (tid < 256) hist[tid] = 0;
        __syncthreads();
        each([&](int k, uint64_t key) {
            const bool in = k < count && (shift == 56 || key >> (shift + 8) == prefix);
            const int digit = static_cast<int>(key >> shift) & 255;
            // a wave whose keys share the digit (the first ones: sign and exponent) counts them at once
            const uint64_t mask = __ballot(in);
            if (mask == 0) return;
            const int lead = __builtin_amdgcn_readlane(digit, __builtin_ctzll(mask));
            const uint64_t same = __ballot(in && digit == lead);
            if (lane == 0) atomicAdd(&hist[lead], __popcll(same));
            if (in && digit != lead) atomicAdd(&hist[digit], 1);
        });
        __syncthreads();
        if (wave == 0) {
            // lane i: buckets 255 - 4 i down to 252 - 4 i
            int n[4], mine = 0;
#pragma unroll
            for (int c = 0; c < 4; ++c) { n[c] = hist[255 - 4 * lane - c]; mine += n[c]; }
            int upto = mine;
#pragma unroll
            for (int m = 1; m < kWave; m <<= 1) {
                const int o = __shfl_up(upto, m, kWave);
                upto += lane >= m ? o : 0;
            }
            int above = upto - mine;
            if (above < need && need <= upto) {
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    if (above < need && need <= above + n[c]) {
                        found[0] = 255 - 4 * lane - c;
                        found[1] = above;
                        found[2] = n[c];
                    }
                    above += n[c];
                }
            }
        }
        __syncthreads();
        prefix = prefix << 8 | static_cast<uint64_t>(found[0]);
        need -= found[1];
        if (found[2] == need || shift == 0) break;  // (uniform: all threads read the same)
    }
    int placed = 0, equal = 0, turn = 0;
    each([&](int k, uint64_t key) {
        const uint64_t upper = key >> shift;
        const bool at = k < count && upper == prefix, over = k < count && upper > prefix;
        const uint64_t at_mask = __ballot(at), over_mask = __ballot(over), below = (1ull << lane) - 1;
        if (lane == 0) {
            sums[turn][0][wave] = __popcll(at_mask);
            sums[turn][1][wave] = __popcll(over_mask);
        }
        __syncthreads();  // (one per round: the next one writes the other half)
        int at_before = equal + __popcll(at_mask & below), over_before = placed + __popcll(over_mask & below);
#pragma unroll
        for (int v = 0; v < W; ++v) {
            if (v < wave) { at_before += sums[turn][0][v]; over_before += sums[turn][1][v]; }
            equal += sums[turn][0][v];
            placed += sums[turn][1][v];
        }
        // in front of this one: all above the prefix, and of those at it as many as are needed
        const int place = over_before + min(at_before, need);
        if ((over || (at && at_before < need)) && place < top) out[place] = k;
        turn ^= 1;
    });
}

template <int T, int Hold>
void launch_top(const SelectArgs& a, hipStream_t stream) {
    hipLaunchKernelGGL((int4_top_kernel<T, Hold>), dim3(1, a.L.n_kv * a.q_len, a.L.batch), dim3(T), 0, stream, a);
}

}  // namespace

int64_t int4_keys_bytes(const lf_int4_layer& L, int q_len) {
    return static_cast<int64_t>(L.batch) * L.n_kv * q_len * (L.cap_tokens / L.page_size) * 8;
}

int launch_int4_select(const lf_int4_layer& L, const lf_int4_args& A, hipStream_t stream) {
    SelectArgs a{};
    a.L = L;
    a.q = A.query;
    a.qb = A.q_strides[0]; a.qh = A.q_strides[1]; a.qt = A.q_strides[2];
    a.q_lens = A.q_lens;
    a.g = A.n_q / L.n_kv; a.q_len = A.q_len; a.dtype = A.dtype;
    a.vec = A.dtype != LF_FP32 && reinterpret_cast<uintptr_t>(A.query) % 16 == 0;
    for (int i = 0; i < 3; ++i) a.vec = a.vec && A.q_strides[i] % 8 == 0;
    a.n_pages = A.n_pages;
    a.pages = A.pages;
    a.keys = static_cast<uint64_t*>(A.workspace);
    const int pages = L.cap_tokens / L.page_size;
    const dim3 grid((pages + score_pages(L.head_dim) - 1) / score_pages(L.head_dim), L.n_kv * A.q_len, L.batch);
    const int st = int4_dispatch(L, [&](auto shape) {
        hipLaunchKernelGGL((int4_score_kernel<decltype(shape)::d>), grid, dim3(256), 0, stream, a);
        return LF_OK;
    });
    if (st != LF_OK) return st;
    // By the capacity: the device alone knows the lengths.  Scores and choice of 8 (sequence, kv head)s, us: 1 000 pages
    // 12.2 with four waves, 16.2 with sixteen; 4 000 pages from sixteen waves' registers 25.0, from memory 29.5, 16 000 61.5
    // and 79.6.
    if (pages <= 1024) launch_top<256, 4>(a, stream);
    else if (pages <= 16384) launch_top<1024, 16>(a, stream);
    else launch_top<1024, 0>(a, stream);
    const hipError_t err = hipGetLastError();
    return err == hipSuccess ? LF_OK : static_cast<int>(err);
}

}  // namespace lf
