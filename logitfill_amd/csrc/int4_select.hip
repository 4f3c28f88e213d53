// Page selection of the 4-bit row cache: a score per page from its Keys' bounds, and the pages of highest score.
//
// score(page) = max over the kv head's query heads of sum_c max(q_c lo_c, q_c hi_c): no Key of the page has a larger
// q . k.  Products of a bf16 bound and a query element are exact in float64 and so, but for queries whose elements
// span more than 2^20, are their sums: the choice does not hang on the order in which they are formed.
#include "int4_common.hpp"

namespace lf {
namespace {

struct SelectArgs {
    lf_int4_layer L;
    const void* q;
    int64_t qb, qh, qt;
    const int32_t* q_lens;
    int g, q_len, dtype;
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


// D / 8 lanes take a page, eight channels each; a workgroup takes kScorePages pages of one (query token, kv head).
constexpr int kScorePages = 64;
template <int D>
__global__ __launch_bounds__(256) void int4_score_kernel(SelectArgs a) {
    constexpr int LR = D / 8, RP = 256 / LR;
    const int b = blockIdx.z, h = blockIdx.y / a.q_len, j = blockIdx.y % a.q_len;
    const int count = candidates(a, b, j);
    const int p0 = blockIdx.x * kScorePages;
    if (p0 >= count || count <= a.n_pages) return;
    const int w = threadIdx.x % LR;
    const int pages = a.L.cap_tokens / a.L.page_size;
    const uint16_t* bounds = a.L.bounds + (static_cast<int64_t>(b) * a.L.n_kv + h) * pages * 2 * D + 8 * w;
    uint64_t* keys = a.keys + ((static_cast<int64_t>(b) * a.L.n_kv + h) * a.q_len + j) * pages;
    const int p1 = min(p0 + kScorePages, count);
    for (int base = p0; base < p1; base += RP) {
        const int page = base + threadIdx.x / LR, from = min(page, p1 - 1);
        const u32x4 lo = *reinterpret_cast<const u32x4*>(bounds + static_cast<int64_t>(from) * 2 * D);
        const u32x4 hi = *reinterpret_cast<const u32x4*>(bounds + static_cast<int64_t>(from) * 2 * D + D);
        double best = -__builtin_inf();
        bool bad = false;
        for (int i = 0; i < a.g; ++i) {
            double sum = 0.;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float q = load_as_f32(a.q, b * a.qb + static_cast<int64_t>(h * a.g + i) * a.qh + j * a.qt + 8 * w + e, a.dtype);
                const uint32_t l = e & 1 ? lo[e >> 1] & 0xffff0000u : lo[e >> 1] << 16, u = e & 1 ? hi[e >> 1] & 0xffff0000u : hi[e >> 1] << 16;
                const float k = __uint_as_float(q < 0.f ? l : u);
                sum = fma(static_cast<double>(q), static_cast<double>(k), sum);
            }
#pragma unroll
            for (int m = 1; m < LR; m <<= 1) sum += __shfl_xor(sum, m, kWave);
            bad |= sum != sum;
            best = sum > best ? sum : best;
        }
        if (page < p1 && w == 0) keys[page] = bad ? 0 : score_key(best);
    }
}

// A workgroup per (query token, kv head): the n_pages-th largest key, eight bits at a time, then the pages above it
// and the first of those at it, in order.
__global__ __launch_bounds__(256) void int4_top_kernel(SelectArgs a) {
    __shared__ int hist[256];
    __shared__ int found[2];      // bucket, keys above it
    __shared__ int wave_sum[2][4];
    const int b = blockIdx.z, h = blockIdx.y / a.q_len, j = blockIdx.y % a.q_len, tid = threadIdx.x;
    const int count = candidates(a, b, j), top = a.n_pages;
    const int pages = a.L.cap_tokens / a.L.page_size;
    const int64_t slot = (static_cast<int64_t>(b) * a.L.n_kv + h) * a.q_len + j;
    int32_t* out = a.pages + slot * top;
    if (count <= top) {
        for (int k = tid; k < top; k += 256) out[k] = k < count ? k : -1;
        return;
    }
    const uint64_t* keys = a.keys + slot * pages;
    uint64_t prefix = 0;
    int need = top;  // keys still to find at the prefix
    for (int shift = 56; shift >= 0; shift -= 8) {
        hist[tid] = 0;
        __syncthreads();
        for (int k = tid; k < count; k += 256)
            if (shift == 56 || keys[k] >> (shift + 8) == prefix) atomicAdd(&hist[(keys[k] >> shift) & 255], 1);
        __syncthreads();
        if (tid == 0) {
            int above = 0, bucket = 255;
            while (bucket > 0 && above + hist[bucket] < need) above += hist[bucket--];
            found[0] = bucket;
            found[1] = above;
        }
        __syncthreads();
        prefix = prefix << 8 | static_cast<uint64_t>(found[0]);
        need -= found[1];
        __syncthreads();
    }
    // keys above the prefix are in, and the first ``need`` equal to it
    int placed = 0, equal = 0;
    for (int k0 = 0; k0 < count; k0 += 256) {
        const int k = k0 + tid;
        const uint64_t key = k < count ? keys[k] : 0;
        const bool is_equal = k < count && key == prefix;
        const uint64_t eq = __ballot(is_equal);
        const int lane = tid % kWave, wave = tid / kWave;
        const uint64_t below = (1ull << lane) - 1;
        if (lane == 0) wave_sum[0][wave] = __popcll(eq);
        __syncthreads();
        int eq_before = equal + __popcll(eq & below), eq_all = equal;
        for (int v = 0; v < 4; ++v) {
            if (v < wave) eq_before += wave_sum[0][v];
            eq_all += wave_sum[0][v];
        }
        const bool in = k < count && (key > prefix || (is_equal && eq_before < need));
        const uint64_t take = __ballot(in);
        if (lane == 0) wave_sum[1][wave] = __popcll(take);
        __syncthreads();
        int at = placed + __popcll(take & below);
        for (int v = 0; v < 4; ++v) {
            if (v < wave) at += wave_sum[1][v];
            placed += wave_sum[1][v];
        }
        equal = eq_all;
        if (in && at < top) out[at] = k;
        __syncthreads();
    }
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
    a.n_pages = A.n_pages;
    a.pages = A.pages;
    a.keys = static_cast<uint64_t*>(A.workspace);
    const int pages = L.cap_tokens / L.page_size;
    const dim3 grid((pages + kScorePages - 1) / kScorePages, L.n_kv * A.q_len, L.batch);
    const int st = int4_dispatch(L, [&](auto shape) {
        hipLaunchKernelGGL((int4_score_kernel<decltype(shape)::d>), grid, dim3(256), 0, stream, a);
        return LF_OK;
    });
    if (st != LF_OK) return st;
    hipLaunchKernelGGL(int4_top_kernel, dim3(1, L.n_kv * A.q_len, L.batch), dim3(256), 0, stream, a);
    const hipError_t err = hipGetLastError();
    return err == hipSuccess ? LF_OK : static_cast<int>(err);
}

}  // namespace lf
