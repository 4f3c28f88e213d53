// Attention over the 4-bit row cache, on the matrix cores.
//
// Scores of 16 tokens and 16 query rows: S^T = Codes . Q^T on v_mfma_f32_16x16x32_bf16, per group g of channels
//     s_t = sum_g scale_t,g (q_g . code_t,g) + min_t,g sum(q_g),
// and the Value product O^T = Codes_V^T . P'^T with P'_t,g = p_t scale_t,g,
//     o_c = sum_t P'_t,g code_t,c + p_t min_t,g.
// A score's lane holds the tokens of exactly the P' operand its lane of the second product needs (Value words hold
// eight tokens of a channel in that order), so nothing is exchanged between the two products.
//
// Codes enter as 16 + code, Keys' in bf16 and Values' in fp16 (one and-or per pair); the 16 is taken out of the scores
// by the accumulator's start value, -16 sum(q_g), and out of the output by a product of P' with a constant.  Queries are
// split into bf16 parts that add up to them exactly (bf16 one, fp16 two).  P' is rounded to fp16, in as many
// parts as the output's type asks for (one, two, two); the codes count from their middle, 7.5, there (sum p (min +
// 7.5 scale) is kept in fp32), so that a rounding of P' weighs as the code's distance from it.  In one part of bf16 the
// roundings of P' were as large as the bf16 output's own (rel. error 2.4e-3 to 2.7e-3 against 1.7e-3); fp16's eight times
// smaller ones need P' in its range: the reference point is moved by log2 of the largest Value scale of the wave's records
// (tops), so that P' stays below 2^15; in two parts, where a group's scales are 2^r below that, its P' is raised by 2^r (a group
// whose Values are 2^10 smaller had a rel. error of 9e-6 in float32, 2^14 smaller 2e-4, against 4e-8 alone).  One part
// loses a weight 2^-31 2^r of its row's largest, r counted from the largest scale of a wave's records; two of them for bf16 rows
// would take their error from 1.683e-3 to the output's own 1.669e-3, and the calls below from 61 to 68 us and 295 to 360.
//
// float32 rows keep more: there both products take code - 7.5 in fp16 (one packed sum per pair), for the 16 and the middle
// are three times what the codes themselves reach and leave their roundings in the scores (rel. error 1.7e-6 to 2.7e-6
// with them, 2e-7 to 4e-7 without), and the queries, times the power of two that fits them into fp16, enter in three fp16 parts.
//
// A workgroup's four waves take the records of its split in turn, each with its own running reference point and
// sums, merged through LDS at the end; several splits of a sequence are merged by int4_merge_kernel.  The
// reference point of a row moves only when a score passes it by 2^8: p stays below 2^8 and the sums are rescaled
// rarely.
// A layer of 16 sequences of 32K tokens (28 / 4 heads of 128, groups of 64, one query each): a call of 57 us, 53 in this kernel
// for 304 MB, 5.7 TB/s, VALU 61 % and matrix cores 14 % busy.  32 ragged ones of 4K to 64K (40 / 8 heads, groups of 32): a
// call of 299 us for 1.36 GB, 4.6 TB/s (under the profiler this kernel alone takes 305 to 410), VALU 65 %: the memory first,
// then the unpacking (four masks and shifts a word) and the factors of 32 channels each.
//
// Registers (the compiler's report): none are spilled but at <128, 32>, 5, 25 and 44 for bf16, fp16 and float32, <256, 32>, 64, 83
// and 148, and <256, 64> float32, 30.
#include "int4_common.hpp"

#include <type_traits>

namespace lf {
int launch_int4_prefix(const Int4Attention& a, hipStream_t stream);
int launch_int4_shared_rows(const Int4Shared& a, hipStream_t stream);

namespace {

constexpr int kWaves = 4, kTile = 16;

template <int NT>
struct Parts {
    bf16x8 t[NT];
};

__device__ __forceinline__ uint32_t upper_pair(float a, float b) {
    return __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
}
__device__ __forceinline__ float upper(float x) { return __uint_as_float(__float_as_uint(x) & 0xffff0000u); }
// Element pairs (a[i], b[i]) in NT bf16 parts; the last part is rounded to nearest, those before it are cut off.
template <int NT>
__device__ __forceinline__ Parts<NT> split(const float (&a)[4], const float (&b)[4]) {
    Parts<NT> r;
    float x[4], y[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) { x[i] = a[i]; y[i] = b[i]; }
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        u32x4 w;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            w[i] = n + 1 < NT ? upper_pair(x[i], y[i]) : pack_bf16(x[i], y[i]);
            if (n + 1 < NT) { x[i] -= upper(x[i]); y[i] -= upper(y[i]); }
        }
        r.t[n] = __builtin_bit_cast(bf16x8, w);
    }
    return r;
}

__device__ __forceinline__ f32x4 mfma(bf16x8 a, bf16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma(f16x8 a, f16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// Element pairs (a[i], b[i]) in NP fp16 parts, each rounded to nearest.
template <int NP>
struct HalfParts {
    f16x8 t[NP];
};
template <int NP>
__device__ __forceinline__ HalfParts<NP> half_parts(const float (&a)[4], const float (&b)[4]) {
    HalfParts<NP> r;
    float x[4], y[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) { x[i] = a[i]; y[i] = b[i]; }
#pragma unroll
    for (int n = 0; n < NP; ++n) {
        u32x4 w;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            w[i] = pack_f16(x[i], y[i]);
            if (n + 1 < NP) {
                const uint32_t pair = w[i];
                x[i] -= pair_scale(pair);
                y[i] -= pair_min(pair);  // (the pair's upper half)
            }
        }
        r.t[n] = __builtin_bit_cast(f16x8, w);
    }
    return r;
}

// LDS reads stay behind this point: hoisted all to a record's start they take more registers than three waves a
// SIMD leave.
__device__ __forceinline__ void phase() { asm volatile("" ::: "memory"); }

// A wave's ring of records in LDS, filled by DMA: ``kRing`` - 1 of them are on their way while one is worked on.
constexpr int kRing = 2;
template <int D, int GROUP>
struct Ring {
    using R = Int4Rec<D, GROUP>;
    static constexpr int loads = (R::bytes + 1023) / 1024;  // DMA instructions a record takes
    static constexpr int bytes = kWaves * kRing * R::bytes;
    static constexpr int pad = D + 4;                       // floats between rows of the waves' merge
    static constexpr int merge = (kWaves - 1) * kTile * pad * 4;
    static constexpr int lds = bytes > merge ? bytes : merge;

    static __device__ __forceinline__ void load(const uint8_t* rec, uint32_t slot, int lane) {
        const unsigned char* g = rec + 16 * lane;
#pragma unroll
        for (int k = 0; k < R::bytes / 1024; ++k) dma16(g + 1024 * k, slot + 1024 * k);
        constexpr int rest = R::bytes % 1024 / 16;
        if constexpr (rest > 0)
            if (lane < rest) dma16(g + R::bytes / 1024 * 1024, slot + R::bytes / 1024 * 1024);
    }
};

// This wave's DMA so far is done, except the newest N instructions, and so are its LDS reads.
template <int N>
__device__ __forceinline__ void wait_ring() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(N) : "memory");
}

// The layer whose rows a workgroup reads.
__device__ __forceinline__ const lf_int4_layer& layer_of(const Int4Attention& a, bool) { return a.L; }
__device__ __forceinline__ lf_int4_layer layer_of(const Int4Shared& a, bool pre) { return pre ? a.L : a.own; }

// Shared: of prefixes that ``each`` sequences share, whose rows are all their queries (``pre``), and of the sequences' own rows, in
// one launch; the sums are always partial ones.  A prefix's records are read once from HBM, but unpacked for every 16 rows, and
// a wave's unpacking, products and waits follow one another: nothing is busy throughout.  16 sequences of up to 600 tokens behind
// a prefix of 32 768 (28 / 4 heads of 128, groups of 64, bf16, one query each, 112 rows a kv head): a call of 30 to 33 us, 22 MB
// (4 us of a copy), VALU 47 % busy, matrix cores 10 %; sequences with as many rows of their own each take 57.  32 sequences behind
// four of 4 000 to 16 300 (40 / 8 heads, groups of 128, fp16, three queries each): 77 us, VALU 61 %, matrix cores 26 %.  (Two row
// tiles a wave, which share the unpacking: 34 and 79 where this took 32 and 79; its registers leave two waves a SIMD in place of
// three.)
template <int D, int GROUP, int Dt, bool Shared>
__global__ __launch_bounds__(kWaves * kWave, D == 64 ? 4 : D == 128 ? 3 : 2) void int4_attention_kernel(typename Int4Call<Shared>::Args a) {
    using R = Int4Rec<D, GROUP>;
    using S = Ring<D, GROUP>;
    constexpr int G = R::G, CH = R::chunks, CG = CH / G, VT = D / 16, TG = VT / G;
    constexpr int NT = Dt == LF_BF16 ? 1 : Dt == LF_FP16 ? 2 : 3, NP = Dt == LF_BF16 ? 1 : 2;  // parts of q and of P'
    constexpr bool kCentred = Dt == LF_FP32;
    using Codes = std::conditional_t<kCentred, f16x8, bf16x8>;
    using QueryParts = std::conditional_t<kCentred, HalfParts<NT>, Parts<NT>>;
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    __shared__ float lds_ml[kWaves][kTile][2];
    int32_t* lds_pages = reinterpret_cast<int32_t*>(smem + S::lds);  // with pages only
    // Workgroups are dispatched x fastest, one XCD after the other: kv heads first, so that the XCDs get equal shares
    // of sequences of unlike lengths (splits first: 32 ragged contexts of 4K-64K tokens in 4 splits 545 us, against 429: 2 of 8 XCDs
    // had the last, mostly empty split) and the row tiles of a head, which read the same records, few of them; the
    // splits last, so that a long sequence's later ones follow everyone's first.
    int h = blockIdx.x % a.L.n_kv, tile = blockIdx.x / a.L.n_kv, b = blockIdx.y, part = blockIdx.z;
    bool pre = false;
    int splits = a.splits, split_tokens = a.split_tokens, part0 = a.part0;
    if constexpr (Shared) {
        pre = static_cast<int>(blockIdx.x) < a.shared_blocks;
        const int tiles = pre ? a.shared_tiles : a.own_tiles, batch = pre ? a.L.batch : a.own.batch;
        int id = static_cast<int>(blockIdx.x) - (pre ? 0 : a.shared_blocks);
        h = id % a.L.n_kv;
        id /= a.L.n_kv;
        tile = id % tiles;
        id /= tiles;
        b = id % batch;
        part = id / batch;
        if (!pre) {
            part0 = splits;
            splits = a.own_splits;
            split_tokens = a.own_split_tokens;
        }
    }
    const auto& L = layer_of(a, pre);
    const int lane = threadIdx.x % kWave, wave = in_sgpr(static_cast<int>(threadIdx.x / kWave));
    const int col = lane & 15, quad = lane >> 4;
    // rows: (head of the group, token), tokens fastest; with pages, the heads of one token
    int i, j;
    SharedRow row_at = {b, 0, 0, false};
    if constexpr (Shared)
        if (pre) row_at = shared_row(a, b, tile * kTile + col);
    if (pre) {
        i = row_at.i;
        j = row_at.j;
    } else if (!Shared && a.n_pages) {
        j = tile % a.q_len;
        i = tile / a.q_len * kTile + col;
    } else {
        const int r = tile * kTile + col;
        i = r / a.q_len;
        j = r % a.q_len;
    }
    const bool real = pre ? row_at.real : i < a.g;
    const int seq = pre ? row_at.b : b;
    // The first record is on its way before the sequence's length is: where it lies hangs on neither (with pages or
    // behind a many-row prefix it does).  A wave that finds it has none waits for the load all the same.
    const uint8_t* base = int4_block(L, b, h, 0, R::bytes);
    const uint32_t ring = lds_addr(smem) + wave * kRing * R::bytes;
    const int64_t early = static_cast<int64_t>(part) * (split_tokens / kBlock) + wave;
    const bool ahead = (Shared || (!a.n_pages && !a.prefix)) && early < L.cap_tokens / kBlock;
    if (ahead) S::load(base + early * R::bytes, ring, lane);
    const int len = int4_len(L, b);
    const int n = pre ? 0 : a.q_lens ? min(max(a.q_lens[b], 0), a.q_len) : a.q_len;
    int lim = real && j < n ? max(len - n + j + 1, 0) : 0;  // rows this query sees
    if constexpr (Shared)
        if (pre) lim = shared_limit(a, row_at, len);
    int all = real ? lim : 0x7fffffff, top = lim;                 // rows every query of the tile sees, and any
#pragma unroll
    for (int m = 1; m < 16; m <<= 1) {
        all = min(all, __shfl_xor(all, m, kWave));
        top = max(top, __shfl_xor(top, m, kWave));
    }
    all = in_sgpr(all);
    top = in_sgpr(top);

    // records of this split
    const int per_page = a.L.page_size / kBlock;
    const int own = top > 0 ? (top - 1) / a.L.page_size : 0;
    int first, last;
    if (!Shared && a.n_pages) {
        // (rounded up, splits can pass the list's end: those take nothing and read none of it)
        const int records = per_page * (a.n_pages + 1);
        first = min(part * a.split_tokens, records);
        last = min(first + a.split_tokens, records);
        if (top == 0) last = first;
        // the pages of the list that the split takes, -1 for an entry that is none in front of the own page
        const int32_t* list = a.pages + ((static_cast<int64_t>(b) * a.L.n_kv + h) * a.q_len + j) * a.n_pages;
        const int e0 = first / per_page, e1 = (last + per_page - 1) / per_page;
        for (int e = e0 + threadIdx.x; e < e1; e += kWaves * kWave) {
            int page = own;
            if (e > 0) {
                page = list[e - 1];
                if (page < 0 || page >= own || (e > 1 && page <= list[e - 2])) page = -1;
            }
            lds_pages[e - e0] = page;
        }
        __syncthreads();
    } else {
        const int blocks = (top + kBlock - 1) / kBlock, per = split_tokens / kBlock;
        first = !Shared && a.prefix ? min(prefix_records(a, len, n, tile / (kManyRows / kTile)), blocks)
                                    : static_cast<int>(min(static_cast<int64_t>(part) * per, static_cast<int64_t>(blocks)));
        last = part + 1 == splits ? blocks : static_cast<int>(min(static_cast<int64_t>(first) + per, static_cast<int64_t>(blocks)));
    }
    const int count = last > first + wave ? (last - first - wave + kWaves - 1) / kWaves : 0;  // this wave's records
    // The k-th of them, or -1 for one that is not attended (its place in the ring is filled with another).
    const auto block_of = [&](int k) {
        const int at = first + wave + k * kWaves;
        if (Shared || !a.n_pages) return at;
        const int e = at / per_page, page = in_sgpr(lds_pages[e - first / per_page]);
        const int block = page * per_page + (at - e * per_page);
        return page < 0 || block * kBlock >= top ? -1 : block;
    };
    const auto fill = [&](int k, int slot) {
        const int block = block_of(k);
        S::load(base + static_cast<int64_t>(block < 0 ? own * per_page : block) * R::bytes, ring + slot * R::bytes, lane);
    };
#pragma unroll
    for (int k = ahead ? 1 : 0; k < kRing - 1; ++k)
        if (k < count) fill(k, k);
    if (ahead && count == 0) wait_ring<0>();

    // The weights are 2^(score - ref) with ref = largest score + lift: P' <= 2^8 2^-lift scale < 2^15 for this wave's
    // records, whose largest Value scales lie below 2^(lift + 7).  In two parts P' is multiplied by ``raise``, too, up to that bound of
    // its own group's scales: its second part would be lost where they are much smaller.  The scales are read twice for it
    // (16 sequences of 32K tokens, 28 / 4 heads of 128, groups of 64: fp16 73 -> 77 us, float32 85 -> 87).
    const auto block_at = [&](int k) {  // (of an entry that is not attended, the first page's)
        const int at = first + wave + k * kWaves;
        if (Shared || !a.n_pages) return at;
        const int e = at / per_page, page = lds_pages[e - first / per_page];
        return max(page, 0) * per_page + (at - e * per_page);
    };
    const auto exponent = [](uint32_t scale) { return static_cast<int>(__float_as_uint(f16_to_f32(static_cast<uint16_t>(scale))) >> 23); };
    uint32_t most_scale = 0;
    float raise[G];
    if constexpr (NP == 1) {
        for (int k = lane; k < count; k += kWave) most_scale = max(most_scale, static_cast<uint32_t>(*int4_top(L, b, h, block_at(k))));
#pragma unroll
        for (int m = 1; m < kWave; m <<= 1) most_scale = max(most_scale, static_cast<uint32_t>(__shfl_xor(static_cast<int>(most_scale), m, kWave)));
    } else {
        constexpr int Piece = 8 * G, Take = kWave / Piece;  // 16-byte pieces of a record's pairs, and records a load takes
        uint32_t mine = 0;
        for (int k = lane / Piece; k < count; k += Take) {
            const u32x4 pair = reinterpret_cast<const u32x4*>(base + static_cast<int64_t>(block_at(k)) * R::bytes + R::vsm)[lane % Piece];
#pragma unroll
            for (int r = 0; r < 4; ++r) mine = max(mine, pair[r] & 0xffffu);  // (fp16 numbers above zero are ordered as their bits)
        }
        mine = min(mine, 0x7bffu);
#pragma unroll
        for (int m = 1; m < kWave; m <<= 1)
            if (m < 8 || m >= Piece) mine = max(mine, static_cast<uint32_t>(__shfl_xor(static_cast<int>(mine), m, kWave)));
#pragma unroll
        for (int g = 0; g < G; ++g) most_scale = max(most_scale, static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(mine), 8 * g)));
#pragma unroll
        for (int g = 0; g < G; ++g) {
            const uint32_t of = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(mine), 8 * g));
            raise[g] = __uint_as_float(static_cast<uint32_t>(127 + (of ? exponent(most_scale) - exponent(of) : 0)) << 23);
        }
    }
    const float lift = static_cast<float>(exponent(most_scale) - 126 - 7);

    QueryParts q[CH];
    float qsum[G];
    const bool flip = a.qscale < 0.f;  // a negative scale goes into the queries: scores are then compared unscaled
    const int64_t at_q = seq * a.qb + static_cast<int64_t>(h * a.g + i) * a.qh + j * a.qt + 8 * quad;
    float qscale = fabsf(a.qscale), fit = 1.f;  // ``fit``: the power of two that takes the row's largest to 2^13 .. 2^14
    if constexpr (kCentred) {
        float most = 0.f;
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            float x[8] = {};
            if (real) query8<Dt>(a, at_q + 32 * c, x);
#pragma unroll
            for (int e = 0; e < 8; ++e) most = fmaxf(most, fabsf(x[e]));
        }
        const uint32_t e = min(max(__float_as_uint(rows_max(most)) >> 23, 27u), 254u);
        fit = __uint_as_float((267u - e) << 23);
        qscale *= __uint_as_float((e - 13u) << 23);
    }
    qscale = fmaxf(qscale, 1e-37f);
#pragma unroll
    for (int g = 0; g < G; ++g) qsum[g] = 0.f;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        float x[8] = {};
        if (real) query8<Dt>(a, at_q + 32 * c, x);
        if constexpr (kCentred)
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] *= fit;
        if (flip)
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = -x[e];
        const float lo[4] = {x[0], x[1], x[2], x[3]}, hi[4] = {x[4], x[5], x[6], x[7]};
        if constexpr (kCentred) q[c] = half_parts<NT>(lo, hi);
        else q[c] = split<NT>(lo, hi);
        qsum[c / CG] += ((x[0] + x[1]) + (x[2] + x[3])) + ((x[4] + x[5]) + (x[6] + x[7]));
    }
#pragma unroll
    for (int g = 0; g < G; ++g) qsum[g] = rows_sum(qsum[g]);

    const uint32_t key_base = in_vgpr(kCentred ? kKeyBaseHalf : kKeyBase), value_base = in_vgpr(kValueBase);
    // the bias of the codes and their middle: fp16 -23.5 (Values), and -135.5 (Keys that are read as fp16)
    constexpr uint32_t kMiddle = 0xCDE0CDE0u, kKeyMiddle = 0xD83CD83Cu;
    const f16x8 middle = __builtin_bit_cast(f16x8, u32x4{kMiddle, kMiddle, kMiddle, kMiddle});
    const f16x8 key_middle = __builtin_bit_cast(f16x8, u32x4{kKeyMiddle, kKeyMiddle, kKeyMiddle, kKeyMiddle});
    f32x4 o[VT], fix[G];
    float pm[G], l = 0.f, ref = 0.f, limit = -__builtin_inff();
#pragma unroll
    for (int t = 0; t < VT; ++t) o[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int g = 0; g < G; ++g) { fix[g] = f32x4{0.f, 0.f, 0.f, 0.f}; pm[g] = 0.f; }

    // One record, of tokens from t0.  Masked: rows a query does not see get no score, and neither scale nor minimum (what
    // stands there need not be finite).  (Branches around the selects alone: two copies of the body, one without them,
    // took 40 registers more.)
    const auto attend = [&](const unsigned char* rec, bool masked, int t0) {
        const auto seen = [&](int t, int r) { return t0 + 16 * t + 4 * quad + r < lim; };
        float y[2][4];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            uint32_t kw[CH];
            __builtin_memcpy(kw, __builtin_assume_aligned(rec + (16 * t + col) * (D / 2) + CH * 4 * quad, CH == 2 ? 8 : 16), CH * 4);
            const u32x4* sm = reinterpret_cast<const u32x4*>(rec + R::ksm) + 4 * t + quad;
#pragma unroll
            for (int g = 0; g < G; ++g) {
                const u32x4 pair = sm[8 * g];
                float start = kCentred ? 0.f : -kCodeBias * qsum[g];
                // (formed anew per record: kept, the G accumulator starts take the registers of a third wave)
                if constexpr (G > 2) asm volatile("" : "+v"(start));
                f32x4 rest = {start, start, start, start}, acc = {0.f, 0.f, 0.f, 0.f};  // (float32: the lower parts by themselves)
#pragma unroll
                for (int c = g * CG; c < (g + 1) * CG; ++c) {
                    Codes codes = __builtin_bit_cast(Codes, codes8<kKeyMask>(kw[c], key_base));
                    if constexpr (kCentred) codes += key_middle;
#pragma unroll
                    for (int m = NT - 1; m >= (kCentred ? 1 : 0); --m) rest = mfma(codes, q[c].t[m], rest);
                    if constexpr (kCentred) acc = mfma(codes, q[c].t[0], acc);
                }
                if constexpr (kCentred) acc += rest;
                else acc = rest;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    // (a sum with zero where it is a product: it takes the fp16 factor as it is)
                    const float low = kCentred ? fmaf(7.5f, pair_scale(pair[r]), pair_min(pair[r])) : pair_min(pair[r]);
                    const float m = fmaf(low, qsum[g], g == 0 ? 0.f : y[t][r]);
                    y[t][r] = fmaf(pair_scale(pair[r]), acc[r], m);
                }
            }
            phase();
            if (masked)
#pragma unroll
                for (int r = 0; r < 4; ++r) y[t][r] = seen(t, r) ? y[t][r] : -__builtin_inff();
        }
        float most = fmaxf(fmaxf(fmaxf(y[0][0], y[0][1]), fmaxf(y[0][2], y[0][3])),
                           fmaxf(fmaxf(y[1][0], y[1][1]), fmaxf(y[1][2], y[1][3])));
        most *= qscale;
        if (__any(most > limit)) {
            most = rows_max(most);
            const bool moves = most > limit;
            const float scale = !moves ? 1.f : limit == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(ref - most - lift);
            if (moves) { ref = most + lift; limit = most + 8.f; }
            l *= scale;
#pragma unroll
            for (int g = 0; g < G; ++g) { pm[g] *= scale; fix[g] *= scale; }
#pragma unroll
            for (int t = 0; t < VT; ++t) o[t] *= scale;
        }
        float p[2][4];
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                p[t][r] = __builtin_amdgcn_exp2f(fmaf(y[t][r], qscale, -ref));
                l += p[t][r];
            }
        phase();
        const u32x4* vw = reinterpret_cast<const u32x4*>(rec + R::v) + lane;
        const u32x4* sm = reinterpret_cast<const u32x4*>(rec + R::vsm) + quad;
#pragma unroll
        for (int g = 0; g < G; ++g) {
            u32x4 pair[2] = {sm[8 * g], sm[8 * g + 4]};
            if (masked)
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int r = 0; r < 4; ++r) pair[t][r] = seen(t, r) ? pair[t][r] : 0u;
            float x[2][4];
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    x[t][r] = fmaf(p[t][r], pair_scale(pair[t][r]), 0.f);
                    pm[g] = fmaf(p[t][r], pair_min(pair[t][r]), pm[g]);
                    pm[g] = fmaf(7.5f, x[t][r], pm[g]);
                }
            if constexpr (NP > 1)
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int r = 0; r < 4; ++r) x[t][r] *= raise[g];
            const HalfParts<NP> w = half_parts<NP>(x[0], x[1]);
            if constexpr (!kCentred)
#pragma unroll
                for (int m = NP - 1; m >= 0; --m) fix[g] = mfma(middle, w.t[m], fix[g]);
#pragma unroll
            for (int t = g * TG; t < (g + 1) * TG; ++t) {
                f16x8 codes = __builtin_bit_cast(f16x8, codes8<kValueMask>(vw[(t >> 2) * kWave][t & 3], value_base));
                if constexpr (kCentred) codes += middle;
#pragma unroll
                for (int m = NP - 1; m >= 0; --m) o[t] = mfma(codes, w.t[m], o[t]);
            }
            phase();
        }
    };

    int slot = 0;
    for (int k = 0; k < count; ++k) {
        if (k + kRing - 1 <= count) wait_ring<(kRing - 2) * S::loads>();
        else wait_ring<0>();
        if (k + kRing - 1 < count) fill(k + kRing - 1, slot == 0 ? kRing - 1 : slot - 1);
        const unsigned char* rec = smem + (wave * kRing + slot) * R::bytes;
        slot = slot + 1 == kRing ? 0 : slot + 1;
        const int block = block_of(k);
        if (block < 0) continue;

        attend(rec, block * kBlock + kBlock > all, block * kBlock);
    }

    // the waves' sums at one reference point
    l = rows_sum(l);
    const float m_wave = l == 0.f ? -__builtin_inff() : ref;  // (a sum of NaN has a place among the others)
    if (quad == 0) { lds_ml[wave][col][0] = m_wave; lds_ml[wave][col][1] = l; }
#pragma unroll
    for (int g = 0; g < G; ++g) pm[g] = rows_sum(pm[g]);
    __syncthreads();  // every wave is done with its ring, too
    float* lds_o = reinterpret_cast<float*>(smem);
    float m_all = lds_ml[0][col][0];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) m_all = fmaxf(m_all, lds_ml[w][col][0]);
    const float mine = m_wave == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(m_wave - m_all);
#pragma unroll
    for (int t = 0; t < VT; ++t) {
        o[t] += fix[t / TG];
        if constexpr (NP > 1) o[t] *= __uint_as_float((254u << 23) - __float_as_uint(raise[t / TG]));  // (its reciprocal)
        o[t] = (o[t] + pm[t / TG]) * mine;
        if (wave > 0) *reinterpret_cast<f32x4*>(lds_o + ((wave - 1) * kTile + col) * S::pad + 16 * t + 4 * quad) = o[t];
    }
    __syncthreads();
    if (wave > 0) return;
    float l_all = l * mine;
#pragma unroll
    for (int w = 1; w < kWaves; ++w) {
        const float m = lds_ml[w][col][0];
        l_all += m == -__builtin_inff() ? 0.f : lds_ml[w][col][1] * __builtin_amdgcn_exp2f(m - m_all);
#pragma unroll
        for (int t = 0; t < VT; ++t) o[t] += *reinterpret_cast<const f32x4*>(lds_o + ((w - 1) * kTile + col) * S::pad + 16 * t + 4 * quad);
    }
    if (!real) return;
    const int64_t row = (static_cast<int64_t>(seq) * a.n_q + h * a.g + i) * a.q_len + j;
    if (!Shared && a.parts == 1) {
        const float inv = l_all == 0.f ? 0.f : 1.f / l_all;  // (no row seen: zeros)
#pragma unroll
        for (int t = 0; t < VT; ++t) o[t] *= inv;
        each_run<D, GROUP>(o, quad, [&](int c, const float (&x)[4]) { store_row<Dt>(a.out, row * D + c, x); });
        return;
    }
    float* dst = a.part_o + (row * a.parts + part0 + part) * D;
    each_run<D, GROUP>(o, quad, [&](int c, const float (&x)[4]) { store_row<LF_FP32>(dst, c, x); });
    if (quad == 0) {
        float* ml = a.part_ml + (row * a.parts + part0 + part) * 2;
        ml[0] = m_all;
        ml[1] = l_all;
    }
}

// The splits' sums at their largest reference point: a workgroup per output row, whose waves take the splits in
// turn (sixteen of every 64, all loads on their way at once) and add up through LDS.  3 to 5 us, a launch and two dependent
// loads; of 512 queries (14 336 rows, 51 MB of sums) 12.  One wave up to 16 splits, four from there on: attention and
// merge of one sequence of 2K tokens, 16 splits 9.1 us with one and 9.3 with four, 64 splits 11.5 and 9.5.
template <int D>
__global__ __launch_bounds__(256) void int4_merge_kernel(Int4Attention a, int dtype) {
    constexpr int C = D / kWave, kTake = 16;
    __shared__ float lds[4][D];
    const int64_t row = blockIdx.x;
    const int lane = threadIdx.x % kWave, wave = in_sgpr(static_cast<int>(threadIdx.x / kWave)), waves = blockDim.x / kWave;
    const float* ml = a.part_ml + row * a.parts * 2;
    const float* sums = a.part_o + row * a.parts * D + lane * C;
    float x[kTake][C];
    const auto load = [&](int s) {
#pragma unroll
        for (int k = 0; k < kTake; ++k)
#pragma unroll
            for (int c = 0; c < C; ++c) x[k][c] = s + k < a.parts ? sums[(s + k) * D + c] : 0.f;
    };
    load(wave * kTake);  // (on their way while the reference points are compared)
    float m = -__builtin_inff();
    for (int s = lane; s < a.parts; s += kWave) m = fmaxf(m, ml[2 * s]);
    m = wave_max(m);
    float o[C] = {}, l = 0.f;
    for (int s0 = 0; s0 < a.parts; s0 += kWave) {
        float w = 0.f;
        if (s0 + lane < a.parts) {
            const float ms = ml[2 * (s0 + lane)];
            w = ms == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(ms - m);
            l = fmaf(w, ml[2 * (s0 + lane) + 1], l);
        }
        for (int k0 = wave * kTake; k0 < kWave && s0 + k0 < a.parts; k0 += waves * kTake) {
            if (s0 > 0 || k0 > wave * kTake) load(s0 + k0);
#pragma unroll
            for (int k = 0; k < kTake; ++k) {
                const float wk = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, w), k0 + k));
#pragma unroll
                for (int c = 0; c < C; ++c) o[c] = fmaf(wk, x[k][c], o[c]);
            }
        }
    }
    l = wave_sum(l);
    if (waves > 1) {
#pragma unroll
        for (int c = 0; c < C; ++c) lds[wave][lane * C + c] = o[c];
        __syncthreads();
        if (wave > 0) return;
        for (int v = 1; v < waves; ++v)
#pragma unroll
            for (int c = 0; c < C; ++c) o[c] += lds[v][lane * C + c];
    }
#pragma unroll
    for (int c = 0; c < C; ++c) store_from_f32(a.out, row * D + lane * C + c, dtype, l == 0.f ? 0.f : o[c] / l);
}

template <int D>
void launch_merge(const Int4Attention& a, int batch, int dtype, hipStream_t stream) {
    const uint32_t rows = static_cast<uint32_t>(batch) * a.n_q * a.q_len;
    hipLaunchKernelGGL((int4_merge_kernel<D>), dim3(rows), dim3(a.parts > 16 ? 256 : 64), 0, stream, a, dtype);
}

template <int D, int GROUP, int Dt>
int launch_typed(const Int4Attention& a, int tiles, hipStream_t stream) {
    const auto fn = int4_attention_kernel<D, GROUP, Dt, false>;
    int lds = Ring<D, GROUP>::lds;
    if (a.n_pages) lds += 4 * (a.split_tokens / (a.L.page_size / kBlock) + 2);  // the split's entries of the page list
    int st = allow_dynamic_lds(reinterpret_cast<const void*>(fn), lds);
    if (st == LF_OK && a.prefix) st = launch_int4_prefix(a, stream);
    if (st != LF_OK) return st;
    Int4Attention rest = a;  // what a many-row launch leaves
    rest.part0 += a.prefix;
    hipLaunchKernelGGL(fn, dim3(a.L.n_kv * tiles, a.L.batch, a.splits), dim3(kWaves * kWave), lds, stream, rest);
    if (a.parts > 1) launch_merge<D>(a, a.L.batch, Dt, stream);
    const hipError_t err = hipGetLastError();
    return err == hipSuccess ? LF_OK : static_cast<int>(err);
}

// The rows of shared prefixes, 16 at a time, and with own_splits the sequences' own and the merge.
template <int D, int GROUP, int Dt>
int launch_shared_typed(Int4Shared a, hipStream_t stream) {
    const auto fn = int4_attention_kernel<D, GROUP, Dt, true>;
    const int lds = Ring<D, GROUP>::lds;
    const int st = allow_dynamic_lds(reinterpret_cast<const void*>(fn), lds);
    if (st != LF_OK) return st;
    a.shared_tiles = (a.g * a.q_len * a.each + kTile - 1) / kTile;
    a.own_tiles = (a.g * a.q_len + kTile - 1) / kTile;
    a.shared_blocks = a.L.n_kv * a.shared_tiles * a.L.batch * a.splits;
    const int own_blocks = a.own.n_kv * a.own_tiles * a.own.batch * a.own_splits;
    hipLaunchKernelGGL(fn, dim3(a.shared_blocks + own_blocks), dim3(kWaves * kWave), lds, stream, a);
    if (a.own_splits) launch_merge<D>(a, a.own.batch, Dt, stream);
    const hipError_t err = hipGetLastError();
    return err == hipSuccess ? LF_OK : static_cast<int>(err);
}

Int4Attention attention_of(const lf_int4_layer& L, const lf_int4_args& A, int more_parts) {
    Int4Attention a{};
    a.L = L;
    a.q = A.query;
    a.qb = A.q_strides[0]; a.qh = A.q_strides[1]; a.qt = A.q_strides[2];
    const int esize = A.dtype == LF_FP32 ? 4 : 2;
    a.vec = reinterpret_cast<uintptr_t>(A.query) % 16 == 0;
    for (int i = 0; i < 3; ++i) a.vec = a.vec && A.q_strides[i] * esize % 16 == 0;
    a.q_lens = A.q_lens;
    a.out = A.out;
    a.n_q = A.n_q; a.g = A.n_q / L.n_kv; a.q_len = A.q_len;
    a.qscale = A.scaling * kLog2e;
    a.pages = A.pages; a.n_pages = A.n_pages;
    a.splits = A.splits;
    a.prefix = A.prefix_splits;
    a.parts = a.splits + a.prefix + more_parts;
    a.part0 = more_parts;
    a.split_tokens = A.split_tokens;
    const int64_t rows = static_cast<int64_t>(L.batch) * A.n_q * A.q_len;
    a.part_o = static_cast<float*>(A.workspace);
    a.part_ml = a.part_o + rows * a.parts * L.head_dim;
    return a;
}

// The attention of ``a``'s rows over their own cache, and the merge of all parts.
int launch_own(Int4Attention a, const lf_int4_args& A, hipStream_t stream) {
    const lf_int4_layer& L = a.L;
    int tiles = (a.g * A.q_len + kTile - 1) / kTile;
    if (A.n_pages) {
        tiles = (a.g + kTile - 1) / kTile * A.q_len;
        const int records = L.page_size / kBlock * (A.n_pages + 1);
        a.split_tokens = (records + A.splits - 1) / A.splits;
    }
    return int4_dispatch(L, [&](auto shape) {
        constexpr int D = decltype(shape)::d, GROUP = decltype(shape)::group;
        return A.dtype == LF_BF16 ? launch_typed<D, GROUP, LF_BF16>(a, tiles, stream)
               : A.dtype == LF_FP16 ? launch_typed<D, GROUP, LF_FP16>(a, tiles, stream)
                                    : launch_typed<D, GROUP, LF_FP32>(a, tiles, stream);
    });
}

}  // namespace

int64_t int4_part_bytes(const lf_int4_layer& L, int n_q, int q_len, int splits) {
    return splits <= 1 ? 0 : static_cast<int64_t>(L.batch) * n_q * q_len * splits * (L.head_dim + 2) * 4;
}

int launch_int4_attention(const lf_int4_layer& L, const lf_int4_args& A, hipStream_t stream) {
    return launch_own(attention_of(L, A, 0), A, stream);
}

// The prefix's parts come first, then the sequences' own.
int launch_int4_shared(const lf_int4_layer& L, const lf_int4_layer& P, const lf_int4_args& A, int splits, int split_tokens, bool many_rows,
                       hipStream_t stream) {
    const Int4Attention own = attention_of(L, A, splits);
    Int4Shared a{};
    static_cast<Int4Attention&>(a) = own;
    a.L = P;
    a.part0 = a.prefix = 0;
    a.splits = splits;
    a.split_tokens = split_tokens;
    a.each = L.batch / P.batch;
    a.own = L;
    // the sequences' own rows in the same launch, where both are the general kernel's
    const bool one = !many_rows && A.prefix_splits == 0;
    a.own_splits = one ? A.splits : 0;
    a.own_split_tokens = A.split_tokens;
    const int st = many_rows ? launch_int4_shared_rows(a, stream) : int4_dispatch(P, [&](auto shape) {
        constexpr int D = decltype(shape)::d, GROUP = decltype(shape)::group;
        return A.dtype == LF_BF16 ? launch_shared_typed<D, GROUP, LF_BF16>(a, stream)
               : A.dtype == LF_FP16 ? launch_shared_typed<D, GROUP, LF_FP16>(a, stream)
                                    : launch_shared_typed<D, GROUP, LF_FP32>(a, stream);
    });
    return st == LF_OK && !one ? launch_own(own, A, stream) : st;
}

}  // namespace lf
