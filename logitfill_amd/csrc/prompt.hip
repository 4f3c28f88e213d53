// Causal attention of whole prompts on the matrix cores: sequences of any lengths, grouped heads, queries that are the last of
// their sequence's Keys.
//
// A workgroup takes a tile of query rows of one kv head -- row r is token r / g of the sequence and head r % g of the group, so
// that a tile's rows see nearly the same Keys -- and walks the Keys in tiles.  Per tile and wave, for 32 rows, on
// v_mfma_f32_32x32x16:
//     S^T = K . Q^T,   p = 2^(c S - ref),   O^T += V^T . P^T,   l += sum p.
// A score's lane holds eight of the sixteen Keys that its lane of the second product takes, so P goes from one to the other
// in registers; the Value operand is read with its Keys in that order by LDS transpose reads.  The reference point of a row
// moves only when a score passes it by 2^8.
//
// Keys and Values of one tile lie in LDS: Values come by DMA while the Keys are multiplied, the next Keys while the Values
// are.  32 KB of 64 Keys (head_dim 128) and 168 registers let a compute unit hold three workgroups, whose products and
// exponentials fill each other's waits.
//
// Scores and sums are fp32; P is rounded to the rows' type (bf16: 2^-8 of a weight at most, averaged over the Keys, beside the
// output's own; fp16: formed as up to 2^15, so that it keeps weights down to 2^-31 of their row's largest).  Its lower part would
// be a third product beside two, in a kernel that the matrix cores bound at long prompts.  float32 rows: see prompt_split_kernel,
// or, of heads of 256 and single waves, multiplied as such (32x32x2).  Weights reach 2^8 (fp16: 2^15) before they are divided by
// their sum: Values past 2^119 over the tokens (bf16, fp32) may overflow the sums.
//
// Measured: one prompt of 16 384 tokens, 40 / 8 heads of 128, bf16: 2.36 to 2.5 ms, 1 100 to 1 165 TFLOP/s of the products that
// are not masked (an 8 192^3 bf16 product of the library: 1 220).  Matrix cores 65 % busy, VALU 51 %, LDS 49 %, no bank
// conflicts, 97 % of the Keys' and Values' reads from L2; the clock falls to 2.0 GHz under that load.  Eight prompts of 300
// to 8 190 tokens, 28 / 4 heads: 1.35 to 1.4 ms (1 090); 512 tokens behind 16 384: 138 us, 8 of them the merge; 1 061 tokens
// alone 26.6; float32, two of 1 500, 8 heads of 256: 181 (8.4 a Key tile, 6.8 of them float32 products).  16-bit heads of 256, 8 192
// tokens, 16 / 8 heads: 530 to 590 (1 010).  Single tokens, 28 / 4 heads of 128: sixteen behind 32 768 each 201 us, 5.3 TB/s (float32
// 669, 3.2), one 34, four behind 1 000 15.  At head_dim 64 a wave's exponentials and products follow
// one another, and four waves a SIMD do not fill all of it.  Sixteen of 1 to 1 500 tokens, 14 / 2 heads, fp16: 43 us, 0.69 a Key
// tile and compute unit, 0.43 of them VALU work (VALU 46 % busy, matrix cores 21 %); 8 192 tokens, 16 / 8 heads, bf16: 169, 815
// TFLOP/s (61 %, 42 %).
// Not faster at 16 384 tokens: Keys buffered twice (two workgroups a CU; the same long, 8 % less of 1 061 tokens alone, where two groups
// now do more); tiles of 32 Keys (2.5 against 2.45 ms); 64 rows a wave (its sums spill: 9.1); operands read a product
// ahead; waves' priorities (2.53); sums of the rounded weights by dot products (the same; at head_dim 64 46.5 us for 45, the error
// 2.3e-4 for 2.6e-4).
#include "lf_common.hpp"
#include "decode_common.hpp"

#include <type_traits>

namespace lf {
namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

struct Prompt {
    const void *q, *k, *v;
    void* out;
    int64_t qs[3], ks[3], vs[3], os[3];  // elements per batch row, head and token
    const lf_prompt_item* items;
    int n_q, n_kv, g;
    float qscale;   // scaling * log2(e)
    int far;        // a tile's rows span more than 32-bit offsets reach
    float* part_o;  // [slots][n_kv][rows of a tile][D]
    float* part_ml; // [slots][n_kv][rows of a tile][2]
};

template <int Dt> struct Element;
template <> struct Element<LF_BF16> {
    using x8 = bf16x8;
    static constexpr uint32_t bits = 0x7fff7fffu, least = 0x00800080u;  // all but the signs; infinity's distance from the next sign
    static constexpr float headroom = 0.f;
    static __device__ __forceinline__ f32x16 mfma(x8 a, x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
    static __device__ __forceinline__ uint32_t pack(float a, float b) {
        typedef float f32x2 __attribute__((ext_vector_type(2)));
        typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
        return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{a, b}, bf16x2));
    }
};
template <> struct Element<LF_FP16> {
    using x8 = f16x8;
    static constexpr uint32_t bits = 0x7fff7fffu, least = 0x04000400u;
    static constexpr float headroom = 7.f;
    static __device__ __forceinline__ f32x16 mfma(x8 a, x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
    static __device__ __forceinline__ uint32_t pack(float a, float b) {
        typedef float f32x2 __attribute__((ext_vector_type(2)));
        typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
        return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{a, b}, f16x2));
    }
};

template <> struct Element<LF_FP32> {
    using x8 = f32x4;  // (four channels or Keys, one a product: v_mfma_f32_32x32x2)
    static constexpr uint32_t bits = 0x7fffffffu, least = 0x00800000u;
    static constexpr float headroom = 0.f;
};

// A tile of Keys or Values in LDS: rows in 16-byte pieces, whose places are exchanged by row so that the products'
// operand reads take all banks.
template <int D, int Dt>
struct Tile {
    static constexpr int esize = Dt == LF_FP32 ? 4 : 2;
    static constexpr int keys = D == 256 || Dt == LF_FP32 ? 32 : 64;
    static constexpr int row = esize * D, bytes = keys * row, pieces = row / 16;
    static constexpr int rows_per_load = 1024 / row, loads = bytes / 1024;
    static constexpr int lds = 2 * bytes;  // Keys, then Values
    static __device__ __forceinline__ int key_swap(int r) { return r & (pieces < 16 ? pieces - 1 : 15); }
    static __device__ __forceinline__ int value_swap(int r) { return Dt == LF_FP32 ? (r & 4) << 1 : D == 64 ? (r & 2) << 1 : (r & 3) << 2; }
};

// Max and sum over the two lanes of a query.
__device__ __forceinline__ float halves_max(float x) {
    float a, b;
    swap_rows<true>(x, a, b);
    return fmaxf(a, b);
}

__device__ __forceinline__ u32x2 read_tr(uint32_t at) {
    typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
    return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<lds_s16x4*>(static_cast<uintptr_t>(at))));
}
// LDS-DMA (dma16 without its streaming hint: other workgroups read the same Keys): each lane's 16 bytes, at an offset from a
// uniform base or at an address of its own, land at lds + 16 * lane.  (A base that a vector instruction wrote, as a
// readfirstlane, is read five wait states later at the earliest, and M0 one after its write.)
__device__ __forceinline__ void dma16_at(const unsigned char* base, uint32_t offset, uint32_t lds) {
    asm volatile("s_nop 4\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(offset), "s"(in_sgpr(base)), "{m0}"(lds) : "memory");
}
__device__ __forceinline__ void dma16_far(const unsigned char* g, uint32_t lds) {
    asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(g), "{m0}"(lds) : "memory");
}

__device__ __forceinline__ uint32_t read4(uint32_t at) {
    typedef __attribute__((address_space(3))) const uint32_t lds_u32;
    return *reinterpret_cast<lds_u32*>(static_cast<uintptr_t>(at));
}
__device__ __forceinline__ u32x4 read16(uint32_t at) {
    typedef __attribute__((address_space(3))) const u32x4 lds_u32x4;
    return *reinterpret_cast<lds_u32x4*>(static_cast<uintptr_t>(at));
}

__device__ __forceinline__ lf_prompt_item load_item(const Prompt& a) {
    lf_prompt_item item = a.items[blockIdx.x / a.n_kv];
    item.q_row = in_sgpr(item.q_row); item.q_start = in_sgpr(item.q_start); item.n_q = in_sgpr(item.n_q);
    item.k_row = in_sgpr(item.k_row); item.k_start = in_sgpr(item.k_start); item.n_k = in_sgpr(item.n_k);
    item.tile = in_sgpr(item.tile); item.slot = in_sgpr(item.slot);
    item.begin = in_sgpr(item.begin); item.end = in_sgpr(item.end);
    return item;
}

// How a workgroup's NW waves bring tiles of an item's Keys and Values into LDS: a load instruction takes rows_per_load rows.
// Of a whole tile a lane's offset from the tile's start is the same in every tile, but for the pieces' exchange, which is
// linear in the row's bits.
template <int D, int Dt, int NW>
struct Loader {
    using T = Tile<D, Dt>;
    static constexpr int kStep = NW * T::rows_per_load;
    struct Side {
        const unsigned char* base;
        int64_t stride;        // bytes from row to row
        uint32_t row, piece;   // this lane's offsets
        int swapped[2];        // (row0, its piece) for rows of their own
        bool value;
    };
    Side keys, values;
    int reach, wave;
    bool far;

    __device__ __forceinline__ Loader(const Prompt& a, const lf_prompt_item& item, int h, int wave_, int lane, int reach_) {
        reach = reach_;
        wave = wave_;
        far = a.far;
        const int row0 = wave * T::rows_per_load + lane / T::pieces, piece0 = lane % T::pieces;
        keys = side(a.k, a.ks, item, h, row0, piece0, false);
        values = side(a.v, a.vs, item, h, row0, piece0, true);
    }
    static __device__ __forceinline__ Side side(const void* p, const int64_t (&s)[3], const lf_prompt_item& item, int h, int row0, int piece0, bool value) {
        const int64_t at = item.k_row * s[0] + h * s[1] + static_cast<int64_t>(item.k_start) * s[2];
        const int64_t stride = s[2] * T::esize;
        return {in_sgpr(static_cast<const unsigned char*>(p) + at * T::esize), stride, static_cast<uint32_t>(row0 * stride),
                static_cast<uint32_t>(16 * (piece0 ^ (value ? T::value_swap(row0) : T::key_swap(row0)))), {row0, piece0}, value};
    }
    static __device__ __forceinline__ int swap(bool value, int r) { return value ? T::value_swap(r) : T::key_swap(r); }
    // Tile t to LDS address ``at``.
    __device__ __forceinline__ void fill(const Side& s, int t, uint32_t at) const {
        const uint32_t to = at + wave * 1024;
        if (!far && t * T::keys + T::keys <= reach) {
            const unsigned char* from = s.base + static_cast<int64_t>(t) * T::keys * s.stride;
#pragma unroll
            for (int n = 0; n < T::loads / NW; ++n)
                dma16_at(from + static_cast<int64_t>(n * kStep) * s.stride, s.row + (s.piece ^ (16 * swap(s.value, n * kStep))), to + n * NW * 1024);
            return;
        }
        // (in place of Keys past the last one that is seen, that one; the empty statement keeps what this rare way needs out of the
        // registers of the others)
        int row0 = s.swapped[0], piece0 = s.swapped[1];
        asm volatile("" : "+v"(row0), "+v"(piece0));
#pragma unroll
        for (int n = 0; n < T::loads / NW; ++n) {
            const int r = row0 + n * kStep;
            const int64_t row = min(t * T::keys + r, reach - 1);
            dma16_far(s.base + row * s.stride + 16 * (piece0 ^ swap(s.value, r)), to + n * NW * 1024);
        }
    }
};

// LDS reads stay behind this point: all hoisted to a tile's start they take more registers than there are.
__device__ __forceinline__ void phase() { asm volatile("" ::: "memory"); }

// A row's attention to Keys first .. end - 1 by itself, in the pair of lanes that holds it (half ``hi`` of its channels each): to
// ``out``, or as a split's sums where that is null.
template <int D, int Dt>
__device__ __attribute__((noinline)) void one_row(const unsigned char* q, const unsigned char* k, const unsigned char* v, int64_t kstride,
                                                  int64_t vstride, int first, int end, int hi, float qscale, unsigned char* out, float* part_o,
                                                  float* part_ml) {
    constexpr int H = D / 2;
    float o[H], m = -__builtin_inff(), l = 0.f;
#pragma unroll
    for (int c = 0; c < H; ++c) o[c] = 0.f;
#pragma unroll 1
    for (int key = first; key < end; ++key) {
        float s = 0.f;
#pragma unroll 1
        for (int c = 0; c < D; c += 8) {
            float x[8], y[8];
            load8_as_f32(q, c, Dt, x);
            load8_as_f32(k + key * kstride, c, Dt, y);
#pragma unroll
            for (int e = 0; e < 8; ++e) s = fmaf(x[e], y[e], s);
        }
        s *= qscale;
        if (s > m) {
            const float down = __builtin_amdgcn_exp2f(m - s);
            m = s;
            l *= down;
#pragma unroll
            for (int c = 0; c < H; ++c) o[c] *= down;
        }
        // (a weight of zero counts, too: times a Value that is not finite it is NaN, as in the products)
        const float w = s == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(s - (m == -__builtin_inff() ? 0.f : m));
        l += w;
#pragma unroll
        for (int c = 0; c < H; c += 8) {
            float y[8];
            load8_as_f32(v + key * vstride, hi * H + c, Dt, y);
#pragma unroll
            for (int e = 0; e < 8; ++e) o[c + e] = fmaf(w, y[e], o[c + e]);
        }
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
    for (int c = 0; c < H; ++c) {
        if (out) store_from_f32(out, hi * H + c, Dt, o[c] * inv);
        else part_o[hi * H + c] = o[c];
    }
    if (!out && hi == 0) {
        part_ml[0] = l == 0.f ? -__builtin_inff() : m;
        part_ml[1] = l;
    }
}

// The end of an item for the pair of lanes (col, hi) that holds a row: its output, or a split's sums; rows of a tile with Values
// that are not finite are formed anew over Keys begin .. end - 1.
template <int D, int Dt, int NW>
__device__ __forceinline__ void finish(const Prompt& a, const lf_prompt_item& item, int h, int wave, int col, int hi, int i, int j, bool real,
                                       int lim, int begin, int end, bool odd, float l, float ref, const f32x16 (&o)[D / 32]) {
    using E = Element<Dt>;
    constexpr bool kWide = Dt == LF_FP32;
    constexpr int ES = kWide ? 4 : 2, CB = D / 32, kRows = 32 * NW;
    if (odd) {
        if (!real) return;
        const unsigned char* src = static_cast<const unsigned char*>(a.q) +
            ES * (item.q_row * a.qs[0] + static_cast<int64_t>(h * a.g + i) * a.qs[1] + static_cast<int64_t>(item.q_start + j) * a.qs[2]);
        const int64_t to = item.q_row * a.os[0] + static_cast<int64_t>(h * a.g + i) * a.os[1] + static_cast<int64_t>(item.q_start + j) * a.os[2];
        const int64_t at = (static_cast<int64_t>(item.slot) * a.n_kv + h) * kRows + wave * 32 + col;
        const int64_t k = item.k_row * a.ks[0] + h * a.ks[1] + static_cast<int64_t>(item.k_start) * a.ks[2];
        const int64_t v = item.k_row * a.vs[0] + h * a.vs[1] + static_cast<int64_t>(item.k_start) * a.vs[2];
        const unsigned char *kbase = static_cast<const unsigned char*>(a.k) + ES * k, *vbase = static_cast<const unsigned char*>(a.v) + ES * v;
        one_row<D, Dt>(src, kbase, vbase, ES * a.ks[2], ES * a.vs[2], begin, min(end, lim), hi, a.qscale,
                       item.slot < 0 ? static_cast<unsigned char*>(a.out) + ES * to : nullptr, a.part_o + at * D, a.part_ml + 2 * at);
        return;
    }
    if (!real) return;
    // channels 32 c + 8 n + 4 hi .. + 3
    if (item.slot < 0) {
        const float inv = l == 0.f ? 0.f : 1.f / l;  // (no Key seen: zeros)
        const int64_t to = item.q_row * a.os[0] + static_cast<int64_t>(h * a.g + i) * a.os[1] + static_cast<int64_t>(item.q_start + j) * a.os[2] + 4 * hi;
#pragma unroll
        for (int c = 0; c < CB; ++c)
#pragma unroll
            for (int n = 0; n < 4; ++n) {
                const f32x4 x = {o[c][4 * n] * inv, o[c][4 * n + 1] * inv, o[c][4 * n + 2] * inv, o[c][4 * n + 3] * inv};
                if constexpr (kWide) *reinterpret_cast<f32x4*>(static_cast<float*>(a.out) + to + 32 * c + 8 * n) = x;
                else *reinterpret_cast<u32x2*>(static_cast<uint16_t*>(a.out) + to + 32 * c + 8 * n) = u32x2{E::pack(x[0], x[1]), E::pack(x[2], x[3])};
            }
        return;
    }
    const int64_t at = (static_cast<int64_t>(item.slot) * a.n_kv + h) * kRows + wave * 32 + col;
    float* dst = a.part_o + at * D + 4 * hi;
#pragma unroll
    for (int c = 0; c < CB; ++c)
#pragma unroll
        for (int n = 0; n < 4; ++n)
            *reinterpret_cast<f32x4*>(dst + 32 * c + 8 * n) = f32x4{o[c][4 * n], o[c][4 * n + 1], o[c][4 * n + 2], o[c][4 * n + 3]};
    if (hi == 0) {
        a.part_ml[2 * at] = l == 0.f ? -__builtin_inff() : ref;
        a.part_ml[2 * at + 1] = l;
    }
}

// Groups of NW waves of 32 rows each, that take an item's Key tiles in turn and are joined through LDS at its end: where there is a
// workgroup a compute unit at most, two groups do what two workgroups would, without partial sums and the merge's launch (1 061
// tokens, 28 / 4 heads of 128: 26.6 us; one group 32, the Keys divided in two or three and merged 31 and 30).
template <int D, int Dt>
constexpr int kPerSimd = Dt == LF_FP32 ? (D == 64 ? 3 : D == 128 ? 2 : 1) : (D == 64 ? 4 : D == 128 ? 3 : 2);  // waves, by their registers

template <int D, int Dt, int NW, int Groups>
struct Shape {
    static constexpr int sums = NW * kWave * D * 2;  // bytes of a group's sums: D / 2 floats a lane
    static constexpr int lds = Groups == 1 ? Tile<D, Dt>::lds : (2 * Tile<D, Dt>::lds > sums ? 2 * Tile<D, Dt>::lds : sums) + NW * kWave * 16;
};

template <int D, int Dt, int NW, int Groups>
__global__ __launch_bounds__(Groups * NW * kWave, (Groups > 1 ? 2 : kPerSimd<D, Dt>)) void prompt_kernel(Prompt a) {
    using T = Tile<D, Dt>;
    using E = Element<Dt>;
    using x8 = typename E::x8;
    constexpr bool kWide = Dt == LF_FP32;
    constexpr int ES = T::esize, KT = T::keys, KB = KT / 32, SQ = D * ES / 32, CB = D / 32, KK = kWide ? KT / 8 : KT / 16;
    constexpr int kRows = 32 * NW;
    extern __shared__ __attribute__((aligned(1024))) unsigned char smem[];
    const int h = blockIdx.x % a.n_kv;
    const lf_prompt_item item = load_item(a);
    const int lane = threadIdx.x % kWave, turn = Groups == 1 ? 0 : in_sgpr(static_cast<int>(threadIdx.x / (NW * kWave)));
    const int wave = in_sgpr(static_cast<int>(threadIdx.x / kWave)) - turn * NW;
    const int col = lane & 31, hi = lane >> 5;
    const uint32_t lds = lds_addr(smem) + turn * T::lds;

    const int row = item.tile * kRows + wave * 32 + col;
    const int j = row / a.g, i = row - j * a.g;
    const bool real = j < item.n_q;
    const int lim = real ? max(item.n_k - item.n_q + j + 1, 0) : 0;  // Keys this row sees
    int all = real ? lim : 0x7fffffff;                               // that every row of the wave sees
#pragma unroll
    for (int m = 1; m < 32; m <<= 1) all = min(all, __shfl_xor(all, m, kWave));
    all = in_sgpr(all);
    // the workgroup's last row that is real sees the most
    const int last_token = min((item.tile * kRows + kRows - 1) / a.g, item.n_q - 1);
    const int reach = max(item.n_k - item.n_q + last_token + 1, 0);
    const int first = item.begin, last = min(item.end, (reach + KT - 1) / KT);

    const Loader<D, Dt, NW> loader(a, item, h, wave, lane, reach);
    if (first + turn < last) loader.fill(loader.keys, first + turn, lds);

    x8 q[SQ];
    {
        // a lane's channels: of every 16 (float32: 8), the half hi
        const unsigned char* src = static_cast<const unsigned char*>(a.q) + 16 * hi +
            ES * (item.q_row * a.qs[0] + static_cast<int64_t>(h * a.g + i) * a.qs[1] + static_cast<int64_t>(item.q_start + j) * a.qs[2]);
#pragma unroll
        for (int s = 0; s < SQ; ++s) {
            u32x4 w = {0, 0, 0, 0};
            if (real && reach > 0) w = *reinterpret_cast<const u32x4*>(src + 32 * s);
            q[s] = __builtin_bit_cast(x8, w);
        }
    }
    // A negative scale would make the largest score the smallest: it goes into the queries' signs.
    if (a.qscale < 0.f)
#pragma unroll
        for (int s = 0; s < SQ; ++s) q[s] = -q[s];
    const float scale = fmaxf(fabsf(a.qscale), 1e-37f);  // (above zero: -inf stays -inf)

    f32x16 o[CB];
#pragma unroll
    for (int c = 0; c < CB; ++c) o[c] = f32x16{};
    float l = 0.f, ref = 0.f, limit = -__builtin_inff();
    bool odd = false;

    // operand addresses inside a tile
    // (the rows are whole multiples of what is exchanged: further pieces are an exclusive or away, further rows a constant)
    const uint32_t key_at = col * T::row + 16 * (hi ^ T::key_swap(col));
    const int group = lane >> 4, in16 = lane & 15;  // 16 lanes transpose four rows of sixteen channels
    const int vrow = 4 * (group >> 1) + (in16 >> 2), vcol = 16 * (group & 1) + 4 * (in16 & 3);
    const uint32_t value_at = T::bytes + (kWide ? 4 * hi * T::row + 16 * ((col / 4) ^ T::value_swap(4 * hi)) + 4 * (col & 3)
                                                : vrow * T::row + 16 * ((vcol / 8) ^ T::value_swap(vrow)) + 2 * (vcol & 7));

    // Tiles that every row of the wave sees whole come first (a branch in one body became selects in every tile).
    const auto tile = [&](auto masked_tile, int t) __attribute__((always_inline)) {
        constexpr bool masked = decltype(masked_tile)::value;
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __syncthreads();  // the tile's Keys are there, and nobody reads the last one's Values any more
        loader.fill(loader.values, t, lds + T::bytes);
        phase();
        const int k0 = t * KT;
        const uint32_t keys = lds + key_at, values = lds + value_at;
        f32x16 s[KB];
#pragma unroll
        for (int n = 0; n < SQ; ++n) {
            if (n % 4 == 0) phase();
#pragma unroll
            for (int b = 0; b < KB; ++b) {
                const u32x4 w = read16((keys ^ (32 * n)) + 32 * b * T::row);
                if constexpr (kWide) {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        s[b] = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(w[e]), q[n][e], n + e == 0 ? f32x16{} : s[b], 0, 0, 0);
                } else {
                    s[b] = E::mfma(__builtin_bit_cast(x8, w), q[n], n == 0 ? f32x16{} : s[b]);
                }
            }
        }
        if constexpr (masked)
#pragma unroll
            for (int b = 0; b < KB; ++b)
#pragma unroll
                for (int r = 0; r < 16; ++r) s[b][r] = k0 + 32 * b + 8 * (r / 4) + 4 * hi + r % 4 < lim ? s[b][r] : -__builtin_inff();
        float most = -__builtin_inff();
#pragma unroll
        for (int b = 0; b < KB; ++b)
#pragma unroll
            for (int r = 0; r < 16; ++r) most = fmaxf(most, s[b][r]);
        most *= scale;
        if (__any(most > limit)) {
            most = halves_max(most);
            const bool moves = most > limit;
            const float down = !moves ? 1.f : limit == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(ref - most + E::headroom);
            if (moves) { ref = most - E::headroom; limit = most + 8.f; }
            l *= down;
#pragma unroll
            for (int c = 0; c < CB; ++c) o[c] *= down;
        }
        // P as the second product's operands: eight Keys each, 16 kk + 4 hi .. + 3 and 16 kk + 8 + 4 hi .. + 3 (float32: four in
        // turn, one a product)
        x8 p[KK];
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) {
            if constexpr (kWide) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    p[kk][e] = __builtin_amdgcn_exp2f(fmaf(s[0][4 * kk + e], scale, -ref));
                    l += p[kk][e];
                }
            } else {
                u32x4 w;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float x = __builtin_amdgcn_exp2f(fmaf(s[kk / 2][8 * (kk & 1) + 2 * e], scale, -ref));
                    const float y = __builtin_amdgcn_exp2f(fmaf(s[kk / 2][8 * (kk & 1) + 2 * e + 1], scale, -ref));
                    l += x + y;
                    w[e] = E::pack(x, y);
                }
                p[kk] = __builtin_bit_cast(x8, w);
            }
        }
        // The same Keys' Values in channels 32 c + col.
        const auto value = [&](int kk, int c) __attribute__((always_inline)) {
            if constexpr (kWide) {
                u32x4 w;
#pragma unroll
                for (int e = 0; e < 4; ++e) w[e] = read4((values ^ (128 * c)) + (8 * kk + e) * T::row);
                return w;
            } else {
                const uint32_t at = (values ^ (64 * c)) + 16 * kk * T::row;
                const u32x2 x = read_tr(at), y = read_tr(at + 8 * T::row);
                return u32x4{x[0], x[1], y[0], y[1]};
            }
        };
        const auto multiply = [](u32x4 w, x8 weights, f32x16 sum) __attribute__((always_inline)) {
            if constexpr (kWide) {
#pragma unroll
                for (int e = 0; e < 4; ++e) sum = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(w[e]), weights[e], sum, 0, 0, 0);
                return sum;
            } else {
                return E::mfma(__builtin_bit_cast(x8, w), weights, sum);
            }
        };
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __syncthreads();  // the tile's Values are there, and nobody reads its Keys any more
        if (t + Groups < last) loader.fill(loader.keys, t + Groups, lds);
        phase();
        // What stands where a row does not see need not be finite, and 0 * NaN is NaN: rows of a tile that holds such Values are
        // formed anew.
        if constexpr (masked) {
            uint32_t found = 0;
#pragma unroll 4
            for (int n = 0; n < T::loads; ++n) {
                const u32x4 w = read16(lds + T::bytes + 1024 * n + 16 * lane);
#pragma unroll
                for (int x = 0; x < 4; ++x) found |= (w[x] & E::bits) + E::least;
            }
            odd = odd || __any((found & ~E::bits) != 0);
        }
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) {
            phase();
#pragma unroll
            for (int c = 0; c < CB; ++c) o[c] = multiply(value(kk, c), p[kk], o[c]);
        }
    };
    const int whole = min(all / KT, last);
    int t = first + turn;
    for (; t < whole; t += Groups) tile(std::false_type(), t);
    for (; t < last; t += Groups) tile(std::true_type(), t);
    l = halves_sum(l);
    if constexpr (Groups == 2) {
        if (turn == 1 && first < last && (last - first) % 2 != 0) {  // (a tile fewer: its two barriers)
            __syncthreads();
            __syncthreads();
        }
        __syncthreads();
        f32x4* sums = reinterpret_cast<f32x4*>(smem) + wave * kWave + lane;
        f32x4* stats = reinterpret_cast<f32x4*>(smem + Shape<D, Dt, NW, Groups>::lds - NW * kWave * 16) + wave * kWave + lane;
        if (turn == 1) {
#pragma unroll
            for (int n = 0; n < 4 * CB; ++n) {
                const f32x16& x = o[n / 4];
                sums[n * NW * kWave] = f32x4{x[4 * (n % 4)], x[4 * (n % 4) + 1], x[4 * (n % 4) + 2], x[4 * (n % 4) + 3]};
            }
            *stats = f32x4{ref, l, odd ? 1.f : 0.f, 0.f};
        }
        __syncthreads();
        if (turn == 1) return;
        const f32x4 other = *stats;
        const float mine = l == 0.f ? -__builtin_inff() : ref, its = other[1] == 0.f ? -__builtin_inff() : other[0];
        const float top = fmaxf(mine, its);
        const float w0 = l == 0.f ? 0.f : __builtin_amdgcn_exp2f(mine - top), w1 = other[1] == 0.f ? 0.f : __builtin_amdgcn_exp2f(its - top);
        odd = odd || __any(other[2] != 0.f);
        ref = top;
        l = l * w0 + other[1] * w1;
#pragma unroll
        for (int n = 0; n < 4 * CB; ++n) {
            const f32x4 x = sums[n * NW * kWave];
#pragma unroll
            for (int e = 0; e < 4; ++e) o[n / 4][4 * (n % 4) + e] = o[n / 4][4 * (n % 4) + e] * w0 + x[e] * w1;
        }
    }

    finish<D, Dt, NW>(a, item, h, wave, col, hi, i, j, real, lim, first * KT, last * KT, odd, l, ref, o);
}

// float32 rows of 64 and 128 channels, 128 query rows a workgroup, on the bf16 matrix cores: a number is the sum of three bf16
// parts of eight bits each, and of the nine products of two numbers' parts the six largest are formed, that of the first parts
// apart from the others; those left out are 2^-21 of |x y| or less.  Six products at sixteen times the float32 products' rate.
// Keys and Values are taken apart once, on their way from registers to LDS (32 of each a tile, three planes of bf16 rows);
// the next tile's loads run beside the products.
//
// A part below 2^-133, bf16's least, is lost: numbers below 2^-110 are off by up to that (Values of 1e-34: 5e-7 of them, of 1e-38
// 5e-3).  Parts of what is not finite are not it: one Key or Value that is not, in any tile that a workgroup walks, seen by its rows or
// not, has all its rows formed anew one Key at a time (a NaN at token 10 of one prompt, the four prompts below, heads of 128: 32 ms for
// 1.06, of 64 16; prompt_kernel, which looks at masked tiles only, 3.4 ms for 3.2 at 256).
//
// Four prompts of 2 000 to 4 096 tokens, 16 / 8 heads of 128: 1 040 to 1 080 us (1 060 TFLOP/s of bf16 products), of 64: 520 to 650; by
// float32 products 1 450 and 840, and the largest error among 700 tokens falls from 1.2e-6 to 5.6e-7 and from 9.5e-7 to 7.1e-7.  Two
// waves a SIMD at both sizes (at 128 29 registers are spilled; three waves at 64 spilled 48: 750 us).  At head_dim 256 query
// parts and sums pass the registers (152 spilled, 4 250 us against 3 240), and a single wave's 32 rows would share the parting
// of their Keys with nobody: those are multiplied as they are.
template <int D>
struct Planes {
    using T = Tile<D, LF_BF16>;
    static constexpr int keys = 32, plane = keys * T::row;
    static constexpr int units = keys * D / 8 / 256;  // eight channels of a row, of Keys and of Values each, per thread
    static constexpr int lds = 6 * plane;
};
// x's and y's parts, a word of each: eight bits of what is left, so that the three are the number, cut rather than rounded (the
// largest numbers stay finite).
__device__ __forceinline__ void three_parts(float x, float y, uint32_t (&w)[3]) {
#pragma unroll
    for (int n = 0; n < 3; ++n) {
        const uint32_t u = __float_as_uint(x), v = __float_as_uint(y);
        w[n] = __builtin_amdgcn_perm(v, u, 0x07060302);
        x -= __uint_as_float(u & 0xffff0000u);
        y -= __uint_as_float(v & 0xffff0000u);
    }
}
__device__ __forceinline__ bool finite(float x) { return fabsf(x) < __builtin_inff(); }

template <int D>
__global__ __launch_bounds__(4 * kWave, 2) void prompt_split_kernel(Prompt a) {
    using P = Planes<D>;
    using T = typename P::T;
    using E = Element<LF_BF16>;
    constexpr int NW = 4, KT = P::keys, SQ = D / 16, CB = D / 32, KK = 2, U = P::units;
    constexpr int kRows = 32 * NW;
    extern __shared__ __attribute__((aligned(1024))) unsigned char smem[];  // three planes of Keys, three of Values
    __shared__ int odd_rows;  // whether Keys or Values were not finite: parts of infinity are not
    if (threadIdx.x == 0) odd_rows = 0;
    __syncthreads();
    const int h = blockIdx.x % a.n_kv;
    const lf_prompt_item item = load_item(a);
    const int lane = threadIdx.x % kWave, wave = in_sgpr(static_cast<int>(threadIdx.x / kWave));
    const int col = lane & 31, hi = lane >> 5;
    const uint32_t lds = lds_addr(smem);

    const int row = item.tile * kRows + wave * 32 + col;
    const int j = row / a.g, i = row - j * a.g;
    const bool real = j < item.n_q;
    const int lim = real ? max(item.n_k - item.n_q + j + 1, 0) : 0;
    int all = real ? lim : 0x7fffffff;
#pragma unroll
    for (int m = 1; m < 32; m <<= 1) all = min(all, __shfl_xor(all, m, kWave));
    all = in_sgpr(all);
    const int last_token = min((item.tile * kRows + kRows - 1) / a.g, item.n_q - 1);
    const int reach = max(item.n_k - item.n_q + last_token + 1, 0);
    const int first = item.begin, last = min(item.end, (reach + KT - 1) / KT);

    const unsigned char* kbase = in_sgpr(static_cast<const unsigned char*>(a.k) + 4 * (item.k_row * a.ks[0] + h * a.ks[1] + static_cast<int64_t>(item.k_start) * a.ks[2]));
    const unsigned char* vbase = in_sgpr(static_cast<const unsigned char*>(a.v) + 4 * (item.k_row * a.vs[0] + h * a.vs[1] + static_cast<int64_t>(item.k_start) * a.vs[2]));
    const int64_t kstride = 4 * a.ks[2], vstride = 4 * a.vs[2];
    f32x4 next[2][U][2];  // the next tile's eight channels of Keys, of Values
    const auto load = [&](int t) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int unit = u * 256 + threadIdx.x, r = unit / (D / 8), c = unit % (D / 8);
            const int64_t at = min(t * KT + r, reach - 1);  // (in place of Keys past the last one that is seen, that one)
            const f32x4* k = reinterpret_cast<const f32x4*>(kbase + at * kstride + 32 * c);
            const f32x4* v = reinterpret_cast<const f32x4*>(vbase + at * vstride + 32 * c);
            next[0][u][0] = k[0];
            next[0][u][1] = k[1];
            next[1][u][0] = v[0];
            next[1][u][1] = v[1];
        }
    };
    const auto stage = [&]() __attribute__((always_inline)) {
        bool fine = true;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int unit = u * 256 + threadIdx.x, r = unit / (D / 8), c = unit % (D / 8);
#pragma unroll
            for (int side = 0; side < 2; ++side) {
                u32x4 w[3];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    uint32_t parts[3];
                    const f32x4& x = next[side][u][e / 2];
                    fine = fine && finite(x[2 * (e % 2)]) && finite(x[2 * (e % 2) + 1]);
                    three_parts(x[2 * (e % 2)], x[2 * (e % 2) + 1], parts);
#pragma unroll
                    for (int n = 0; n < 3; ++n) w[n][e] = parts[n];
                }
                unsigned char* to = smem + (side ? 3 * P::plane : 0) + r * T::row + 16 * (c ^ (side ? T::value_swap(r) : T::key_swap(r)));
#pragma unroll
                for (int n = 0; n < 3; ++n) *reinterpret_cast<u32x4*>(to + n * P::plane) = w[n];
            }
        }
        if (!fine) odd_rows = 1;
    };
    if (first < last) load(first);

    bool odd = false;
    bf16x8 q[SQ][3];
    {
        const float* src = static_cast<const float*>(a.q) + item.q_row * a.qs[0] + static_cast<int64_t>(h * a.g + i) * a.qs[1] +
                           static_cast<int64_t>(item.q_start + j) * a.qs[2] + 8 * hi;
#pragma unroll
        for (int n = 0; n < SQ; ++n) {
            f32x4 x = {0.f, 0.f, 0.f, 0.f}, y = x;
            if (real && reach > 0) {
                x = *reinterpret_cast<const f32x4*>(src + 16 * n);
                y = *reinterpret_cast<const f32x4*>(src + 16 * n + 4);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) odd = odd || !finite(x[e]) || !finite(y[e]);
            if (a.qscale < 0.f) {
                x = -x;
                y = -y;
            }
            u32x4 w[3];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                uint32_t parts[3];
                three_parts(e < 2 ? x[2 * e] : y[2 * e - 4], e < 2 ? x[2 * e + 1] : y[2 * e - 3], parts);
#pragma unroll
                for (int m = 0; m < 3; ++m) w[m][e] = parts[m];
            }
#pragma unroll
            for (int m = 0; m < 3; ++m) q[n][m] = __builtin_bit_cast(bf16x8, w[m]);
        }
    }
    const float scale = fmaxf(fabsf(a.qscale), 1e-37f);

    f32x16 o[CB];
#pragma unroll
    for (int c = 0; c < CB; ++c) o[c] = f32x16{};
    float l = 0.f, ref = 0.f, limit = -__builtin_inff();
    const uint32_t keys = lds + col * T::row + 16 * (hi ^ T::key_swap(col));
    const int group = lane >> 4, in16 = lane & 15;
    const int vrow = 4 * (group >> 1) + (in16 >> 2), vcol = 16 * (group & 1) + 4 * (in16 & 3);
    const uint32_t values = lds + 3 * P::plane + vrow * T::row + 16 * ((vcol / 8) ^ T::value_swap(vrow)) + 2 * (vcol & 7);

    for (int t = first; t < last; ++t) {
        __syncthreads();  // nobody reads the last tile any more
        stage();
        __syncthreads();
        if (t + 1 < last) load(t + 1);
        const int k0 = t * KT;
        f32x16 s = f32x16{}, rest = f32x16{};
#pragma unroll
        for (int n = 0; n < SQ; ++n) {
            bf16x8 k[3];
#pragma unroll
            for (int m = 0; m < 3; ++m) k[m] = __builtin_bit_cast(bf16x8, read16((keys ^ (32 * n)) + m * P::plane));
#pragma unroll
            for (int sum = 2; sum > 0; --sum)
#pragma unroll
                for (int m = 0; m <= sum; ++m) rest = E::mfma(k[m], q[n][sum - m], rest);
            s = E::mfma(k[0], q[n][0], s);
            if (n % 2 == 1) phase();
        }
        s += rest;
        const bool masked = k0 + KT > all;
        if (masked) {
            phase();  // (a branch, not selects in every tile)
#pragma unroll
            for (int r = 0; r < 16; ++r) s[r] = k0 + 8 * (r / 4) + 4 * hi + r % 4 < lim ? s[r] : -__builtin_inff();
        }
        float most = -__builtin_inff();
#pragma unroll
        for (int r = 0; r < 16; ++r) most = fmaxf(most, s[r]);
        most *= scale;
        if (__any(most > limit)) {
            most = halves_max(most);
            const bool moves = most > limit;
            const float down = !moves ? 1.f : limit == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(ref - most);
            if (moves) { ref = most; limit = most + 8.f; }
            l *= down;
#pragma unroll
            for (int c = 0; c < CB; ++c) o[c] *= down;
        }
        bf16x8 p[KK][3];
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) {
            u32x4 w[3];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float x = __builtin_amdgcn_exp2f(fmaf(s[8 * kk + 2 * e], scale, -ref));
                const float y = __builtin_amdgcn_exp2f(fmaf(s[8 * kk + 2 * e + 1], scale, -ref));
                l += x + y;
                uint32_t parts[3];
                three_parts(x, y, parts);
#pragma unroll
                for (int m = 0; m < 3; ++m) w[m][e] = parts[m];
            }
#pragma unroll
            for (int m = 0; m < 3; ++m) p[kk][m] = __builtin_bit_cast(bf16x8, w[m]);
        }
#pragma unroll
        for (int kk = 0; kk < KK; ++kk)
#pragma unroll
            for (int c = 0; c < CB; ++c) {
                bf16x8 v[3];
#pragma unroll
                for (int m = 0; m < 3; ++m) {
                    const uint32_t at = (values ^ (64 * c)) + m * P::plane + 16 * kk * T::row;
                    const u32x2 x = read_tr(at), y = read_tr(at + 8 * T::row);
                    v[m] = __builtin_bit_cast(bf16x8, u32x4{x[0], x[1], y[0], y[1]});
                }
#pragma unroll
                for (int sum = 2; sum >= 0; --sum)
#pragma unroll
                    for (int m = 0; m <= sum; ++m) o[c] = E::mfma(v[m], p[kk][sum - m], o[c]);
                if (c % 2 == 1) phase();
            }
    }
    // (the last barrier is behind every tile's Keys and Values)
    finish<D, LF_FP32, NW>(a, item, h, wave, col, hi, i, j, real, lim, first * KT, last * KT, __any(odd) || odd_rows != 0, halves_sum(l), ref, o);
}

// The splits' sums of a tile's rows at their largest reference point: D / 4 lanes a row, eight splits' loads at once.  (8 us for
// 34 MB of 112 tiles in four parts: HBM and the launch.)
template <int D, int Dt>
__global__ __launch_bounds__(256) void prompt_merge_kernel(Prompt a, const lf_prompt_item* items, int tile_rows) {
    constexpr int L = D / 4;
    const int h = blockIdx.x % a.n_kv;
    const lf_prompt_item item = items[blockIdx.x / a.n_kv];
    const int r = blockIdx.y * (256 / L) + threadIdx.x / L, c = threadIdx.x % L * 4;
    const int row = item.tile * tile_rows + r, j = row / a.g, i = row - j * a.g;
    if (r >= tile_rows || j >= item.n_q) return;
    const int64_t step = static_cast<int64_t>(a.n_kv) * tile_rows, at = item.slot * step + static_cast<int64_t>(h) * tile_rows + r;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
    float m = -__builtin_inff(), l = 0.f;
    constexpr int kTake = 8;  // splits whose loads are on their way at once
    for (int s0 = 0; s0 < item.parts; s0 += kTake) {
        f32x4 x[kTake];
        float ms[kTake], ls[kTake], top = m;
#pragma unroll
        for (int k = 0; k < kTake; ++k) {
            const int64_t of = at + min(s0 + k, item.parts - 1) * step;
            ms[k] = a.part_ml[2 * of];
            ls[k] = a.part_ml[2 * of + 1];
            x[k] = *reinterpret_cast<const f32x4*>(a.part_o + of * D + c);
        }
#pragma unroll
        for (int k = 0; k < kTake; ++k) top = fmaxf(top, ms[k]);
        const float down = m == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(m - top);
        m = top;
        l *= down;
        o *= down;
#pragma unroll
        for (int k = 0; k < kTake; ++k) {
            if (s0 + k >= item.parts) continue;
            // (of a split without a weight above zero the sums are zeros, or NaN from a Value that is not finite)
            const float w = ms[k] == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(ms[k] - m);
            l = fmaf(w, ls[k], l);
            o += w * x[k];
        }
    }
    o *= l == 0.f ? 0.f : 1.f / l;
    const int64_t to = item.q_row * a.os[0] + static_cast<int64_t>(h * a.g + i) * a.os[1] + static_cast<int64_t>(item.q_start + j) * a.os[2] + c;
    if constexpr (Dt == LF_FP32) *reinterpret_cast<f32x4*>(static_cast<float*>(a.out) + to) = o;
    else *reinterpret_cast<u32x2*>(static_cast<uint16_t*>(a.out) + to) = u32x2{Element<Dt>::pack(o[0], o[1]), Element<Dt>::pack(o[2], o[3])};
}

template <int D, int Dt>
int launch_rows(void (*fn)(Prompt), int waves, int lds, const Prompt& a, const lf_prompt_args& A, hipStream_t stream) {
    const int st = allow_dynamic_lds(reinterpret_cast<const void*>(fn), lds);
    if (st != LF_OK) return st;
    hipLaunchKernelGGL(fn, dim3(static_cast<uint32_t>(A.n_items) * A.n_kv), dim3(waves * kWave), lds, stream, a);
    if (A.n_merges) {
        const int rows = A.tile_rows, per = 256 / (D / 4);
        hipLaunchKernelGGL((prompt_merge_kernel<D, Dt>), dim3(static_cast<uint32_t>(A.n_merges) * A.n_kv, (rows + per - 1) / per), dim3(256), 0,
                           stream, a, A.merges, rows);
    }
    const hipError_t err = hipGetLastError();
    return err == hipSuccess ? LF_OK : static_cast<int>(err);
}

template <int D, int Dt>
int launch_typed(const Prompt& a, const lf_prompt_args& A, hipStream_t stream) {
    if (A.tile_rows == 32) return launch_rows<D, Dt>(prompt_kernel<D, Dt, 1, 1>, 1, Shape<D, Dt, 1, 1>::lds, a, A, stream);
    if constexpr (D <= 128 && Dt == LF_FP32) {
        return launch_rows<D, Dt>(prompt_split_kernel<D>, 4, Planes<D>::lds, a, A, stream);
    } else {
        if constexpr (D <= 128)
            if (A.groups == 2) return launch_rows<D, Dt>(prompt_kernel<D, Dt, 4, 2>, 8, Shape<D, Dt, 4, 2>::lds, a, A, stream);
        return launch_rows<D, Dt>(prompt_kernel<D, Dt, 4, 1>, 4, Shape<D, Dt, 4, 1>::lds, a, A, stream);
    }
}

template <int D>
int launch_dim(const Prompt& a, const lf_prompt_args& A, hipStream_t stream) {
    return A.dtype == LF_BF16 ? launch_typed<D, LF_BF16>(a, A, stream)
           : A.dtype == LF_FP16 ? launch_typed<D, LF_FP16>(a, A, stream)
                                : launch_typed<D, LF_FP32>(a, A, stream);
}

}  // namespace

int64_t prompt_part_bytes(int n_kv, int head_dim, int tile_rows, int slots) {
    return static_cast<int64_t>(slots) * n_kv * tile_rows * (head_dim + 2) * 4;
}

int launch_prompt(const lf_prompt_args& A, hipStream_t stream) {
    Prompt a{};
    a.q = A.query; a.k = A.key; a.v = A.value; a.out = A.out;
    for (int i = 0; i < 3; ++i) {
        a.qs[i] = A.q_strides[i]; a.ks[i] = A.k_strides[i];
        a.vs[i] = A.v_strides[i]; a.os[i] = A.out_strides[i];
    }
    a.items = A.items;
    a.n_q = A.n_q; a.n_kv = A.n_kv; a.g = A.n_q / A.n_kv;
    a.qscale = A.scaling * kLog2e;
    const int64_t near = (1ll << 31) / (64 * 4);
    a.far = A.k_strides[2] < 0 || A.v_strides[2] < 0 || A.k_strides[2] >= near || A.v_strides[2] >= near;
    a.part_o = static_cast<float*>(A.workspace);
    a.part_ml = a.part_o + static_cast<int64_t>(A.n_slots) * A.n_kv * A.tile_rows * A.head_dim;
    return A.head_dim == 64 ? launch_dim<64>(a, A, stream) : A.head_dim == 128 ? launch_dim<128>(a, A, stream) : launch_dim<256>(a, A, stream);
}

}  // namespace lf
