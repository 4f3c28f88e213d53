// The work of a prompt-attention call, planned on the host: row tiles of the sequences, and how many Key tiles a workgroup takes.
#include "lf_common.hpp"

#include <algorithm>
#include <functional>
#include <new>
#include <queue>
#include <vector>

namespace {

// Microseconds of a Key tile for a workgroup that has its compute unit to itself, and a compute unit's share of one where it
// holds as many as it can (four waves); of a workgroup's start and end; of the launch that merges divided row tiles; of
// joining a workgroup's two groups.  Measured on one kv head's Keys, 8 192 of them, read by 32 to 1 024 workgroups of four waves.
// Workgroups of one wave (few rows) are planned by the same figures, and no term stands for HBM, which bounds them: sixteen
// tokens behind 32 768 each get 128 workgroups a kv head and 201 us, their bytes take 210 at a copy's rate; in float32 669 and 421.
struct Cost { double alone, shared; };
constexpr double kItem = 3.0, kMerge = 5.0, kPair = 1.5;

Cost tile_cost(const lf_prompt_batch& B) {
    if (B.dtype == LF_FP32) return B.head_dim == 64 ? Cost{1.95, 1.5} : B.head_dim == 128 ? Cost{3.5, 2.7} : Cost{8.4, 8.4};
    return B.head_dim == 64 ? Cost{0.9, 0.69} : B.head_dim == 128 ? Cost{1.5, 0.95} : Cost{1.5, 1.25};
}

// Workgroups that a compute unit holds: of four waves by their registers, of one by the LDS of its tiles.
int per_unit(const lf_prompt_batch& B) {
    const bool wide = B.dtype == LF_FP32;
    if (B.tile_rows == 32) return 163840 / 2 / (LF_PROMPT_KEYS(B.head_dim, B.dtype) * B.head_dim * (wide ? 4 : 2));
    return B.head_dim == 64 ? wide ? 2 : 4 : B.head_dim == 128 ? wide ? 2 : 3 : wide ? 1 : 2;
}

int64_t up(int64_t a, int64_t b) { return (a + b - 1) / b; }
uint32_t up(uint32_t a, uint32_t b) { return (a + b - 1) / b; }  // (of rows and tiles: below 2^31 together)

int32_t check(const lf_prompt_batch* batch) {
    if (!batch || !batch->lengths || !batch->key_lengths) return LF_E_NULL;
    const lf_prompt_batch& B = *batch;
    if (B.dtype != LF_BF16 && B.dtype != LF_FP16 && B.dtype != LF_FP32) return LF_E_DTYPE;
    if (B.head_dim != 64 && B.head_dim != 128 && B.head_dim != 256) return LF_E_UNSUPPORTED;
    if (B.batch <= 0 || B.tokens < 0 || B.group <= 0 || B.n_kv <= 0 || B.compute_units <= 0) return LF_E_SHAPE;
    if (B.tile_rows != 32 && B.tile_rows != 128) return LF_E_SHAPE;
    int64_t total = 0, keys = 0;
    for (int32_t b = 0; b < B.batch; ++b) {
        if (B.lengths[b] < 0 || B.key_lengths[b] < 0 || B.lengths[b] > LF_PROMPT_TOKENS || B.key_lengths[b] > LF_PROMPT_TOKENS) return LF_E_SHAPE;
        if (static_cast<int64_t>(B.lengths[b]) * B.group > 1 << 30) return LF_E_SHAPE;
        total += B.lengths[b];
        keys += B.key_lengths[b];
    }
    if (static_cast<int64_t>(B.tokens) * B.group > 1 << 30) return LF_E_SHAPE;
    if ((B.packed_q && total >= 1ll << 31) || (B.packed_k && keys >= 1ll << 31)) return LF_E_SHAPE;
    return LF_OK;
}

// Calls use(item, Key tiles) for every row tile: of the sequences, then of what lies behind them in rows of B.tokens, queries
// that see no Key.
template <typename Use>
void each_row_tile(const lf_prompt_batch& B, Use use) {
    const uint32_t keys = LF_PROMPT_KEYS(B.head_dim, B.dtype), group = B.group, rows = B.tile_rows;
    const auto sequence = [&](lf_prompt_item x) {
        const uint32_t tiles = up(static_cast<uint32_t>(x.n_q) * group, rows);
        for (uint32_t t = 0; t < tiles; ++t) {
            const int32_t last = std::min<int32_t>(((t + 1) * rows - 1) / group, x.n_q - 1);
            const int32_t reach = std::max(x.n_k - x.n_q + last + 1, 0);
            x.tile = static_cast<int32_t>(t);
            use(x, up(static_cast<uint32_t>(reach), keys));
        }
    };
    lf_prompt_item x{};
    int32_t q = 0, k = 0;
    for (int32_t b = 0; b < B.batch; ++b) {
        x.q_row = B.packed_q ? 0 : b;
        x.q_start = B.packed_q ? q : 0;
        x.n_q = B.lengths[b];
        x.k_row = B.packed_k ? 0 : b;
        x.k_start = B.packed_k ? k : 0;
        x.n_k = B.key_lengths[b];
        sequence(x);
        q += B.packed_q ? x.n_q : 0;
        k += B.packed_k ? x.n_k : 0;
    }
    x.k_row = x.k_start = x.n_k = 0;
    for (int32_t b = 0; b < (B.packed_q ? 1 : B.batch); ++b) {
        x.q_row = b;
        x.q_start = B.packed_q ? q : B.lengths[b];
        x.n_q = std::max(B.tokens - x.q_start, 0);
        sequence(x);
    }
}

// How a row tile of ``tiles`` Key tiles is divided where a workgroup takes ``size`` at most: parts of ``each`` (none is empty).
struct Parts { uint32_t parts, each; };
Parts divide(uint32_t tiles, uint32_t size) {
    if (tiles <= size) return {1, tiles};
    const uint32_t each = up(tiles, up(tiles, size));
    return {up(tiles, each), each};
}

// (Key tiles that a workgroup takes at most, its groups) of least estimated time.  A division's gain is the compute units that
// it sets to work, its price the partial sums, written and read once, and the launch that merges them.  Two groups
// share a workgroup's tiles without either, where a compute unit has one workgroup at most.
void choose(const lf_prompt_batch& B, int32_t* split) {
    std::vector<int64_t> of;  // row tiles of so many Key tiles
    each_row_tile(B, [&](const lf_prompt_item&, uint32_t tiles) {
        if (tiles >= of.size()) of.resize(tiles + 1);
        ++of[tiles];
    });
    const int64_t longest = std::max<int64_t>(static_cast<int64_t>(of.size()) - 1, 1);
    of.resize(longest + 1);
    const Cost cost = tile_cost(B);
    const int64_t units = B.compute_units, slots = units * per_unit(B);
    const bool one = per_unit(B) == 1, pairs = B.tile_rows == 128 && B.head_dim <= 128 && B.dtype != LF_FP32;
    std::vector<int64_t> sizes, items;
    for (const int64_t parts : {1, 2, 3, 4, 5, 6, 8, 10, 12, 16, 24, 32, 48, 64, 96, 128, 192, 256}) {
        if (parts > longest) break;
        const int64_t size = up(longest, parts);
        sizes.push_back(size);
        // (the ends of a compute unit of one workgroup, which takes them in turn, hang on a tile more or less)
        if (one && size > 1) sizes.push_back(size - 1);
    }
    std::sort(sizes.begin(), sizes.end(), [](int64_t a, int64_t b) { return a > b; });
    sizes.erase(std::unique(sizes.begin(), sizes.end()), sizes.end());
    double best = -1;
    split[0] = static_cast<int32_t>(longest);
    split[1] = 1;
    for (const int64_t size : sizes) {
        const bool whole = size >= longest;
        items.assign(size + 1, 0);  // workgroups of so many Key tiles
        int64_t n = 0, sum = 0, divided = 0;
        for (int64_t t = 1; t <= longest; ++t) {
            if (!of[t]) continue;
            const int64_t parts = up(t, size), count = of[t] * parts * B.n_kv;
            items[up(t, parts)] += count;
            n += count;
            sum += up(t, parts) * count;
            if (parts > 1) divided += of[t] * parts;
        }
        const double more = whole ? 0 : kMerge + 8e-6 * divided * B.n_kv * B.tile_rows * (B.head_dim + 2) / 4;
        double even = (sum * cost.shared + n * 0.25 * kItem) / units;
        // the workgroups of the compute unit that has the longest ones of each rank at once
        double first = kItem;
        if (one && n > slots) {  // one after the other: the next goes to the unit that ends first
            first = std::max(size * cost.shared + kItem, (sum * cost.shared + n * kItem) / slots);
            if (n <= 64 * slots && (best < 0 || first + more < 0.97 * best)) {
                std::priority_queue<double, std::vector<double>, std::greater<double>> ends;
                for (int64_t i = 0; i < slots; ++i) ends.push(0);
                for (int64_t s = size; s > 0; --s)
                    for (int64_t i = 0; i < items[s]; ++i) {
                        const double end = ends.top() + s * cost.shared + kItem;
                        ends.pop();
                        ends.push(end);
                        first = std::max(first, end);
                    }
            }
        } else {
            int64_t rank = 0, behind = 0;  // of the longest first; tiles past the slots
            for (int64_t s = size; s > 0; --s) {
                const int64_t end = rank + items[s], in = std::min(end, slots);
                if (in > rank) first += s * cost.shared * (up(in, units) - up(rank, units));
                if (end > slots) behind += s * (end - std::max(rank, slots));
                rank = end;
            }
            if (n > slots) even += 0.3 * behind / (n - slots) * cost.shared;
        }
        double least = std::max({first, even, size * cost.alone + kItem});
        int groups = 1;
        const double paired = up(size, 2) * std::max(1.2 * cost.alone, 2.2 * cost.shared) + kItem + kPair;
        const bool can = pairs && n <= units && size > 1;
        if (best < 0 || least + more < 0.97 * best) {
            best = least + more;
            split[0] = static_cast<int32_t>(size);
            split[1] = groups;
        }
        if (can && paired + more < 0.97 * best) {
            best = paired + more;
            split[0] = static_cast<int32_t>(size);
            split[1] = 2;
        }
        if (can) least = std::min(least, paired);
        if (whole && n >= 4 * slots) break;  // (as many row tiles keep every compute unit at work)
        if (least + more > 1.5 * best) break;
    }
}

int32_t list(const lf_prompt_batch& B, int32_t size, lf_prompt_item* items, int32_t cap, int32_t* counts) {
    // the longest first: the short ones fill what is left
    int64_t n = 0, merges = 0, slots = 0;
    uint32_t longest = 0;
    each_row_tile(B, [&](const lf_prompt_item&, uint32_t tiles) {
        const Parts p = divide(tiles, size);
        n += p.parts;
        merges += p.parts > 1;
        slots += p.parts > 1 ? p.parts : 0;
        longest = std::max(longest, p.each);
    });
    if (n >= 1ll << 31 || n + merges >= 1ll << 31) return LF_E_SHAPE;
    counts[0] = static_cast<int32_t>(n);
    counts[1] = static_cast<int32_t>(merges);
    counts[2] = static_cast<int32_t>(slots);
    if (cap < n + merges || !items) return cap <= 0 || items ? LF_E_WORKSPACE : LF_E_NULL;
    std::vector<int64_t> at(longest + 1);  // first place of the items of so many Key tiles
    each_row_tile(B, [&](const lf_prompt_item&, uint32_t tiles) {
        const Parts p = divide(tiles, size);
        at[p.each] += p.parts - 1;
        ++at[tiles - (p.parts - 1) * p.each];
    });
    int64_t before = 0;
    for (int64_t s = longest; s >= 0; --s) {
        const int64_t count = at[s];
        at[s] = before;
        before += count;
    }
    int32_t slot = 0;
    lf_prompt_item* merge = items + n;
    each_row_tile(B, [&](lf_prompt_item x, uint32_t tiles) {
        const Parts p = divide(tiles, size);
        x.parts = static_cast<int32_t>(p.parts);
        x.slot = slot;
        if (p.parts > 1) *merge++ = x;
        for (uint32_t i = 0; i < p.parts; ++i) {
            x.begin = static_cast<int32_t>(i * p.each);
            x.end = static_cast<int32_t>(std::min((i + 1) * p.each, tiles));
            x.slot = p.parts > 1 ? slot++ : -1;
            items[at[x.end - x.begin]++] = x;
        }
    });
    return LF_OK;
}

}  // namespace

extern "C" {

int32_t lf_prompt_split(const lf_prompt_batch* batch, int32_t* split) {
    const int32_t st = check(batch);
    if (st != LF_OK) return st;
    if (!split) return LF_E_NULL;
    try {
        choose(*batch, split);
    } catch (const std::bad_alloc&) {
        return LF_E_WORKSPACE;
    }
    return LF_OK;
}

int32_t lf_prompt_items(const lf_prompt_batch* batch, int32_t split_size, lf_prompt_item* items, int32_t cap, int32_t* counts) {
    const int32_t st = check(batch);
    if (st != LF_OK) return st;
    if (!counts) return LF_E_NULL;
    if (split_size <= 0) return LF_E_SHAPE;
    try {
        return list(*batch, split_size, items, cap, counts);
    } catch (const std::bad_alloc&) {
        return LF_E_WORKSPACE;
    }
}

}  // extern "C"
