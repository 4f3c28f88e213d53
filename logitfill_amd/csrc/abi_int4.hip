// extern "C" entry points of the 4-bit row cache: arguments are checked here, before anything is enqueued.
#include "int4_common.hpp"

#include <cmath>

namespace lf {
int launch_int4_set_lens(const lf_int4_layer& L, const int32_t* lens, hipStream_t stream);
int launch_int4_append(const lf_int4_layer& L, const void* k_src, const void* v_src, int dtype, const int64_t* k_strides,
                       const int64_t* v_strides, const int32_t* starts, const int32_t* counts, int tokens,
                       hipStream_t stream);
int launch_int4_read(const lf_int4_layer& L, const int32_t* starts, int tokens, void* k_out, void* v_out, int dtype,
                     hipStream_t stream);
int launch_int4_attention(const lf_int4_layer& L, const lf_int4_args& A, hipStream_t stream);
int launch_int4_shared(const lf_int4_layer& L, const lf_int4_layer& P, const lf_int4_args& A, int splits, int split_tokens, bool many_rows,
                       hipStream_t stream);
int launch_int4_select(const lf_int4_layer& L, const lf_int4_args& A, hipStream_t stream);
int64_t int4_part_bytes(const lf_int4_layer& L, int n_q, int q_len, int splits);
int64_t int4_keys_bytes(const lf_int4_layer& L, int q_len);
}  // namespace lf

namespace {

constexpr int kMaxSplits = 1024, kMaxPages = 1024;
constexpr int kGrid = 65535;  // of the y and z dimensions

bool valid_dtype(int32_t d) { return d == LF_BF16 || d == LF_FP16 || d == LF_FP32; }
bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

int32_t check_int4(const lf_int4_layer* L) {
    if (!L || !L->blocks || !L->bounds || !L->lens || !L->tops) return LF_E_NULL;
    if (L->batch <= 0 || L->n_kv <= 0 || L->batch > kGrid || L->n_kv > kGrid) return LF_E_SHAPE;
    if (L->head_dim != 64 && L->head_dim != 128 && L->head_dim != 256) return LF_E_UNSUPPORTED;
    if ((L->group != 32 && L->group != 64 && L->group != 128) || L->group > L->head_dim) return LF_E_UNSUPPORTED;
    if (L->page_size <= 0 || L->page_size % 32 != 0 || L->page_size > 1024) return LF_E_SHAPE;
    if (L->cap_tokens <= 0 || L->cap_tokens % L->page_size != 0 || L->cap_tokens > (1 << 30)) return LF_E_SHAPE;
    if (!aligned16(L->blocks) || !aligned16(L->bounds)) return LF_E_SHAPE;
    return LF_OK;
}

// Query rows of an attention or selection call.
int32_t check_query(const lf_int4_layer* L, const lf_int4_args* A) {
    const int32_t st = check_int4(L);
    if (st != LF_OK) return st;
    if (!A || !A->query) return LF_E_NULL;
    if (!valid_dtype(A->dtype)) return LF_E_DTYPE;
    if (A->n_q <= 0 || A->n_q % L->n_kv != 0 || A->q_len <= 0) return LF_E_SHAPE;
    if (static_cast<int64_t>(A->n_q) * A->q_len > (1 << 20)) return LF_E_SHAPE;
    if (static_cast<int64_t>(A->n_q) * A->q_len * L->batch >= 1 << 24) return LF_E_SHAPE;  // (256 threads a row, 2^32 in a grid)
    // a workgroup row per (kv head, query token) or (kv head, 16 rows), whichever are more
    const int64_t g = A->n_q / L->n_kv, rows = A->n_pages > 0 ? (g + 15) / 16 * A->q_len : (g * A->q_len + 15) / 16;
    if (rows * L->n_kv > kGrid) return LF_E_SHAPE;
    if (A->n_pages < 0 || A->n_pages > kMaxPages) return LF_E_SHAPE;
    if (A->n_pages > 0 && !A->pages) return LF_E_NULL;
    return LF_OK;
}

// An attention call's arguments, with ``shared`` parts in front of its own.
int32_t check_attention(const lf_int4_layer* layer, const lf_int4_args* args, int shared) {
    const int32_t st = check_query(layer, args);
    if (st != LF_OK) return st;
    const lf_int4_args& A = *args;
    if (!A.out) return LF_E_NULL;
    if (!aligned16(A.out)) return LF_E_SHAPE;
    if (!std::isfinite(A.scaling)) return LF_E_SHAPE;  // (the kernels take the larger of it and 1e-37)
    if (A.splits <= 0 || A.splits > kMaxSplits) return LF_E_SHAPE;
    if (A.n_pages == 0 && A.splits > 1 && (A.split_tokens <= 0 || A.split_tokens % 32 != 0)) return LF_E_SHAPE;
    if (A.prefix_splits < 0 || A.prefix_splits > kMaxSplits) return LF_E_SHAPE;
    if (A.prefix_splits > 0) {
        if (A.splits != 1) return LF_E_SHAPE;
        if (A.n_pages > 0 || A.dtype != LF_BF16 || layer->head_dim > 128) return LF_E_UNSUPPORTED;
    }
    const int parts = A.splits + A.prefix_splits + shared;
    if (parts > 1) {
        if (!A.workspace) return LF_E_NULL;
        if (!aligned16(A.workspace)) return LF_E_SHAPE;
        if (A.workspace_bytes < lf::int4_part_bytes(*layer, A.n_q, A.q_len, parts)) return LF_E_WORKSPACE;
    }
    return LF_OK;
}

}  // namespace

extern "C" {

int32_t lf_int4_set_lens(const lf_int4_layer* layer, const int32_t* lens, void* stream) {
    const int32_t st = check_int4(layer);
    if (st != LF_OK) return st;
    if (!lens) return LF_E_NULL;
    for (int32_t b = 0; b < layer->batch; ++b)
        if (lens[b] < 0 || lens[b] > layer->cap_tokens) return LF_E_SHAPE;
    return lf::launch_int4_set_lens(*layer, lens, static_cast<hipStream_t>(stream));
}

int32_t lf_int4_append(const lf_int4_layer* layer, const void* k_src, const void* v_src, int32_t dtype,
                       const int64_t* k_strides, const int64_t* v_strides, const int32_t* starts, const int32_t* counts,
                       int32_t tokens, void* stream) {
    const int32_t st = check_int4(layer);
    if (st != LF_OK) return st;
    if (!valid_dtype(dtype)) return LF_E_DTYPE;
    if (tokens < 0 || tokens > (1 << 30)) return LF_E_SHAPE;
    if (tokens == 0) return LF_OK;
    if (!k_src || !v_src || !k_strides || !v_strides) return LF_E_NULL;
    for (int32_t b = 0; counts && b < layer->batch; ++b)
        if (counts[b] < 0 || counts[b] > tokens) return LF_E_SHAPE;
    for (int32_t b = 0; starts && b < layer->batch; ++b)
        if (starts[b] < 0 || starts[b] > layer->cap_tokens) return LF_E_SHAPE;
    return lf::launch_int4_append(*layer, k_src, v_src, dtype, k_strides, v_strides, starts, counts, tokens,
                                  static_cast<hipStream_t>(stream));
}

int32_t lf_int4_read(const lf_int4_layer* layer, const int32_t* starts, int32_t tokens, void* k_out, void* v_out,
                     int32_t dtype, void* stream) {
    const int32_t st = check_int4(layer);
    if (st != LF_OK) return st;
    if (!valid_dtype(dtype)) return LF_E_DTYPE;
    if (tokens < 0 || tokens > (1 << 30)) return LF_E_SHAPE;
    if (!k_out && !v_out) return LF_E_NULL;
    if (!aligned16(k_out) || !aligned16(v_out)) return LF_E_SHAPE;
    for (int32_t b = 0; starts && b < layer->batch; ++b)
        if (starts[b] < 0 || starts[b] > (1 << 30)) return LF_E_SHAPE;
    if (tokens == 0) return LF_OK;
    return lf::launch_int4_read(*layer, starts, tokens, k_out, v_out, dtype, static_cast<hipStream_t>(stream));
}

int64_t lf_int4_workspace_bytes(const lf_int4_layer* layer, int32_t n_q, int32_t q_len, int32_t splits) {
    if (!layer || layer->batch <= 0 || layer->head_dim <= 0 || n_q <= 0 || q_len <= 0 || splits <= 0 || splits > kMaxSplits + 1)
        return LF_E_SHAPE;
    return lf::int4_part_bytes(*layer, n_q, q_len, splits);
}

int32_t lf_int4_attention(const lf_int4_layer* layer, const lf_int4_args* args, void* stream) {
    const int32_t st = check_attention(layer, args, 0);
    return st != LF_OK ? st : lf::launch_int4_attention(*layer, *args, static_cast<hipStream_t>(stream));
}

int32_t lf_int4_shared_attention(const lf_int4_layer* layer, const lf_int4_layer* prefix, const lf_int4_args* args,
                                 int32_t shared_splits, int32_t shared_split_tokens, int32_t many_rows, void* stream) {
    int32_t st = check_int4(prefix);
    if (st != LF_OK) return st;
    if (shared_splits <= 0 || shared_splits > kMaxSplits) return LF_E_SHAPE;
    st = check_attention(layer, args, shared_splits);
    if (st != LF_OK) return st;
    const lf_int4_args& A = *args;
    if (A.splits + A.prefix_splits + shared_splits > kMaxSplits + 1) return LF_E_SHAPE;
    if (prefix->n_kv != layer->n_kv || prefix->head_dim != layer->head_dim || prefix->group != layer->group) return LF_E_SHAPE;
    if (layer->batch % prefix->batch != 0) return LF_E_SHAPE;
    if (A.n_pages > 0) return LF_E_UNSUPPORTED;
    if (many_rows ? A.dtype != LF_BF16 || layer->head_dim > 128 : shared_split_tokens <= 0 || shared_split_tokens % 32 != 0)
        return many_rows ? LF_E_UNSUPPORTED : LF_E_SHAPE;
    // (256 threads a workgroup, 2^32 in a grid)
    const int64_t g = A.n_q / layer->n_kv, rows = g * A.q_len * (layer->batch / prefix->batch), tile = many_rows ? 128 : 16;
    const int64_t shared = (rows + tile - 1) / tile * layer->n_kv * prefix->batch * shared_splits;
    const int64_t own = (g * A.q_len + 15) / 16 * layer->n_kv * layer->batch * A.splits;
    if (shared + own >= 1 << 24) return LF_E_SHAPE;
    return lf::launch_int4_shared(*layer, *prefix, A, shared_splits, shared_split_tokens, many_rows != 0, static_cast<hipStream_t>(stream));
}

int64_t lf_int4_select_workspace_bytes(const lf_int4_layer* layer, int32_t q_len) {
    if (!layer || layer->batch <= 0 || layer->n_kv <= 0 || layer->page_size <= 0 || layer->cap_tokens < 0 || q_len <= 0)
        return LF_E_SHAPE;
    return lf::int4_keys_bytes(*layer, q_len);
}

int32_t lf_int4_select(const lf_int4_layer* layer, const lf_int4_args* args, void* stream) {
    const int32_t st = check_query(layer, args);
    if (st != LF_OK) return st;
    const lf_int4_args& A = *args;
    if (A.n_pages == 0) return LF_E_SHAPE;
    if (static_cast<int64_t>(layer->n_kv) * A.q_len > kGrid) return LF_E_SHAPE;
    if (!A.workspace) return LF_E_NULL;
    if (!aligned16(A.workspace)) return LF_E_SHAPE;
    if (A.workspace_bytes < lf::int4_keys_bytes(*layer, A.q_len)) return LF_E_WORKSPACE;
    return lf::launch_int4_select(*layer, A, static_cast<hipStream_t>(stream));
}

}  // extern "C"
