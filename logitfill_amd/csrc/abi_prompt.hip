// extern "C" entry points of a prompt's operators: arguments are checked here, before anything is enqueued.
#include "lf_common.hpp"

#include <cmath>

namespace lf {
int launch_rotary(const lf_rotary_args& A, hipStream_t stream);
int launch_prompt(const lf_prompt_args& A, hipStream_t stream);
int64_t prompt_part_bytes(int n_kv, int head_dim, int tile_rows, int slots);
}  // namespace lf

namespace {

bool valid_dtype(int32_t d) { return d == LF_BF16 || d == LF_FP16 || d == LF_FP32; }
bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }
bool aligned16(const void* p, const int64_t* strides, int esize) {
    return aligned16(p) && strides[0] * esize % 16 == 0 && strides[1] * esize % 16 == 0 && strides[2] * esize % 16 == 0;
}

}  // namespace

extern "C" {

int32_t lf_rotary(const lf_rotary_args* args, void* stream) {
    if (!args) return LF_E_NULL;
    const lf_rotary_args& A = *args;
    if (!valid_dtype(A.dtype)) return LF_E_DTYPE;
    if (A.batch < 0 || A.tokens < 0 || A.n_q < 0 || A.n_kv < 0) return LF_E_SHAPE;
    if (A.head_dim < 2 || A.head_dim > 512 || A.head_dim % 2 != 0) return LF_E_SHAPE;
    if (A.rotary_dim < 2 || A.rotary_dim > A.head_dim || A.rotary_dim % 2 != 0) return LF_E_SHAPE;
    if (static_cast<int64_t>(A.batch) * A.tokens >= 1ll << 27) return LF_E_SHAPE;
    if (static_cast<int64_t>(A.n_q) + A.n_kv > 4096) return LF_E_SHAPE;
    if (!std::isfinite(A.factor)) return LF_E_SHAPE;
    if (!A.positions && (A.start < -(1ll << 53) || A.start > 1ll << 53)) return LF_E_SHAPE;
    if (A.batch == 0 || A.tokens == 0 || A.n_q + A.n_kv == 0) return LF_OK;
    if (!A.turns || (A.n_q && (!A.query || !A.query_out)) || (A.n_kv && (!A.key || !A.key_out))) return LF_E_NULL;
    return lf::launch_rotary(A, static_cast<hipStream_t>(stream));
}

int64_t lf_prompt_workspace_bytes(int32_t n_kv, int32_t head_dim, int32_t tile_rows, int32_t n_slots) {
    if (n_kv <= 0 || head_dim <= 0 || tile_rows <= 0 || n_slots < 0) return LF_E_SHAPE;
    return lf::prompt_part_bytes(n_kv, head_dim, tile_rows, n_slots);
}

int32_t lf_prompt_attention(const lf_prompt_args* args, void* stream) {
    if (!args) return LF_E_NULL;
    const lf_prompt_args& A = *args;
    if (!valid_dtype(A.dtype)) return LF_E_DTYPE;
    if (A.head_dim != 64 && A.head_dim != 128 && A.head_dim != 256) return LF_E_UNSUPPORTED;
    if (A.n_kv <= 0 || A.n_q <= 0 || A.n_q % A.n_kv != 0 || A.n_items < 0 || A.n_merges < 0 || A.n_slots < 0) return LF_E_SHAPE;
    if (A.tile_rows != 32 && A.tile_rows != 128) return LF_E_SHAPE;
    if (A.groups != 1 && (A.groups != 2 || A.tile_rows != 128 || A.head_dim > 128 || A.dtype == LF_FP32)) return LF_E_SHAPE;
    // (2^32 threads in a grid)
    const int64_t threads = A.tile_rows == 32 ? 64 : 256 * A.groups;
    if (static_cast<int64_t>(A.n_items) * A.n_kv * threads >= 1ll << 32 || static_cast<int64_t>(A.n_merges) * A.n_kv * 256 >= 1ll << 32) return LF_E_SHAPE;
    if (!std::isfinite(A.scaling)) return LF_E_SHAPE;
    if (A.n_items == 0) return LF_OK;
    if (!A.query || !A.key || !A.value || !A.out || !A.items || (A.n_merges && !A.merges)) return LF_E_NULL;
    const int esize = A.dtype == LF_FP32 ? 4 : 2;
    if (!aligned16(A.query, A.q_strides, esize) || !aligned16(A.key, A.k_strides, esize) || !aligned16(A.value, A.v_strides, esize) ||
        !aligned16(A.out, A.out_strides, esize))
        return LF_E_SHAPE;
    if (A.n_slots < 2ll * A.n_merges) return LF_E_SHAPE;
    if (A.n_slots) {
        if (!A.workspace) return LF_E_NULL;
        if (!aligned16(A.workspace)) return LF_E_SHAPE;
        if (A.workspace_bytes < lf::prompt_part_bytes(A.n_kv, A.head_dim, A.tile_rows, A.n_slots)) return LF_E_WORKSPACE;
    }
    return lf::launch_prompt(A, static_cast<hipStream_t>(stream));
}

}  // extern "C"
