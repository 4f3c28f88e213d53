// extern "C" entry points of a prompt's operators: arguments are checked here, before anything is enqueued.
#include "lf_common.hpp"

#include <cmath>

namespace lf {
int launch_rotary(const lf_rotary_args& A, hipStream_t stream);
}  // namespace lf

namespace {

bool valid_dtype(int32_t d) { return d == LF_BF16 || d == LF_FP16 || d == LF_FP32; }

}  // namespace

extern "C" {

int32_t lf_rotary(const lf_rotary_args* args, void* stream) {
    if (!args) return LF_E_NULL;
    const lf_rotary_args& A = *args;
    if (!valid_dtype(A.dtype)) return LF_E_DTYPE;
    if (A.batch < 0 || A.tokens < 0 || A.n_q < 0 || A.n_kv < 0) return LF_E_SHAPE;
    if (A.head_dim < 2 || A.head_dim > 512 || A.head_dim % 2 != 0) return LF_E_SHAPE;
    if (A.rotary_dim < 2 || A.rotary_dim > A.head_dim || A.rotary_dim % 2 != 0) return LF_E_SHAPE;
    if (static_cast<int64_t>(A.batch) * A.tokens >= 1ll << 31) return LF_E_SHAPE;
    if (static_cast<int64_t>(A.n_q) + A.n_kv > 4096) return LF_E_SHAPE;
    if (!std::isfinite(A.factor)) return LF_E_SHAPE;
    if (A.batch == 0 || A.tokens == 0 || A.n_q + A.n_kv == 0) return LF_OK;
    if (!A.turns || (A.n_q && (!A.query || !A.query_out)) || (A.n_kv && (!A.key || !A.key_out))) return LF_E_NULL;
    return lf::launch_rotary(A, static_cast<hipStream_t>(stream));
}

}  // extern "C"
