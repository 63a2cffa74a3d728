#pragma once
// Norm, rotation and append of q / k / v rows (no counterpart in the reference, whose callers norm and rotate elsewhere):
// the C ABI's pd_qk_norm_rope and pd_append_qkv behind the error behaviour of the other decode:: headers.

#include "decode.hpp"

#include <vector>

namespace decode {

using QKVRows      = pd_qkv;            // rows of one call, see pd_b200.h; zero-initialise and fill
using AppendTarget = pd_append_target;

// A rotation of the first 2 * inv_freq.size() dims of every head; `axes` names the row of the positions that drives each
// frequency (empty: one axis).  May be destroyed as soon as the calls it was passed to have returned.
class Rope {
public:
    explicit Rope(const std::vector<double>& inv_freq, bool interleaved = false, const std::vector<int>& axes = {}, float scale = 1.0f) {
        if (!axes.empty() && axes.size() != inv_freq.size()) throw std::invalid_argument("Rope: one axis per frequency");
        check(pd_rope_create(2 * static_cast<int>(inv_freq.size()), inv_freq.data(), axes.empty() ? nullptr : axes.data(),
                             interleaved, scale, &h_));
    }
    ~Rope() { pd_rope_destroy(h_); }
    Rope(const Rope&)            = delete;
    Rope& operator=(const Rope&) = delete;
    const pd_rope* handle() const { return h_; }

private:
    pd_rope* h_ = nullptr;
};

// rope may be null: norm only.  Output strides in elements; 0: dense.
inline void qk_norm_rope(const QKVRows& x, const Rope* rope, void* q_out, long long q_out_stride, void* k_out,
                         long long k_out_stride, cudaStream_t stream = 0) {
    check(pd_qk_norm_rope(&x, rope ? rope->handle() : nullptr, q_out, q_out_stride, k_out, k_out_stride, stream));
}

inline int scale_block_tokens(int page_size) { return pd_scale_block_tokens(page_size); }

inline void append_qkv(KVDtype dtype, const QKVRows& x, const Rope* rope, const AppendTarget& target, half* q_out,
                       cudaStream_t stream = 0) {
    check(pd_append_qkv(static_cast<int>(dtype), &x, rope ? rope->handle() : nullptr, &target, q_out, stream));
}

}  // namespace decode
