// Norm, rotation and append of q / k / v rows: argument checks and launches.  Part of pd_abi.cu (included there, after
// the error helpers); not a stand-alone header.
#pragma once

struct pd_rope {
    pdk::RopeArgs args{};
};

namespace {

// Largest power of two that divides the page, at most 16: blocks tile every page, whatever its size.
int scale_block_log2(int page_size) {
    int lb = 0;
    while (lb < 4 && page_size % (2 << lb) == 0) lb++;
    return lb;
}

bool unaligned4(const void* p) { return reinterpret_cast<uintptr_t>(p) % 4 != 0; }
bool unaligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 != 0; }

// One of q, k, v: rows of heads * 128 elements, `stride` elements apart (0: dense).
int check_rows(const char* who, const char* name, const void* p, long long* stride, int heads) {
    const long long width = static_cast<long long>(heads) * 128;
    if (*stride == 0) *stride = width;
    if (heads == 0) return PD_OK;
    if (!p) return set_error(PD_INVALID_ARGUMENT, "%s: %s is null", who, name);
    if (unaligned16(p)) return set_error(PD_INVALID_ARGUMENT, "%s: %s must be 16-byte aligned", who, name);
    if (*stride < width || *stride % 8 != 0)
        return set_error(PD_INVALID_ARGUMENT, "%s: %s rows must be at least %lld elements apart, in multiples of 8", who, name, width);
    return PD_OK;
}

// What norm_rope and append share.  `own_positions`: the rows' places in the cache stand in for missing positions.
int fill_rows(const char* who, const pd_qkv* x, const pd_rope* rope, bool own_positions, pdk::RowArgs* a, pdk::RopeArgs* r) {
    if (!x) return set_error(PD_INVALID_ARGUMENT, "%s: null rows", who);
    if (x->act_dtype != PD_ACT_FP16 && x->act_dtype != PD_ACT_BF16) return set_error(PD_INVALID_ARGUMENT, "%s: unsupported row dtype %d", who, x->act_dtype);
    if (x->head_dim != 128) return set_error(PD_INVALID_ARGUMENT, "%s: head_dim must be 128", who);
    if (x->num_tokens < 0 || x->num_q_heads < 0 || x->num_kv_heads < 0 || x->num_q_heads > 65536 || x->num_kv_heads > 65536)
        return set_error(PD_INVALID_ARGUMENT, "%s: bad token or head count", who);
    *a = pdk::RowArgs{};
    a->q = x->q; a->k = x->k; a->v = x->v;
    a->q_stride = x->q_stride; a->k_stride = x->k_stride; a->v_stride = x->v_stride;
    a->tokens = x->num_tokens; a->hq = x->num_q_heads; a->hkv = x->num_kv_heads;
    a->q_norm = x->q_norm; a->k_norm = x->k_norm; a->eps = x->eps;
    if (unaligned16(x->q_norm) || unaligned16(x->k_norm)) return set_error(PD_INVALID_ARGUMENT, "%s: norm weights must be 16-byte aligned", who);
    if ((x->q_norm || x->k_norm) && !(x->eps >= 0.f && std::isfinite(x->eps)))
        return set_error(PD_INVALID_ARGUMENT, "%s: eps must be finite and not negative", who);
    *r = rope ? rope->args : pdk::RopeArgs{};
    if (unaligned4(x->positions)) return set_error(PD_INVALID_ARGUMENT, "%s: positions must be 4-byte aligned", who);
    if (rope && rope->args.rotary_dim) {
        if (!x->positions && !own_positions) return set_error(PD_INVALID_ARGUMENT, "%s: a rotation needs positions", who);
        if (x->positions && x->num_axes < rope->args.axes)
            return set_error(PD_INVALID_ARGUMENT, "%s: the rotation uses %d position axes, %d are given", who, rope->args.axes, x->num_axes);
        if (x->positions && x->num_axes > 1 && x->positions_stride < x->num_tokens)
            return set_error(PD_INVALID_ARGUMENT, "%s: positions_stride must be at least num_tokens", who);
        a->positions = x->positions;
        a->positions_stride = x->positions_stride;
    }
    return PD_OK;
}

// A row's units (four heads of q, k or v) go to as many warps as still fit on the SMs at once, 16 of the 20 an SM takes: one
// token goes to 12 warps instead of one, 1000 to two warps each, and from 2400 on each row to one warp, which then computes
// the row's sines once.  (A second wave costs more than longer rows: 2000 rows of 40 heads took 12.8 us with two warps each, 10.0
// with one; 600 rows 5.7 us with one each, 4.8 with four.)
void spread_rows(pdk::RowArgs* a, int kv_kinds) {
    const int units = std::max(1, (a->hq + 3) / 4 + kv_kinds * ((a->hkv + 3) / 4));
    a->warps_per_row = std::max(1, std::min(units, 148 * 16 / std::max(1, a->tokens)));
}
long long row_ctas(const pdk::RowArgs& a) {
    return (static_cast<long long>(a.tokens) * a.warps_per_row + pdk::ROWS_WARPS - 1) / pdk::ROWS_WARPS;
}

template<int SINK>
void launch_rows(int act, const pdk::RowArgs& a, const pdk::RopeArgs& r, const pdk::PageArgs& t, long long ctas, cudaStream_t stream) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>(ctas));
    cfg.blockDim = dim3(pdk::ROWS_THREADS);
    cfg.stream = stream;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    const bool halves = r.rotary_dim == 128 && !r.interleaved;
    if (act == PD_ACT_FP16) cudaLaunchKernelEx(&cfg, halves ? pdk::rows_kernel<__half, SINK, true> : pdk::rows_kernel<__half, SINK, false>, a, r, t);
    else cudaLaunchKernelEx(&cfg, halves ? pdk::rows_kernel<__nv_bfloat16, SINK, true> : pdk::rows_kernel<__nv_bfloat16, SINK, false>, a, r, t);
}

// Appends rows to the pages; `a` and `t` are complete but for the work distribution.
int launch_append(int dtype, int act, pdk::RowArgs a, const pdk::RopeArgs& r, pdk::PageArgs t, cudaStream_t stream) {
    if (a.tokens == 0) return PD_OK;
    if (dtype == PD_FP8_E4M3 && t.block_scales) {
        t.log2_block = scale_block_log2(t.page_size);
        // A window is the run of rows whose blocks one CTA writes: one row where sequences bring about one token each (all
        // blocks then start in different windows), a block's worth where they bring many.
        t.window = (t.token_begin || t.one_sequence) && a.tokens >= 8ll * t.batch ? pdk::MAX_BLOCK : 1;
        const long long windows = (a.tokens + static_cast<long long>(t.window) - 1) / t.window;
        // The 2 * hkv (head, K or V) units of a block go to the CTA's pairs of warps, or single warps where blocks get few rows.
        // Calls with few windows share a window between CTAs until there are about two per SM: with more than fit on the
        // SMs beside the q rows a second wave starts (128 sequences of one token: 5.6 us with one CTA per window, 4.6 with two,
        // 5.6 with four; 1000 tokens of one sequence: 15.0 us with one, 9.5 with four).
        const int teams = t.window == 1 ? pdk::ROWS_WARPS : pdk::ROWS_WARPS / 2;
        t.splits = static_cast<int>(std::max<long long>(1, std::min<long long>((2ll * a.hkv + teams - 1) / teams, 148 * 2 / windows)));
        const long long kv = windows * t.splits;
        spread_rows(&a, 0);
        const long long ctas = kv + (a.hq ? row_ctas(a) : 0);
        if (ctas > 0x7fffffff) return set_error(PD_LENGTH_ERROR, "append: too many tokens in one call");
        t.kv_ctas = static_cast<int>(kv);
        launch_rows<pdk::SINK_BLOCKS>(act, a, r, t, ctas, stream);
    } else {
        spread_rows(&a, 2);
        if (dtype == PD_FP16) launch_rows<pdk::SINK_FP16>(act, a, r, t, row_ctas(a), stream);
        else                  launch_rows<pdk::SINK_E4M3>(act, a, r, t, row_ctas(a), stream);
    }
    PD_CUDA(cudaGetLastError());
    return PD_OK;
}

}  // namespace

extern "C" {

int pd_scale_block_tokens(int page_size) { return page_size > 0 ? 1 << scale_block_log2(page_size) : 0; }

int pd_rope_create(int rotary_dim, const double* inv_freq, const int* axes, int interleaved, float scale, pd_rope** out) {
    if (!out) return set_error(PD_INVALID_ARGUMENT, "rope_create: null argument");
    if (rotary_dim < 16 || rotary_dim > 128 || rotary_dim % 16 != 0)
        return set_error(PD_INVALID_ARGUMENT, "rope_create: rotary_dim must be a multiple of 16 from 16 to 128");
    if (!inv_freq) return set_error(PD_INVALID_ARGUMENT, "rope_create: null frequencies");
    if (!std::isfinite(scale)) return set_error(PD_INVALID_ARGUMENT, "rope_create: scale must be finite");
    pdk::RopeArgs r{};
    r.rotary_dim = rotary_dim;
    r.interleaved = interleaved != 0;
    r.scale = scale;
    r.axes = 1;
    for (int i = 0; i < rotary_dim / 2; i++) {
        if (!std::isfinite(inv_freq[i]) || std::fabs(inv_freq[i]) > 1e6)
            return set_error(PD_INVALID_ARGUMENT, "rope_create: frequency %d is not usable", i);
        // radians per position -> turns, of which only the fraction matters; 64 bits of it
        long double turn = static_cast<long double>(inv_freq[i]) / 6.283185307179586476925286766559005768L;
        turn -= std::floor(turn);
        r.step[i] = turn >= 1.0L ? 0ull : static_cast<unsigned long long>(turn * 18446744073709551616.0L);
        const int axis = axes ? axes[i] : 0;
        if (axis < 0 || axis > 3) return set_error(PD_INVALID_ARGUMENT, "rope_create: axis %d of frequency %d is outside 0..3", axis, i);
        r.axis[i] = static_cast<unsigned char>(axis);
        r.axes = std::max(r.axes, axis + 1);
    }
    pd_rope* rope = new (std::nothrow) pd_rope();
    if (!rope) return set_error(PD_INTERNAL, "rope_create: out of host memory");
    rope->args = r;
    *out = rope;
    return PD_OK;
}

void pd_rope_destroy(pd_rope* rope) { delete rope; }

int pd_qk_norm_rope(const pd_qkv* x, const pd_rope* rope, void* q_out, long long q_out_stride, void* k_out,
                    long long k_out_stride, void* stream) {
    pdk::RowArgs a;
    pdk::RopeArgs r;
    if (int rc = fill_rows("qk_norm_rope", x, rope, false, &a, &r)) return rc;
    if (a.tokens == 0 || a.hq + a.hkv == 0) return PD_OK;
    if (int rc = check_rows("qk_norm_rope", "q", a.q, &a.q_stride, a.hq)) return rc;
    if (int rc = check_rows("qk_norm_rope", "k", a.k, &a.k_stride, a.hkv)) return rc;
    if (int rc = check_rows("qk_norm_rope", "q_out", q_out, &q_out_stride, a.hq)) return rc;
    if (int rc = check_rows("qk_norm_rope", "k_out", k_out, &k_out_stride, a.hkv)) return rc;
    if ((a.hq && q_out == a.q && q_out_stride != a.q_stride) || (a.hkv && k_out == a.k && k_out_stride != a.k_stride))
        return set_error(PD_INVALID_ARGUMENT, "qk_norm_rope: in place needs the same row stride");
    a.q_out = q_out; a.q_out_stride = q_out_stride;
    a.k_out = k_out; a.k_out_stride = k_out_stride;
    spread_rows(&a, 1);
    launch_rows<pdk::SINK_DENSE>(x->act_dtype, a, r, pdk::PageArgs{}, row_ctas(a), static_cast<cudaStream_t>(stream));
    PD_CUDA(cudaGetLastError());
    return PD_OK;
}

int pd_append_qkv(int dtype, const pd_qkv* x, const pd_rope* rope, const pd_append_target* t, void* q_out, void* stream) {
    const char* who = "append_qkv";
    if (dtype != PD_FP16 && dtype != PD_FP8_E4M3) return set_error(PD_INVALID_ARGUMENT, "unsupported KV dtype %d", dtype);
    pdk::RowArgs a;
    pdk::RopeArgs r;
    if (int rc = fill_rows(who, x, rope, true, &a, &r)) return rc;
    if (!t) return set_error(PD_INVALID_ARGUMENT, "append_qkv: null target");
    if (a.hkv == 0) return set_error(PD_INVALID_ARGUMENT, "append_qkv: num_kv_heads must be positive");
    if (t->page_size <= 0 || t->num_pages <= 0 || t->num_slots <= 0 || t->block_table_stride <= 0 || t->batch < 0)
        return set_error(PD_INVALID_ARGUMENT, "append_qkv: page_size, num_pages, num_slots and block_table_stride must be positive");
    if (a.tokens == 0 || t->batch == 0) return PD_OK;
    if (int rc = check_rows(who, "q", a.q, &a.q_stride, a.hq)) return rc;
    if (int rc = check_rows(who, "k", a.k, &a.k_stride, a.hkv)) return rc;
    if (int rc = check_rows(who, "v", a.v, &a.v_stride, a.hkv)) return rc;
    long long out_stride = 0;
    if (int rc = check_rows(who, "q_out", q_out, &out_stride, a.hq)) return rc;
    if (!t->k_cache || !t->v_cache || !t->block_table || !t->start_pos) return set_error(PD_INVALID_ARGUMENT, "append_qkv: null device pointer");
    if (unaligned16(t->k_cache) || unaligned16(t->v_cache)) return set_error(PD_INVALID_ARGUMENT, "append_qkv: pools must be 16-byte aligned");
    if (unaligned4(t->block_table) || unaligned4(t->start_pos) || unaligned4(t->token_begin) || unaligned4(t->slot_ids) ||
        unaligned4(t->d_k_scales) || unaligned4(t->d_v_scales))
        return set_error(PD_INVALID_ARGUMENT, "append_qkv: lists and scales must be 4-byte aligned");
    if (t->d_block_scales) {
        if (dtype != PD_FP8_E4M3) return set_error(PD_INVALID_ARGUMENT, "append_qkv: only an fp8 cache is quantised");
        if (t->d_k_scales || t->d_v_scales) return set_error(PD_INVALID_ARGUMENT, "append_qkv: head scales and block scales exclude each other");
        if (reinterpret_cast<uintptr_t>(t->d_block_scales) % 8 != 0) return set_error(PD_INVALID_ARGUMENT, "append_qkv: block scales must be 8-byte aligned");
    } else if (dtype == PD_FP8_E4M3 && ((!t->d_k_scales && !(t->k_scale > 0.f)) || (!t->d_v_scales && !(t->v_scale > 0.f)))) {
        return set_error(PD_INVALID_ARGUMENT, "append_qkv: fp8 scales must be positive");
    }
    pdk::PageArgs p{};
    p.k_cache = t->k_cache; p.v_cache = t->v_cache;
    p.block_table = t->block_table; p.start_pos = t->start_pos; p.token_begin = t->token_begin; p.slot_ids = t->slot_ids;
    if (dtype == PD_FP8_E4M3) {
        p.k_head_scales = t->d_k_scales; p.v_head_scales = t->d_v_scales;
        p.block_scales = t->d_block_scales;
        p.inv_k = 1.f / t->k_scale; p.inv_v = 1.f / t->v_scale;
    }
    p.table_stride = t->block_table_stride; p.num_slots = t->num_slots; p.batch = t->batch;
    p.num_pages = t->num_pages; p.page_size = t->page_size;
    if (int rc = status_word(&p.status)) return rc;
    a.q_out = q_out; a.q_out_stride = out_stride;
    return launch_append(dtype, x->act_dtype, a, r, p, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
