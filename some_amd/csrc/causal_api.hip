// C ABI of the causal attention operators (include/some_amd.h, "causal attention over packed clips"): argument checks + launches.
#include <cmath>
#include <cstring>
#include <string>

#include "internal.h"

namespace {

int cfail(SomeHandle* h, int code, const char* fn, const char* msg) noexcept {
    try {
        h->err = std::string(fn) + ": " + msg;
    } catch (...) {                                          // (no memory for the text: the code alone)
    }
    return code;
}
#define C_CHECK(cond, msg) do { if (!(cond)) return cfail(h, SOME_EINVAL, __func__, msg); } while (0)
#define C_TRY(expr)                                                                                      \
    do {                                                                                                 \
        const hipError_t _e = (expr);                                                                    \
        if (_e != hipSuccess) return cfail(h, SOME_EHIP, __func__, hipGetErrorString(_e));               \
    } while (0)

constexpr int64_t kMaxRows = (int64_t)1 << 29;
constexpr int64_t kMaxBlocks = ((int64_t)1 << 24) - 1;       // a launch has fewer than 2^32 threads a dimension; blocks are of 256
constexpr int kMaxHeads = 1024;

// 16-byte aligned rows and heads; a tile of 128 rows stays inside 31 bits
bool laid_out(int dtype, const Rows3& x) {
    const int64_t size = dtype == 0 ? 4 : 2;
    return (reinterpret_cast<uintptr_t>(x.p) & 15) == 0 && x.row >= 0 && x.head >= 0 && (x.row * size) % 16 == 0 && (x.head * size) % 16 == 0 &&
           x.row < ((int64_t)1 << 24) / size;
}
bool type_ok(int dtype, int head_dim) { return dtype >= 0 && dtype <= 2 && (head_dim == 64 || head_dim == 128); }
bool heads_ok(int heads, int kv_heads) { return kv_heads > 0 && heads > 0 && heads <= kMaxHeads && heads % kv_heads == 0; }

bool scale_ok(float scale) { return scale > 0.f && std::isfinite(scale * 1.4426950408889634f); }      // (the exponentials are of base 2)

const char* kType = "dtype must be SOME_DTYPE_F32, F16 or BF16 and head_dim 64 or 128";
const char* kHeadsMsg = "heads must be a multiple of kv_heads, at most 1024";
const char* kLayout = "arrays must be 16-byte aligned, strides non-negative multiples of 16 bytes, rows below 16 MiB apart";

Rows3 rows3(const void* p, int64_t row, int64_t head) { return {const_cast<void*>(p), row, head}; }

size_t dsum_bytes(int heads, int64_t q_rows) { return ((size_t)heads * q_rows * sizeof(float) + 255) / 256 * 256 + 256; }

bool fill_turns(NormRopeArgs& a, double theta, int head_dim) {
    if (!(theta > 0.0) || !std::isfinite(theta)) return false;
    // the last table of this thread (a function of these two values alone): 32 powers are 2 us of a 10 us call
    thread_local double last_theta = 0.0, table[64];
    thread_local int last_dim = 0;
    if (theta != last_theta || head_dim != last_dim) {
        for (int i = 0; i < head_dim / 2; ++i) table[i] = std::pow(theta, -2.0 * i / head_dim) / 6.283185307179586476925286766559;
        last_theta = theta;
        last_dim = head_dim;
    }
    std::memcpy(a.turns, table, sizeof(table));
    return true;
}

}  // namespace

extern "C" {

int some_op_qk_norm_rope(SomeHandle* h, int32_t dtype, int32_t head_dim, const void* q_dev, int64_t q_row, int64_t q_head, int32_t heads, const void* k_dev,
                         int64_t k_row, int64_t k_head, int32_t kv_heads, int64_t rows, const float* gamma_q_dev, const float* gamma_k_dev,
                         const void* positions_dev, int32_t positions64, double theta, float eps, void* q_out_dev, int64_t qo_row, int64_t qo_head,
                         void* k_out_dev, int64_t ko_row, int64_t ko_head, void* stream) {
    if (!h) return SOME_EINVAL;
    C_CHECK(type_ok(dtype, head_dim), kType);
    C_CHECK(heads > 0 && kv_heads > 0 && heads <= kMaxHeads && kv_heads <= kMaxHeads, "1 to 1024 heads");
    C_CHECK(rows >= 0 && rows < kMaxRows, "rows must be below 2^29");
    if (rows == 0) return SOME_OK;
    C_CHECK(q_dev && k_dev && q_out_dev && k_out_dev && gamma_q_dev && gamma_k_dev && positions_dev, "null pointer");
    NormRopeArgs a{};
    a.q = rows3(q_dev, q_row, q_head); a.k = rows3(k_dev, k_row, k_head);
    a.q_out = rows3(q_out_dev, qo_row, qo_head); a.k_out = rows3(k_out_dev, ko_row, ko_head);
    C_CHECK(laid_out(dtype, a.q) && laid_out(dtype, a.k) && laid_out(dtype, a.q_out) && laid_out(dtype, a.k_out), kLayout);
    C_CHECK(((reinterpret_cast<uintptr_t>(gamma_q_dev) | reinterpret_cast<uintptr_t>(gamma_k_dev)) & 15) == 0, "gains must be 16-byte aligned");
    C_CHECK((reinterpret_cast<uintptr_t>(positions_dev) & (positions64 ? 7 : 3)) == 0, "positions must be aligned");
    C_CHECK(eps >= 0.f && std::isfinite(eps), "eps must be finite and not negative");
    C_CHECK(fill_turns(a, theta, head_dim), "theta must be finite and positive");
    a.gamma_q = gamma_q_dev; a.gamma_k = gamma_k_dev; a.positions = positions_dev; a.positions64 = positions64;
    a.rows = rows; a.heads = heads; a.kv_heads = kv_heads; a.eps = eps;
    C_CHECK(norm_rope_blocks(rows, heads, kv_heads, head_dim) <= kMaxBlocks, "too many rows and heads for one launch");
    C_TRY(launch_norm_rope(dtype, head_dim, a, static_cast<hipStream_t>(stream)));
    return SOME_OK;
}

size_t some_train_qk_norm_rope_bytes(const SomeHandle* h, int64_t rows, int32_t heads, int32_t kv_heads, int32_t head_dim) {
    (void)h;
    if (rows < 0 || rows >= kMaxRows || heads <= 0 || kv_heads <= 0 || (head_dim != 64 && head_dim != 128)) return 256;
    const size_t n = (size_t)norm_rope_bwd_blocks(rows, heads, kv_heads, head_dim) * head_dim * sizeof(float);
    return n < 1024 ? 1024 : n;
}

int some_train_qk_norm_rope_bwd(SomeHandle* h, int32_t dtype, int32_t head_dim, const void* q_dev, int64_t q_row, int64_t q_head, int32_t heads,
                                const void* k_dev, int64_t k_row, int64_t k_head, int32_t kv_heads, int64_t rows, const float* gamma_q_dev,
                                const float* gamma_k_dev, const void* positions_dev, int32_t positions64, double theta, float eps, const void* dqo_dev,
                                int64_t dqo_row, int64_t dqo_head, const void* dko_dev, int64_t dko_row, int64_t dko_head, void* dq_dev, int64_t dq_row,
                                int64_t dq_head, void* dk_dev, int64_t dk_row, int64_t dk_head, float* dgamma_q_dev, float* dgamma_k_dev, int32_t accumulate,
                                void* scratch_dev, size_t scratch_bytes, void* stream) {
    if (!h) return SOME_EINVAL;
    C_CHECK(type_ok(dtype, head_dim), kType);
    C_CHECK(heads > 0 && kv_heads > 0 && heads <= kMaxHeads && kv_heads <= kMaxHeads, "1 to 1024 heads");
    C_CHECK(rows >= 0 && rows < kMaxRows, "rows must be below 2^29");
    C_CHECK(dgamma_q_dev && dgamma_k_dev && scratch_dev, "null pointer");
    C_CHECK(rows == 0 || (q_dev && k_dev && dqo_dev && dko_dev && dq_dev && dk_dev && gamma_q_dev && gamma_k_dev && positions_dev), "null pointer");
    NormRopeArgs a{};
    a.q = rows3(q_dev, q_row, q_head); a.k = rows3(k_dev, k_row, k_head);
    a.dq_in = rows3(dqo_dev, dqo_row, dqo_head); a.dk_in = rows3(dko_dev, dko_row, dko_head);
    a.q_out = rows3(dq_dev, dq_row, dq_head); a.k_out = rows3(dk_dev, dk_row, dk_head);
    C_CHECK(laid_out(dtype, a.q) && laid_out(dtype, a.k) && laid_out(dtype, a.dq_in) && laid_out(dtype, a.dk_in) && laid_out(dtype, a.q_out) &&
            laid_out(dtype, a.k_out), kLayout);
    C_CHECK(((reinterpret_cast<uintptr_t>(gamma_q_dev) | reinterpret_cast<uintptr_t>(gamma_k_dev)) & 15) == 0, "gains must be 16-byte aligned");
    C_CHECK(((reinterpret_cast<uintptr_t>(dgamma_q_dev) | reinterpret_cast<uintptr_t>(dgamma_k_dev)) & 3) == 0, "gain gradients must be 4-byte aligned");
    C_CHECK((reinterpret_cast<uintptr_t>(scratch_dev) & 15) == 0, "scratch must be 16-byte aligned");
    C_CHECK((reinterpret_cast<uintptr_t>(positions_dev) & (positions64 ? 7 : 3)) == 0, "positions must be aligned");
    C_CHECK(eps >= 0.f && std::isfinite(eps), "eps must be finite and not negative");
    C_CHECK(fill_turns(a, theta, head_dim), "theta must be finite and positive");
    if (scratch_bytes < some_train_qk_norm_rope_bytes(h, rows, heads, kv_heads, head_dim))
        return cfail(h, SOME_ENOMEM, __func__, "scratch too small (some_train_qk_norm_rope_bytes)");
    const uintptr_t gq = reinterpret_cast<uintptr_t>(dgamma_q_dev), gk = reinterpret_cast<uintptr_t>(dgamma_k_dev);
    C_CHECK((gq < gk ? gk - gq : gq - gk) >= head_dim * sizeof(float), "gain gradients must not overlap (they are written, or added to, at the same time)");
    a.gamma_q = gamma_q_dev; a.gamma_k = gamma_k_dev; a.positions = positions_dev; a.positions64 = positions64;
    a.partial = static_cast<float*>(scratch_dev);
    a.rows = rows; a.heads = heads; a.kv_heads = kv_heads; a.eps = eps;
    C_TRY(launch_norm_rope_bwd(dtype, head_dim, a, dgamma_q_dev, dgamma_k_dev, accumulate, static_cast<hipStream_t>(stream)));
    return SOME_OK;
}

size_t some_op_causal_attention_bytes(const SomeHandle* h, int32_t dtype, int32_t heads, int32_t kv_heads, int32_t head_dim, int32_t B, int64_t q_rows, int64_t k_rows) {
    (void)h;
    if (!heads_ok(heads, kv_heads) || head_dim <= 0 || B <= 0 || q_rows <= 0 || k_rows <= 0 || q_rows >= kMaxRows || k_rows >= kMaxRows) return 0;
    const int parts = causal_fwd_parts(dtype, q_rows, k_rows, B, heads, kv_heads);
    return parts > 1 ? (size_t)parts * q_rows * heads * (head_dim + 2) * sizeof(float) : 0;
}

size_t some_train_causal_attention_bytes(const SomeHandle* h, int32_t dtype, int32_t heads, int32_t kv_heads, int32_t head_dim, int32_t B, int64_t q_rows,
                                         int64_t k_rows) {
    (void)h;
    if (!heads_ok(heads, kv_heads) || head_dim <= 0 || B <= 0 || q_rows < 0 || k_rows < 0 || q_rows >= kMaxRows || k_rows >= kMaxRows) return 256;
    const int parts = causal_bwd_parts(q_rows, k_rows, B, heads, kv_heads);
    const size_t keys = parts > 1 ? (size_t)parts * k_rows * kv_heads * head_dim * 2 * sizeof(float) : 0;
    const size_t queries = some_op_causal_attention_bytes(h, dtype, heads, kv_heads, head_dim, B, q_rows, k_rows);
    return dsum_bytes(heads, q_rows) + (keys > queries ? keys : queries);
}

int some_op_causal_attention(SomeHandle* h, int32_t dtype, int32_t head_dim, const void* q_dev, int64_t q_row, int64_t q_head, int32_t heads,
                             const void* k_dev, int64_t k_row, int64_t k_head, const void* v_dev, int64_t v_row, int64_t v_head, int32_t kv_heads,
                             const int32_t* q_offsets_dev, const int32_t* k_offsets_dev, int32_t B, int64_t q_rows, int64_t k_rows, int32_t causal,
                             float scale, void* out_dev, int64_t o_row, int64_t o_head, void* rest_dev, float* lse_dev, void* workspace_dev,
                             size_t workspace_bytes, void* stream) {
    if (!h) return SOME_EINVAL;
    C_CHECK(type_ok(dtype, head_dim), kType);
    C_CHECK(heads_ok(heads, kv_heads), kHeadsMsg);
    C_CHECK(B >= 0 && q_rows >= 0 && k_rows >= 0 && q_rows < kMaxRows && k_rows < kMaxRows && B < kMaxRows, "clips and rows must be below 2^29");
    C_CHECK(scale_ok(scale), "scale must be positive and log2(e) times it finite");
    if (B == 0 || q_rows == 0) return SOME_OK;
    C_CHECK(q_dev && out_dev && q_offsets_dev && k_offsets_dev && (k_rows == 0 || (k_dev && v_dev)), "null pointer");
    CausalArgs a{};
    a.q = rows3(q_dev, q_row, q_head); a.k = rows3(k_dev, k_row, k_head); a.v = rows3(v_dev, v_row, v_head); a.out = rows3(out_dev, o_row, o_head);
    C_CHECK(laid_out(dtype, a.q) && laid_out(dtype, a.k) && laid_out(dtype, a.v) && laid_out(dtype, a.out), kLayout);
    C_CHECK((reinterpret_cast<uintptr_t>(rest_dev) & 15) == 0, "rest must be 16-byte aligned");
    a.rest = dtype ? rest_dev : nullptr; a.lse = lse_dev; a.q_offsets = q_offsets_dev; a.k_offsets = k_offsets_dev; a.q_rows = q_rows;
    a.B = B; a.kv_heads = kv_heads; a.group = heads / kv_heads; a.causal = causal; a.scale = scale;
    a.parts = k_rows > 0 ? causal_fwd_parts(dtype, q_rows, k_rows, B, heads, kv_heads) : 1;
    if (a.parts > 1) {
        if (!workspace_dev || workspace_bytes < some_op_causal_attention_bytes(h, dtype, heads, kv_heads, head_dim, B, q_rows, k_rows))
            return cfail(h, SOME_ENOMEM, __func__, "workspace too small (some_op_causal_attention_bytes)");
        C_CHECK((reinterpret_cast<uintptr_t>(workspace_dev) & 15) == 0, "workspace must be 16-byte aligned");
        a.part_o = static_cast<float*>(workspace_dev);
        a.part_ml = a.part_o + (int64_t)a.parts * q_rows * heads * head_dim;
    }
    C_CHECK(q_rows * a.group < 0x7fffff00ll && k_rows * a.group < (1ll << 36) && causal_fwd_blocks(a) <= kMaxBlocks, "too many rows, clips and heads for one launch");
    C_TRY(launch_causal_fwd(dtype, head_dim, a, static_cast<hipStream_t>(stream)));
    return SOME_OK;
}

int some_train_causal_attention_bwd(SomeHandle* h, int32_t dtype, int32_t head_dim, const void* q_dev, int64_t q_row, int64_t q_head, int32_t heads,
                                    const void* k_dev, int64_t k_row, int64_t k_head, const void* v_dev, int64_t v_row, int64_t v_head, int32_t kv_heads,
                                    const int32_t* q_offsets_dev, const int32_t* k_offsets_dev, int32_t B, int64_t q_rows, int64_t k_rows, int32_t causal,
                                    float scale, const void* out_dev, int64_t o_row, int64_t o_head, const void* rest_dev, const float* lse_dev,
                                    const void* dout_dev, int64_t do_row, int64_t do_head, void* dq_dev, int64_t dq_row, int64_t dq_head, void* dk_dev, int64_t dk_row,
                                    int64_t dk_head, void* dv_dev, int64_t dv_row, int64_t dv_head, void* workspace_dev, size_t workspace_bytes, void* stream) {
    if (!h) return SOME_EINVAL;
    C_CHECK(type_ok(dtype, head_dim), kType);
    C_CHECK(heads_ok(heads, kv_heads), kHeadsMsg);
    C_CHECK(B >= 0 && q_rows >= 0 && k_rows >= 0 && q_rows < kMaxRows && k_rows < kMaxRows && B < kMaxRows, "clips and rows must be below 2^29");
    C_CHECK(scale_ok(scale), "scale must be positive and log2(e) times it finite");
    if (B == 0 || (q_rows == 0 && k_rows == 0)) return SOME_OK;
    C_CHECK(q_offsets_dev && k_offsets_dev && workspace_dev, "null pointer");
    C_CHECK(q_rows == 0 || (q_dev && out_dev && lse_dev && dout_dev && dq_dev), "null pointer");
    C_CHECK(k_rows == 0 || (k_dev && v_dev && dk_dev && dv_dev), "null pointer");
    CausalBwdArgs b{};
    CausalArgs& a = b.f;
    a.q = rows3(q_dev, q_row, q_head); a.k = rows3(k_dev, k_row, k_head); a.v = rows3(v_dev, v_row, v_head); a.out = rows3(out_dev, o_row, o_head);
    b.dout = rows3(dout_dev, do_row, do_head); b.dq = rows3(dq_dev, dq_row, dq_head); b.dk = rows3(dk_dev, dk_row, dk_head); b.dv = rows3(dv_dev, dv_row, dv_head);
    C_CHECK(laid_out(dtype, a.q) && laid_out(dtype, a.k) && laid_out(dtype, a.v) && laid_out(dtype, a.out) && laid_out(dtype, b.dout) && laid_out(dtype, b.dq) &&
            laid_out(dtype, b.dk) && laid_out(dtype, b.dv), kLayout);
    C_CHECK((reinterpret_cast<uintptr_t>(rest_dev) & 15) == 0, "rest must be 16-byte aligned");
    a.rest = dtype ? const_cast<void*>(rest_dev) : nullptr; a.lse = const_cast<float*>(lse_dev); a.q_offsets = q_offsets_dev; a.k_offsets = k_offsets_dev; a.q_rows = q_rows;
    a.B = B; a.kv_heads = kv_heads; a.group = heads / kv_heads; a.causal = causal; a.scale = scale;
    a.parts = k_rows > 0 ? causal_fwd_parts(dtype, q_rows, k_rows, B, heads, kv_heads) : 1;
    b.k_rows = k_rows;
    b.parts = causal_bwd_parts(q_rows, k_rows, B, heads, kv_heads);
    if (workspace_bytes < some_train_causal_attention_bytes(h, dtype, heads, kv_heads, head_dim, B, q_rows, k_rows))
        return cfail(h, SOME_ENOMEM, __func__, "workspace too small (some_train_causal_attention_bytes)");
    C_CHECK((reinterpret_cast<uintptr_t>(workspace_dev) & 15) == 0, "workspace must be 16-byte aligned");
    b.dsum = static_cast<float*>(workspace_dev);
    b.part_q = b.part_k = reinterpret_cast<float*>(static_cast<char*>(workspace_dev) + dsum_bytes(heads, q_rows));
    b.part_v = b.part_k + (int64_t)b.parts * k_rows * kv_heads * head_dim;
    C_CHECK(q_rows * a.group < 0x7fffff00ll && k_rows * a.group < (1ll << 36) && causal_fwd_blocks(a) <= kMaxBlocks && causal_bwd_blocks(b) <= kMaxBlocks,
            "too many rows, clips and heads for one launch");
    C_TRY(launch_causal_bwd(dtype, head_dim, b, static_cast<hipStream_t>(stream)));
    return SOME_OK;
}

size_t some_op_attention_step_bytes(const SomeHandle* h, int32_t dtype, int32_t B, int32_t heads, int32_t kv_heads, int32_t head_dim, int32_t max_length) {
    (void)h;
    if (B <= 0 || !heads_ok(heads, kv_heads) || head_dim <= 0 || max_length <= 0) return 256;
    const int n = step_plan(dtype, head_dim, B, kv_heads, heads / kv_heads, max_length).chunks;
    return n > 1 ? (size_t)B * heads * n * (head_dim + 2) * sizeof(float) : 0;
}

int some_op_attention_step(SomeHandle* h, int32_t dtype, int32_t head_dim, const void* q_dev, int64_t q_row, int64_t q_head, int32_t heads,
                           const void* k_dev, int64_t k_batch, int64_t k_row, int64_t k_head, const void* v_dev, int64_t v_batch, int64_t v_row,
                           int64_t v_head, int32_t kv_heads, const int32_t* lengths_dev, int32_t B, int32_t max_length, float scale, void* out_dev,
                           int64_t o_row, int64_t o_head, void* workspace_dev, size_t workspace_bytes, void* stream) {
    if (!h) return SOME_EINVAL;
    C_CHECK(type_ok(dtype, head_dim), kType);
    C_CHECK(heads_ok(heads, kv_heads), kHeadsMsg);
    C_CHECK(B >= 0 && B <= 65535, "at most 65535 streams");
    C_CHECK(max_length >= 0 && max_length < kMaxRows, "max_length must be below 2^29");
    C_CHECK(scale_ok(scale), "scale must be positive and log2(e) times it finite");
    if (B == 0) return SOME_OK;
    C_CHECK(q_dev && out_dev && lengths_dev && (max_length == 0 || (k_dev && v_dev)), "null pointer");
    StepArgs a{};
    a.q = rows3(q_dev, q_row, q_head); a.k = rows3(k_dev, k_row, k_head); a.v = rows3(v_dev, v_row, v_head); a.out = rows3(out_dev, o_row, o_head);
    const int64_t size = dtype == 0 ? 4 : 2;
    C_CHECK(laid_out(dtype, a.q) && laid_out(dtype, a.k) && laid_out(dtype, a.v) && laid_out(dtype, a.out), kLayout);
    C_CHECK(k_batch >= 0 && v_batch >= 0 && (k_batch * size) % 16 == 0 && (v_batch * size) % 16 == 0, kLayout);
    a.k_batch = k_batch; a.v_batch = v_batch; a.lengths = lengths_dev; a.B = B; a.capacity = max_length;
    a.kv_heads = kv_heads; a.group = heads / kv_heads; a.scale = scale;
    const StepPlan plan = step_plan(dtype, head_dim, B, kv_heads, a.group, max_length);
    a.chunk = plan.chunk; a.chunks = plan.chunks;
    C_CHECK((int64_t)a.chunks * B * kv_heads * ((a.group + 31) / 32) <= kMaxBlocks, "too many streams and heads for one launch");
    if (a.chunks > 1) {
        if (!workspace_dev || workspace_bytes < some_op_attention_step_bytes(h, dtype, B, heads, kv_heads, head_dim, max_length))
            return cfail(h, SOME_ENOMEM, __func__, "workspace too small (some_op_attention_step_bytes)");
        C_CHECK((reinterpret_cast<uintptr_t>(workspace_dev) & 15) == 0, "workspace must be 16-byte aligned");
        a.part_o = static_cast<float*>(workspace_dev);
        a.part_ml = a.part_o + (int64_t)B * heads * a.chunks * head_dim;
    }
    C_TRY(launch_attention_step(dtype, head_dim, a, static_cast<hipStream_t>(stream)));
    return SOME_OK;
}

}  // extern "C"
