// mtlattn._C for PyTorch-ROCm: the thin torch binding over the C ABI of
// libmtlattn_hip.so. Replaces the reference's pybind11 module
// (src/ext.mm:784-811) with the same function names, argument names and
// defaults. Tensor checks mirror src/ext.mm:306-365 (TORCH_CHECK ->
// RuntimeError); outputs and scratch are allocated through torch's caching
// allocator; work is enqueued on the current HIP stream of the input's device
// with no host synchronisation.
#include <torch/extension.h>

#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/DeviceGuard.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>

#include <tuple>
#include <vector>

#include "../../include/mtlattn_capi.h"

namespace {

int dtype_code(at::ScalarType t) {
    switch (t) {
        case at::kFloat: return MTLATTN_DTYPE_F32;
        case at::kHalf: return MTLATTN_DTYPE_F16;
        case at::kBFloat16: return MTLATTN_DTYPE_BF16;
        default: TORCH_CHECK(false, "mtlattn: unsupported dtype ", t);
    }
    return -1;
}

void check_rc(int rc) { TORCH_CHECK(rc == MTLATTN_OK, mtlattn_last_error()); }

void* current_stream(const at::Tensor& t) {
    return (void*)at::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.device().index()).stream();
}

bool defined(const c10::optional<at::Tensor>& t) { return t.has_value() && t->defined() && t->numel() > 0; }

// q/k/v layout checks of src/ext.mm:306-331.
void check_qkv(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v) {
    TORCH_CHECK(q.is_cuda() && k.is_cuda() && v.is_cuda(), "mtlattn: q/k/v must be GPU (HIP) tensors");
    TORCH_CHECK(q.dim() == 3 && k.dim() == 3 && v.dim() == 3, "mtlattn: q/k/v must be [M, H, D]");
    const auto H = q.size(1), H_kv = k.size(1), D = q.size(2);
    TORCH_CHECK(D >= 1 && D <= 256, "mtlattn: head_dim ", D, " unsupported (expected 1..256)");
    TORCH_CHECK(v.size(1) == H_kv && k.size(2) == D && v.size(2) == D, "mtlattn: k/v head/dim shape mismatch");
    TORCH_CHECK(k.size(0) == v.size(0), "mtlattn: k/v token count mismatch");
    TORCH_CHECK(H_kv > 0 && H % H_kv == 0, "mtlattn: query heads (", H, ") must be a multiple of kv heads (", H_kv,
                ")");
    TORCH_CHECK(q.scalar_type() == k.scalar_type() && q.scalar_type() == v.scalar_type(), "mtlattn: dtype mismatch");
    dtype_code(q.scalar_type());
    for (const auto& t : {q, k, v}) {
        TORCH_CHECK((t.size(2) == 1 || t.stride(2) == 1) && (t.size(1) == 1 || t.stride(1) == D),
                    "mtlattn: inner dims must be contiguous ([M, H, D] with row-only striding)");
        TORCH_CHECK(t.get_device() == q.get_device(), "mtlattn: q/k/v must be on the same device");
    }
}

void check_cu(const at::Tensor& cu_q, const at::Tensor& cu_kv, const at::Tensor& q) {
    TORCH_CHECK(cu_q.is_cuda() && cu_kv.is_cuda(), "mtlattn: cu_seqlens must be on the GPU");
    TORCH_CHECK(cu_q.get_device() == q.get_device() && cu_kv.get_device() == q.get_device(),
                "mtlattn: cu_seqlens must be on the device of q");
    TORCH_CHECK(cu_q.scalar_type() == at::kInt && cu_kv.scalar_type() == at::kInt, "mtlattn: cu_seqlens must be int32");
    TORCH_CHECK(cu_q.dim() == 1 && cu_kv.dim() == 1 && cu_q.numel() == cu_kv.numel() && cu_q.numel() >= 2,
                "mtlattn: cu_seqlens_q/kv must both be [B+1]");
}

// lse / delta of the backward test entries: [total_q, Hq] on q's device.
void check_rowhead(const at::Tensor& t, const at::Tensor& q, const char* name) {
    TORCH_CHECK(t.is_cuda() && t.get_device() == q.get_device() && t.dim() == 2 && t.size(0) == q.size(0) &&
                    t.size(1) == q.size(1),
                "mtlattn: ", name, " must be a [total_q, H] GPU tensor");
}

int64_t row_stride(const at::Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1) * t.size(2); }

// Bias checks of src/ext.mm:348-365, plus the key-dim extent for bounds.
// Also accepted (no counterpart in the reference): a 4-D mask [B or 1,
// H or 1, Nq, max_kv] indexed by (sequence, sequence-local row), used in
// place (the SDPA adapter's dense masks).
void fill_bias(mtlattn_problem& p, const c10::optional<at::Tensor>& attn_bias, const at::Tensor& q,
               at::Tensor& keep) {
    p.bias = nullptr;
    p.bias_q_stride = p.bias_h_stride = p.bias_kv_cols = 0;
    p.bias_seq_local = 0;
    p.bias_seq_stride = p.bias_seq_rows = 0;
    if (!defined(attn_bias)) return;
    keep = *attn_bias;
    TORCH_CHECK(keep.is_cuda() && keep.get_device() == q.get_device(), "mtlattn: attn_mask must be a GPU tensor");
    TORCH_CHECK(keep.scalar_type() == at::kFloat, "mtlattn: attn_mask must be float32");
    if (keep.dim() == 4) {
        TORCH_CHECK(keep.size(0) == p.num_seqs || keep.size(0) == 1,
                    "mtlattn: a 4-D attn_mask's dim0 must be the number of sequences or 1");
        TORCH_CHECK(keep.size(1) == q.size(1) || keep.size(1) == 1, "mtlattn: attn_mask dim1 must be num_heads (",
                    q.size(1), ") or 1 (broadcast)");
        TORCH_CHECK(keep.size(2) >= 1, "mtlattn: a 4-D attn_mask needs at least one query row");
        TORCH_CHECK(keep.size(3) <= 1 || keep.stride(3) == 1, "mtlattn: attn_mask last dim must be contiguous");
        TORCH_CHECK(keep.stride(0) >= 0 && keep.stride(1) >= 0 && keep.stride(2) >= 0,
                    "mtlattn: attn_mask strides must be non-negative");
        p.bias = keep.data_ptr<float>();
        p.bias_seq_local = 1;
        p.bias_seq_stride = keep.size(0) == 1 ? 0 : keep.stride(0);
        p.bias_seq_rows = keep.size(2);
        p.bias_q_stride = keep.stride(2);
        p.bias_h_stride = keep.size(1) == 1 ? 0 : keep.stride(1);
        p.bias_kv_cols = keep.size(3);
        return;
    }
    TORCH_CHECK(keep.dim() == 3, "mtlattn: attn_mask must be [total_q, H or 1, max_kv]");
    TORCH_CHECK(keep.size(0) == q.size(0), "mtlattn: attn_mask dim0 (", keep.size(0), ") must equal total_q (",
                q.size(0), ")");
    TORCH_CHECK(keep.size(1) == q.size(1) || keep.size(1) == 1, "mtlattn: attn_mask dim1 must be num_heads (",
                q.size(1), ") or 1 (broadcast)");
    TORCH_CHECK(keep.size(2) <= 1 || keep.stride(2) == 1, "mtlattn: attn_mask last dim must be contiguous");
    p.bias = keep.data_ptr<float>();
    p.bias_q_stride = keep.stride(0);
    p.bias_h_stride = keep.size(1) == 1 ? 0 : keep.stride(1);
    p.bias_kv_cols = keep.size(2);
}

mtlattn_problem make_problem(const at::Tensor& q, const at::Tensor& k, const at::Tensor& cu_q,
                             const at::Tensor& cu_kv, int64_t max_seqlen_q, double scale, bool causal,
                             int64_t window) {
    mtlattn_problem p;
    std::memset(&p, 0, sizeof(p));
    p.dtype = dtype_code(q.scalar_type());
    p.num_seqs = (int32_t)(cu_q.numel() - 1);
    p.total_q = q.size(0);
    p.total_kv = k.size(0);
    p.num_heads_q = (int32_t)q.size(1);
    p.num_heads_kv = (int32_t)k.size(1);
    p.head_dim = (int32_t)q.size(2);
    p.max_seqlen_q = (int32_t)std::min<int64_t>(max_seqlen_q, 0x7fffffff);
    p.scale = (float)scale;
    p.causal = causal ? 1 : 0;
    p.window = window > 0 ? (int32_t)std::min<int64_t>(window, 0x7fffffff) : 0;
    p.cu_seqlens_q = cu_q.data_ptr<int32_t>();
    p.cu_seqlens_kv = cu_kv.data_ptr<int32_t>();
    return p;
}

at::Tensor workspace(int64_t bytes, const at::Tensor& like) {
    return at::empty({std::max<int64_t>(bytes, 1)}, like.options().dtype(at::kByte));
}

// _C.varlen_attention (src/ext.mm:293-489).
at::Tensor varlen_attention(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                            const at::Tensor& cu_seqlens_q, const at::Tensor& cu_seqlens_kv, int64_t max_seqlen_q,
                            double scale, bool causal, int64_t window, c10::optional<at::Tensor> lse_out,
                            c10::optional<at::Tensor> attn_bias) {
    check_qkv(q, k, v);
    check_cu(cu_seqlens_q, cu_seqlens_kv, q);
    const c10::OptionalDeviceGuard guard(q.device());
    auto cu_q = cu_seqlens_q.contiguous(), cu_kv = cu_seqlens_kv.contiguous();
    auto out = at::empty({q.size(0), q.size(1), q.size(2)}, q.options());
    float* lse = nullptr;
    if (defined(lse_out)) {
        const at::Tensor& l = *lse_out;
        TORCH_CHECK(l.is_cuda() && l.scalar_type() == at::kFloat && l.is_contiguous() && l.dim() == 2 &&
                        l.size(0) == q.size(0) && l.size(1) == q.size(1),
                    "mtlattn: lse_out must be a contiguous fp32 [total_q, H] GPU tensor");
        lse = l.data_ptr<float>();
    }
    if (q.size(0) == 0) return out;
    mtlattn_problem p = make_problem(q, k, cu_q, cu_kv, max_seqlen_q, scale, causal, window);
    at::Tensor bias_keep;
    fill_bias(p, attn_bias, q, bias_keep);
    const size_t ws_bytes = mtlattn_varlen_fwd_workspace_size(&p);
    at::Tensor ws = workspace((int64_t)ws_bytes, q);
    check_rc(mtlattn_varlen_fwd(&p, q.data_ptr(), row_stride(q), k.data_ptr(), row_stride(k), v.data_ptr(),
                                row_stride(v), out.data_ptr(), lse, ws.data_ptr(), ws_bytes, current_stream(q)));
    return out;
}

// _C.dense_attention: the SDPA adapter's [B, H, N, D] forward in place (no
// reference counterpart). None where the kernels need packed rows.
c10::optional<at::Tensor> dense_attention(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, double scale,
                                          bool causal, c10::optional<at::Tensor> lens,
                                          c10::optional<at::Tensor> attn_bias) {
    const auto B = q.size(0), H = q.size(1), N = q.size(2), D = q.size(3), Hkv = k.size(1), Nkv = k.size(2);
    if (!q.is_cuda() || k.get_device() != q.get_device() || v.get_device() != q.get_device() ||
        k.scalar_type() != q.scalar_type() || v.scalar_type() != q.scalar_type() || v.sizes() != k.sizes() ||
        k.size(0) != B || k.size(3) != D || Hkv == 0 || H % Hkv != 0)
        return c10::nullopt;
    for (const auto& t : {q, k, v})
        if (D > 1 && t.stride(3) != 1) return c10::nullopt;
    if (q.scalar_type() != at::kHalf && q.scalar_type() != at::kBFloat16) return c10::nullopt;
    const c10::OptionalDeviceGuard guard(q.device());
    mtlattn_problem p;
    std::memset(&p, 0, sizeof(p));
    p.dtype = dtype_code(q.scalar_type());
    p.num_seqs = (int32_t)B;
    p.num_heads_q = (int32_t)H;
    p.num_heads_kv = (int32_t)Hkv;
    p.head_dim = (int32_t)D;
    p.scale = (float)scale;
    p.causal = causal ? 1 : 0;
    at::Tensor bias_keep, lens_keep;
    if (defined(attn_bias) && attn_bias->dim() != 4) return c10::nullopt;
    fill_bias(p, attn_bias, q, bias_keep);
    if (lens.has_value()) {
        lens_keep = lens->contiguous();
        TORCH_CHECK(lens_keep.is_cuda() && lens_keep.scalar_type() == at::kInt && lens_keep.numel() == B,
                    "mtlattn: lens must be an int32 [B] GPU tensor");
    }
    auto out = at::empty({B, H, N, D}, q.options());
    const int rc = mtlattn_dense_fwd(&p, (int32_t)N, (int32_t)Nkv, q.data_ptr(), q.stride(0), q.stride(1), q.stride(2),
                                     k.data_ptr(), k.stride(0), k.stride(1), k.stride(2), v.data_ptr(), v.stride(0),
                                     v.stride(1), v.stride(2),
                                     lens_keep.defined() ? lens_keep.data_ptr<int32_t>() : nullptr, out.data_ptr(),
                                     current_stream(q));
    if (rc == MTLATTN_ERR_UNSUPPORTED) return c10::nullopt;
    check_rc(rc);
    return out;
}

// The backward into dQ, dK and dV: [M, H, D] tensors or slices of one packed
// tensor (heads contiguous, any row stride, dK's and dV's the same). False,
// with nothing launched, where the kernels only write contiguous gradients.
bool backward_into(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& o,
                   const at::Tensor& dout, const at::Tensor& lse, const at::Tensor& cu_seqlens_q,
                   const at::Tensor& cu_seqlens_kv, double scale, bool causal, int64_t window,
                   const c10::optional<at::Tensor>& attn_bias, at::Tensor dQ, at::Tensor dK, at::Tensor dV) {
    check_qkv(q, k, v);
    check_cu(cu_seqlens_q, cu_seqlens_kv, q);
    TORCH_CHECK(o.sizes() == q.sizes() && dout.sizes() == q.sizes(), "mtlattn: o/dout must match q's shape");
    TORCH_CHECK(o.scalar_type() == q.scalar_type() && dout.scalar_type() == q.scalar_type(),
                "mtlattn: o/dout dtype mismatch");
    check_qkv(o, dout, dout);
    TORCH_CHECK(lse.is_cuda() && lse.scalar_type() == at::kFloat && lse.is_contiguous() && lse.dim() == 2 &&
                    lse.size(0) == q.size(0) && lse.size(1) == q.size(1),
                "mtlattn: lse must be a contiguous fp32 [total_q, H] GPU tensor");
    const c10::OptionalDeviceGuard guard(q.device());
    auto cu_q = cu_seqlens_q.contiguous(), cu_kv = cu_seqlens_kv.contiguous();
    mtlattn_problem p = make_problem(q, k, cu_q, cu_kv, q.size(0), scale, causal, window);
    at::Tensor bias_keep;
    fill_bias(p, attn_bias, q, bias_keep);
    const size_t ws_bytes = mtlattn_varlen_bwd_workspace_size(&p);
    at::Tensor ws = workspace((int64_t)ws_bytes, q);
    if (!(dQ.is_contiguous() && dK.is_contiguous() && dV.is_contiguous())) {
        const int rc = mtlattn_varlen_bwd_strided(
            &p, q.data_ptr(), row_stride(q), k.data_ptr(), row_stride(k), v.data_ptr(), row_stride(v), o.data_ptr(),
            row_stride(o), dout.data_ptr(), row_stride(dout), lse.data_ptr<float>(), dQ.data_ptr(), row_stride(dQ),
            dK.data_ptr(), dV.data_ptr(), row_stride(dK), ws.data_ptr(), ws_bytes, current_stream(q));
        if (rc == MTLATTN_ERR_UNSUPPORTED) return false;
        check_rc(rc);
        return true;
    }
    check_rc(mtlattn_varlen_bwd(&p, q.data_ptr(), row_stride(q), k.data_ptr(), row_stride(k), v.data_ptr(),
                                row_stride(v), o.data_ptr(), row_stride(o), dout.data_ptr(), row_stride(dout),
                                lse.data_ptr<float>(), dQ.data_ptr(), dK.data_ptr(), dV.data_ptr(), ws.data_ptr(),
                                ws_bytes, current_stream(q)));
    return true;
}

// _C.varlen_attention_bwd (src/ext.mm:502-594).
std::tuple<at::Tensor, at::Tensor, at::Tensor> varlen_attention_bwd(
    const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& o, const at::Tensor& dout,
    const at::Tensor& lse, const at::Tensor& cu_seqlens_q, const at::Tensor& cu_seqlens_kv, double scale,
    bool causal, int64_t window, c10::optional<at::Tensor> attn_bias) {
    check_qkv(q, k, v);
    const c10::OptionalDeviceGuard guard(q.device());
    auto dQ = at::empty({q.size(0), q.size(1), q.size(2)}, q.options());
    auto dK = at::empty({k.size(0), k.size(1), k.size(2)}, k.options());
    auto dV = at::empty({v.size(0), v.size(1), v.size(2)}, v.options());
    backward_into(q, k, v, o, dout, lse, cu_seqlens_q, cu_seqlens_kv, scale, causal, window, attn_bias, dQ, dK, dV);
    return {dQ, dK, dV};
}

// The gradient of a packed qkv [M, 3, H, D], or dq and the gradient of a
// packed kv [Mkv, 2, Hkv, D], written in place (no counterpart in the
// reference, whose wrappers stack the views' gradients).
at::Tensor varlen_attention_bwd_qkvpacked(const at::Tensor& qkv, const at::Tensor& o, const at::Tensor& dout,
                                          const at::Tensor& lse, const at::Tensor& cu_seqlens, double scale,
                                          bool causal, int64_t window) {
    TORCH_CHECK(qkv.dim() == 4 && qkv.size(1) == 3, "mtlattn: qkv must be [M, 3, H, D]");
    const c10::OptionalDeviceGuard guard(qkv.device());
    const auto q = qkv.select(1, 0), k = qkv.select(1, 1), v = qkv.select(1, 2);
    auto d = at::empty(qkv.sizes(), qkv.options());
    if (backward_into(q, k, v, o, dout, lse, cu_seqlens, cu_seqlens, scale, causal, window, c10::nullopt,
                      d.select(1, 0), d.select(1, 1), d.select(1, 2)))
        return d;
    d.reset();
    const auto g = varlen_attention_bwd(q, k, v, o, dout, lse, cu_seqlens, cu_seqlens, scale, causal, window,
                                        c10::nullopt);
    return at::stack({std::get<0>(g), std::get<1>(g), std::get<2>(g)}, 1);
}

std::tuple<at::Tensor, at::Tensor> varlen_attention_bwd_kvpacked(
    const at::Tensor& q, const at::Tensor& kv, const at::Tensor& o, const at::Tensor& dout, const at::Tensor& lse,
    const at::Tensor& cu_seqlens_q, const at::Tensor& cu_seqlens_kv, double scale, bool causal, int64_t window) {
    TORCH_CHECK(kv.dim() == 4 && kv.size(1) == 2, "mtlattn: kv must be [Mkv, 2, Hkv, D]");
    const c10::OptionalDeviceGuard guard(q.device());
    const auto k = kv.select(1, 0), v = kv.select(1, 1);
    auto dQ = at::empty({q.size(0), q.size(1), q.size(2)}, q.options());
    auto d = at::empty(kv.sizes(), kv.options());
    if (backward_into(q, k, v, o, dout, lse, cu_seqlens_q, cu_seqlens_kv, scale, causal, window, c10::nullopt, dQ,
                      d.select(1, 0), d.select(1, 1)))
        return {dQ, d};
    dQ.reset();
    d.reset();
    const auto g = varlen_attention_bwd(q, k, v, o, dout, lse, cu_seqlens_q, cu_seqlens_kv, scale, causal, window,
                                        c10::nullopt);
    return {std::get<0>(g), at::stack({std::get<1>(g), std::get<2>(g)}, 1)};
}

// _C.attn_splitkv (src/ext.mm:716-773). `window` and `attn_bias` (after the
// reference's arguments) have no counterpart there: its split path takes
// neither.
at::Tensor attn_splitkv(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& cu_q_in,
                        const at::Tensor& cu_kv_in, int64_t max_seqlen_q, double scale, bool causal,
                        int64_t num_splits, int64_t window, c10::optional<at::Tensor> attn_bias) {
    check_qkv(q, k, v);
    check_cu(cu_q_in, cu_kv_in, q);
    const c10::OptionalDeviceGuard guard(q.device());
    auto cu_q = cu_q_in.contiguous(), cu_kv = cu_kv_in.contiguous();
    auto out = at::empty({q.size(0), q.size(1), q.size(2)}, q.options());
    mtlattn_problem p = make_problem(q, k, cu_q, cu_kv, max_seqlen_q, scale, causal, window);
    at::Tensor bias_keep;
    fill_bias(p, attn_bias, q, bias_keep);
    const size_t ws_bytes = mtlattn_attn_splitkv_workspace_size(&p, (int32_t)num_splits);
    at::Tensor ws = workspace((int64_t)ws_bytes, q);
    check_rc(mtlattn_attn_splitkv(&p, q.data_ptr(), row_stride(q), k.data_ptr(), row_stride(k), v.data_ptr(),
                                  row_stride(v), out.data_ptr(), nullptr, (int32_t)num_splits, ws.data_ptr(), ws_bytes,
                                  current_stream(q)));
    return out;
}

// _C.paged_decode: decode over a paged KV cache (no reference counterpart).
// k_cache / v_cache [num_pages, page_size, Hkv, D] (token rows may be
// strided; pages are page_size consecutive token rows), block_table int32
// [B, max_pages], cu_seqlens_kv the logical KV lengths.
at::Tensor paged_decode(const at::Tensor& q, const at::Tensor& k_cache, const at::Tensor& v_cache,
                        const at::Tensor& cu_seqlens_q, const at::Tensor& cu_seqlens_kv, const at::Tensor& block_table,
                        int64_t max_seqlen_q, int64_t max_seqlen_kv, double scale, bool causal, int64_t window,
                        c10::optional<at::Tensor> lse_out, c10::optional<at::Tensor> attn_bias) {
    TORCH_CHECK(q.is_cuda() && k_cache.is_cuda() && v_cache.is_cuda(), "mtlattn: q/k_cache/v_cache must be GPU tensors");
    TORCH_CHECK(q.dim() == 3, "mtlattn: q must be [M, H, D]");
    TORCH_CHECK(k_cache.dim() == 4 && v_cache.dim() == 4 && k_cache.sizes() == v_cache.sizes(),
                "mtlattn: k_cache/v_cache must both be [num_pages, page_size, Hkv, D]");
    const int64_t D = q.size(2), Hkv = k_cache.size(2), page_size = k_cache.size(1);
    TORCH_CHECK(k_cache.size(3) == D, "mtlattn: k_cache head dim must match q");
    TORCH_CHECK(Hkv > 0 && q.size(1) % Hkv == 0, "mtlattn: query heads must be a multiple of kv heads");
    TORCH_CHECK(q.scalar_type() == k_cache.scalar_type() && q.scalar_type() == v_cache.scalar_type(),
                "mtlattn: dtype mismatch");
    dtype_code(q.scalar_type());
    TORCH_CHECK((q.size(2) == 1 || q.stride(2) == 1) && (q.size(1) == 1 || q.stride(1) == D),
                "mtlattn: q inner dims must be contiguous");
    for (const auto& c : {k_cache, v_cache}) {
        TORCH_CHECK(c.stride(3) == 1 && (Hkv == 1 || c.stride(2) == D),
                    "mtlattn: cache inner dims [Hkv, D] must be contiguous");
        TORCH_CHECK(c.size(0) <= 1 || c.stride(0) == page_size * c.stride(1),
                    "mtlattn: cache pages must be page_size consecutive token rows");
        TORCH_CHECK(c.get_device() == q.get_device(), "mtlattn: q and the caches must be on the same device");
    }
    check_cu(cu_seqlens_q, cu_seqlens_kv, q);
    TORCH_CHECK(block_table.is_cuda() && block_table.get_device() == q.get_device() &&
                    block_table.scalar_type() == at::kInt && block_table.dim() == 2 &&
                    block_table.size(0) == cu_seqlens_q.numel() - 1,
                "mtlattn: block_table must be an int32 [B, max_pages] GPU tensor");
    const c10::OptionalDeviceGuard guard(q.device());
    auto cu_q = cu_seqlens_q.contiguous(), cu_kv = cu_seqlens_kv.contiguous();
    TORCH_CHECK(max_seqlen_kv >= 0 && block_table.size(1) * page_size >= max_seqlen_kv,
                "mtlattn: block_table has ", block_table.size(1), " pages of ", page_size,
                " tokens per sequence, fewer than max_seqlen_kv (", max_seqlen_kv, ")");
    // one row of block_table.size(1) entries per sequence (the kernel clamps
    // its column reads to the row stride, so the rows must be dense)
    auto bt = block_table.contiguous();
    auto out = at::empty({q.size(0), q.size(1), q.size(2)}, q.options());
    float* lse = nullptr;
    if (defined(lse_out)) {
        const at::Tensor& l = *lse_out;
        TORCH_CHECK(l.is_cuda() && l.scalar_type() == at::kFloat && l.is_contiguous() && l.dim() == 2 &&
                        l.size(0) == q.size(0) && l.size(1) == q.size(1),
                    "mtlattn: lse_out must be a contiguous fp32 [total_q, H] GPU tensor");
        lse = l.data_ptr<float>();
    }
    if (q.size(0) == 0) return out;
    mtlattn_problem p;
    std::memset(&p, 0, sizeof(p));
    p.dtype = dtype_code(q.scalar_type());
    p.num_seqs = (int32_t)(cu_q.numel() - 1);
    p.total_q = q.size(0);
    // an upper bound on the logical KV total (cu_seqlens_kv[B]) from the
    // logical lengths alone: sequences may share pages (prefix caching, beam
    // search), so the sum can exceed the cache's capacity
    p.total_kv = std::min<int64_t>((int64_t)p.num_seqs * std::max<int64_t>(max_seqlen_kv, 0), 0x7fffffff);
    p.num_heads_q = (int32_t)q.size(1);
    p.num_heads_kv = (int32_t)Hkv;
    p.head_dim = (int32_t)D;
    p.max_seqlen_q = (int32_t)std::min<int64_t>(max_seqlen_q, 0x7fffffff);
    p.scale = (float)scale;
    p.causal = causal ? 1 : 0;
    p.window = window > 0 ? (int32_t)std::min<int64_t>(window, 0x7fffffff) : 0;
    p.cu_seqlens_q = cu_q.data_ptr<int32_t>();
    p.cu_seqlens_kv = cu_kv.data_ptr<int32_t>();
    at::Tensor bias_keep;
    fill_bias(p, attn_bias, q, bias_keep);
    const size_t ws_bytes = mtlattn_paged_decode_workspace_size(&p, max_seqlen_kv);
    at::Tensor ws = workspace((int64_t)ws_bytes, q);
    const int64_t krs = k_cache.size(1) > 1 ? k_cache.stride(1) : Hkv * D;
    const int64_t vrs = v_cache.size(1) > 1 ? v_cache.stride(1) : Hkv * D;
    check_rc(mtlattn_paged_decode(&p, q.data_ptr(), row_stride(q), k_cache.data_ptr(), krs, v_cache.data_ptr(), vrs,
                                  (int32_t)page_size, k_cache.size(0), bt.data_ptr<int32_t>(), bt.stride(0),
                                  max_seqlen_kv, out.data_ptr(), lse, ws.data_ptr(), ws_bytes, current_stream(q)));
    return out;
}

// An 8-bit paged cache (no reference counterpart): codes
// [num_pages, page_size, Hkv, D] of float8_e4m3fn or int8, laid out as for
// paged_decode, and contiguous fp32 scales [num_pages, page_size / block, Hkv].
// The descriptor points into `table`, which the caller keeps.
mtlattn_cache8 make_cache8(const at::Tensor& k_cache, const at::Tensor& v_cache, const at::Tensor& k_scale,
                           const at::Tensor& v_scale, const at::Tensor& block_table, int64_t num_seqs,
                           at::Tensor& table) {
    TORCH_CHECK(k_cache.is_cuda(), "mtlattn: k_cache/v_cache must be GPU tensors");
    TORCH_CHECK(k_cache.dim() == 4 && v_cache.dim() == 4 && k_cache.sizes() == v_cache.sizes(),
                "mtlattn: k_cache/v_cache must both be [num_pages, page_size, Hkv, D]");
    TORCH_CHECK(k_cache.scalar_type() == v_cache.scalar_type() &&
                    (k_cache.scalar_type() == at::kFloat8_e4m3fn || k_cache.scalar_type() == at::kChar),
                "mtlattn: an 8-bit cache must be float8_e4m3fn or int8, keys and values alike");
    const int64_t pages = k_cache.size(0), page_size = k_cache.size(1), Hkv = k_cache.size(2), D = k_cache.size(3);
    TORCH_CHECK(pages > 0 && page_size > 0 && Hkv > 0 && D > 0, "mtlattn: empty cache");
    for (const auto& c : {k_cache, v_cache}) {
        TORCH_CHECK(c.stride(3) == 1 && (Hkv == 1 || c.stride(2) == D),
                    "mtlattn: cache inner dims [Hkv, D] must be contiguous");
        TORCH_CHECK(c.size(0) <= 1 || c.stride(0) == page_size * c.stride(1),
                    "mtlattn: cache pages must be page_size consecutive token rows");
    }
    for (const auto& t : {k_scale, v_scale})
        TORCH_CHECK(t.scalar_type() == at::kFloat && t.dim() == 3 && t.is_contiguous() && t.size(0) == pages &&
                        t.size(1) == k_scale.size(1) && t.size(1) > 0 && page_size % t.size(1) == 0 && t.size(2) == Hkv,
                    "mtlattn: k_scale/v_scale must be contiguous fp32 [num_pages, page_size / block, Hkv]");
    TORCH_CHECK(block_table.scalar_type() == at::kInt && block_table.dim() == 2 && block_table.size(0) == num_seqs &&
                    block_table.size(1) > 0,
                "mtlattn: block_table must be an int32 [B, max_pages] GPU tensor");
    for (const auto& t : {v_cache, k_scale, v_scale, block_table})
        TORCH_CHECK(t.is_cuda() && t.get_device() == k_cache.get_device(),
                    "mtlattn: the cache, its scales and the block table must be on the same device");
    table = block_table.contiguous();
    mtlattn_cache8 c;
    std::memset(&c, 0, sizeof(c));
    c.code = k_cache.scalar_type() == at::kChar ? MTLATTN_CODE_INT8 : MTLATTN_CODE_E4M3;
    c.page_size = (int32_t)std::min<int64_t>(page_size, 0x7fffffff);
    c.block = (int32_t)std::min<int64_t>(page_size / k_scale.size(1), 0x7fffffff);
    c.num_heads_kv = (int32_t)std::min<int64_t>(Hkv, 0x7fffffff);
    c.head_dim = (int32_t)std::min<int64_t>(D, 0x7fffffff);
    c.num_pages = pages;
    c.k = k_cache.data_ptr();
    c.k_row_stride = page_size > 1 ? k_cache.stride(1) : Hkv * D;
    c.v = v_cache.data_ptr();
    c.v_row_stride = page_size > 1 ? v_cache.stride(1) : Hkv * D;
    c.k_scale = k_scale.data_ptr<float>();
    c.v_scale = v_scale.data_ptr<float>();
    c.block_table = table.data_ptr<int32_t>();
    c.block_table_stride = table.size(1);
    return c;
}

// _C.paged_cache_write: rows k, v [M, Hkv, D] into an 8-bit cache, as the last
// logical tokens of their sequences.
void paged_cache_write(const at::Tensor& k, const at::Tensor& v, const at::Tensor& k_cache, const at::Tensor& v_cache,
                       const at::Tensor& k_scale, const at::Tensor& v_scale, const at::Tensor& cu_seqlens,
                       const at::Tensor& cu_seqlens_kv, const at::Tensor& block_table) {
    check_qkv(k, k, v);
    check_cu(cu_seqlens, cu_seqlens_kv, k);
    at::Tensor table;
    const mtlattn_cache8 c =
        make_cache8(k_cache, v_cache, k_scale, v_scale, block_table, cu_seqlens.numel() - 1, table);
    TORCH_CHECK(k_cache.get_device() == k.get_device(), "mtlattn: k/v and the cache must be on the same device");
    TORCH_CHECK(k.size(1) == k_cache.size(2) && k.size(2) == k_cache.size(3),
                "mtlattn: k/v heads and head dim must be the cache's");
    const c10::OptionalDeviceGuard guard(k.device());
    auto cu = cu_seqlens.contiguous(), cu_kv = cu_seqlens_kv.contiguous();
    check_rc(mtlattn_cache8_write(&c, dtype_code(k.scalar_type()), k.data_ptr(), row_stride(k), v.data_ptr(),
                                  row_stride(v), k.size(0), (int32_t)(cu.numel() - 1), cu.data_ptr<int32_t>(),
                                  cu_kv.data_ptr<int32_t>(), current_stream(k)));
}

// _C.paged_cache_read: the last logical tokens of each sequence as rows
// [total, Hkv, D] of `dtype`.
std::tuple<at::Tensor, at::Tensor> paged_cache_read(const at::Tensor& k_cache, const at::Tensor& v_cache,
                                                    const at::Tensor& k_scale, const at::Tensor& v_scale,
                                                    const at::Tensor& cu_seqlens, const at::Tensor& cu_seqlens_kv,
                                                    const at::Tensor& block_table, int64_t total,
                                                    at::ScalarType dtype) {
    const int code = dtype_code(dtype);
    check_cu(cu_seqlens, cu_seqlens_kv, k_cache);
    at::Tensor table;
    const mtlattn_cache8 c =
        make_cache8(k_cache, v_cache, k_scale, v_scale, block_table, cu_seqlens.numel() - 1, table);
    TORCH_CHECK(total >= 0, "mtlattn: total must not be negative");
    const c10::OptionalDeviceGuard guard(k_cache.device());
    auto cu = cu_seqlens.contiguous(), cu_kv = cu_seqlens_kv.contiguous();
    auto k = at::empty({total, k_cache.size(2), k_cache.size(3)}, k_cache.options().dtype(dtype));
    auto v = at::empty_like(k);
    if (total > 0)
        check_rc(mtlattn_cache8_read(&c, code, k.data_ptr(), v.data_ptr(), total, (int32_t)(cu.numel() - 1),
                                     cu.data_ptr<int32_t>(), cu_kv.data_ptr<int32_t>(), current_stream(k_cache)));
    return {k, v};
}

// Rows [M, H, D] with a free row stride.
void check_rows3(const at::Tensor& t, const char* name) {
    TORCH_CHECK(t.is_cuda(), "mtlattn: ", name, " must be a GPU (HIP) tensor");
    TORCH_CHECK(t.dim() == 3 && t.size(1) > 0 && t.size(2) >= 1 && t.size(2) <= 256, "mtlattn: ", name,
                " must be [M, H, D] with D in 1..256");
    TORCH_CHECK(t.size(0) == 0 || ((t.size(2) == 1 || t.stride(2) == 1) && (t.size(1) == 1 || t.stride(1) == t.size(2))),
                "mtlattn: inner dims must be contiguous ([M, H, D] with row-only striding)");
    dtype_code(t.scalar_type());
}

// A 16-bit paged cache [num_pages, page_size, Hkv, D] (token rows may be strided) for rows like x.
void check_cache16(const at::Tensor& k_cache, const at::Tensor& v_cache, const at::Tensor& x) {
    TORCH_CHECK(k_cache.is_cuda() && v_cache.is_cuda(), "mtlattn: k_cache/v_cache must be GPU tensors");
    TORCH_CHECK(k_cache.dim() == 4 && v_cache.dim() == 4 && k_cache.sizes() == v_cache.sizes() && k_cache.numel() > 0,
                "mtlattn: k_cache/v_cache must both be [num_pages, page_size, Hkv, D]");
    const int64_t page_size = k_cache.size(1), Hkv = k_cache.size(2), D = k_cache.size(3);
    for (const auto& c : {k_cache, v_cache}) {
        TORCH_CHECK(c.scalar_type() == x.scalar_type(), "mtlattn: dtype mismatch");
        TORCH_CHECK((D == 1 || c.stride(3) == 1) && (Hkv == 1 || c.stride(2) == D),
                    "mtlattn: cache inner dims [Hkv, D] must be contiguous");
        TORCH_CHECK(c.size(0) <= 1 || page_size <= 1 || c.stride(0) == page_size * c.stride(1),
                    "mtlattn: cache pages must be page_size consecutive token rows");
        TORCH_CHECK(c.get_device() == x.get_device(), "mtlattn: rows and caches must be on the same device");
    }
}

// The scalar part of a rotation (no reference counterpart) over q [M, Hq, D] and k
// [M, Hkv, D]. inv_freq: fp32 [R / 2] of the first R elements of a head; weights
// [D], fp32 or of the rows' type. The descriptor points into `keep`, which the
// caller keeps.
mtlattn_rotary make_rotary(const at::Tensor& k, int64_t heads_q, const c10::optional<at::Tensor>& positions,
                           const c10::optional<at::Tensor>& inv_freq, bool interleaved, double scale,
                           const c10::optional<at::Tensor>& q_weight, const c10::optional<at::Tensor>& k_weight, double eps,
                           std::vector<at::Tensor>& keep) {
    mtlattn_rotary r;
    std::memset(&r, 0, sizeof(r));
    r.dtype = dtype_code(k.scalar_type());
    r.num_heads_q = (int32_t)std::min<int64_t>(heads_q, 0x7fffffff);
    r.num_heads_kv = (int32_t)std::min<int64_t>(k.size(1), 0x7fffffff);
    r.head_dim = (int32_t)k.size(2);
    r.interleaved = interleaved ? 1 : 0;
    r.scale = (float)scale;
    r.eps = (float)eps;
    r.total = k.size(0);
    auto here = [&](const at::Tensor& t) { return t.is_cuda() && t.get_device() == k.get_device(); };
    if (defined(inv_freq)) {
        TORCH_CHECK(here(*inv_freq) && inv_freq->scalar_type() == at::kFloat && inv_freq->dim() == 1 &&
                        2 * inv_freq->numel() <= k.size(2),
                    "mtlattn: inv_freq must be an fp32 [R / 2] GPU tensor, R at most the head dim");
        keep.push_back(inv_freq->contiguous());
        r.inv_freq = keep.back().data_ptr<float>();
        r.rotary_dim = (int32_t)(2 * inv_freq->numel());
    }
    if (defined(positions)) {
        TORCH_CHECK(here(*positions) && positions->scalar_type() == at::kInt && positions->dim() == 1 &&
                        positions->numel() == k.size(0),
                    "mtlattn: positions must be an int32 [M] GPU tensor");
        keep.push_back(positions->contiguous());
        r.positions = keep.back().data_ptr<int32_t>();
    }
    const c10::optional<at::Tensor>* weights[2] = {&q_weight, &k_weight};
    for (int i = 0; i < 2; ++i) {
        if (!defined(*weights[i])) continue;
        const at::Tensor& t = **weights[i];
        TORCH_CHECK(here(t) && t.dim() == 1 && t.numel() == k.size(2) &&
                        (t.scalar_type() == at::kFloat || t.scalar_type() == k.scalar_type()),
                    "mtlattn: q_weight/k_weight must be [D] GPU tensors, fp32 or of the rows' type");
        const int code = dtype_code(t.scalar_type());
        TORCH_CHECK(i == 0 || r.q_weight == nullptr || code == r.weight_dtype,
                    "mtlattn: q_weight and k_weight must be of one type");
        r.weight_dtype = code;
        keep.push_back(t.contiguous());
        (i == 0 ? r.q_weight : r.k_weight) = keep.back().data_ptr();
    }
    return r;
}

// q and k rows of one rotation.
void check_rotated(const at::Tensor& q, const at::Tensor& k) {
    check_rows3(q, "q");
    check_rows3(k, "k");
    TORCH_CHECK(q.size(0) == k.size(0) && q.size(2) == k.size(2) && q.scalar_type() == k.scalar_type() &&
                    q.get_device() == k.get_device(),
                "mtlattn: q and k must have the same tokens, head dim, dtype and device");
}

// Rows that do not overlap (a broadcast over tokens is laid out); gradients also with
// their inner dims contiguous.
at::Tensor laid_out(const at::Tensor& t) {
    return t.size(0) > 1 && t.stride(0) < t.size(1) * t.size(2) ? t.contiguous() : t;
}
at::Tensor gradient_rows(const at::Tensor& t) {
    const bool inner = t.dim() == 3 && (t.size(2) == 1 || t.stride(2) == 1) && (t.size(1) == 1 || t.stride(1) == t.size(2));
    return inner ? laid_out(t) : t.contiguous();
}

// Tangents of forward-mode differentiation, which no entry carries on.
void check_no_tangents(const at::Tensor& q, const at::Tensor& k, const c10::optional<at::Tensor>& q_weight,
                       const c10::optional<at::Tensor>& k_weight) {
    auto has = [](const at::Tensor& t) { return t._fw_grad(/*level=*/0).defined(); };
    TORCH_CHECK_NOT_IMPLEMENTED(!has(q) && !has(k) && !(defined(q_weight) && has(*q_weight)) &&
                                    !(defined(k_weight) && has(*k_weight)),
                                "mtlattn: rotary has no forward-mode derivative (its inputs have tangents)");
}

// _C.rotary: q and k with their heads normed and rotated.
std::tuple<at::Tensor, at::Tensor> rotary(const at::Tensor& q_, const at::Tensor& k_, const at::Tensor& positions,
                                          const at::Tensor& inv_freq, bool interleaved, double scale,
                                          c10::optional<at::Tensor> q_weight, c10::optional<at::Tensor> k_weight,
                                          double eps) {
    check_no_tangents(q_, k_, q_weight, k_weight);
    check_rotated(q_, k_);
    const c10::OptionalDeviceGuard guard(q_.device());
    const auto q = laid_out(q_), k = laid_out(k_);
    std::vector<at::Tensor> keep;
    const mtlattn_rotary r =
        make_rotary(k, q.size(1), positions, inv_freq, interleaved, scale, q_weight, k_weight, eps, keep);
    auto qo = at::empty(q.sizes(), q.options()), ko = at::empty(k.sizes(), k.options());
    check_rc(mtlattn_rotary_fwd(&r, q.data_ptr(), row_stride(q), k.data_ptr(), row_stride(k), qo.data_ptr(), row_stride(qo),
                                ko.data_ptr(), row_stride(ko), current_stream(q)));
    return {qo, ko};
}

// _C.rotary_bwd: its gradients (dq, dk, dq_weight, dk_weight), the weights' undefined
// without norms. q and k: the rows with norms, else any tensors of their shapes.
std::tuple<at::Tensor, at::Tensor, c10::optional<at::Tensor>, c10::optional<at::Tensor>> rotary_bwd(
    const at::Tensor& q_, const at::Tensor& k_, const at::Tensor& dq_out_, const at::Tensor& dk_out_,
    const at::Tensor& positions, const at::Tensor& inv_freq, bool interleaved, double scale, c10::optional<at::Tensor> q_weight,
    c10::optional<at::Tensor> k_weight, double eps) {
    const c10::OptionalDeviceGuard guard(q_.device());
    const auto q = gradient_rows(q_), k = gradient_rows(k_), dq_out = gradient_rows(dq_out_), dk_out = gradient_rows(dk_out_);
    check_rotated(q, k);
    check_rotated(dq_out, dk_out);
    TORCH_CHECK(q.sizes() == dq_out.sizes() && k.sizes() == dk_out.sizes() && q.scalar_type() == dq_out.scalar_type() &&
                    q.get_device() == dq_out.get_device(),
                "mtlattn: gradients must be like q and k");
    std::vector<at::Tensor> keep;
    const mtlattn_rotary r =
        make_rotary(k, q.size(1), positions, inv_freq, interleaved, scale, q_weight, k_weight, eps, keep);
    auto dq = at::empty(q.sizes(), q.options()), dk = at::empty(k.sizes(), k.options());
    c10::optional<at::Tensor> dqw, dkw;
    if (r.q_weight != nullptr) dqw = at::empty({k.size(2)}, q_weight->options());
    if (r.k_weight != nullptr) dkw = at::empty({k.size(2)}, k_weight->options());
    const size_t ws_bytes = mtlattn_rotary_bwd_workspace_size(&r);
    at::Tensor ws = workspace((int64_t)ws_bytes, q);
    check_rc(mtlattn_rotary_bwd(&r, q.data_ptr(), row_stride(q), k.data_ptr(), row_stride(k), dq_out.data_ptr(),
                                row_stride(dq_out), dk_out.data_ptr(), row_stride(dk_out), dq.data_ptr(), row_stride(dq),
                                dk.data_ptr(), row_stride(dk), dqw ? dqw->data_ptr() : nullptr,
                                dkw ? dkw->data_ptr() : nullptr, ws_bytes ? ws.data_ptr() : nullptr, ws_bytes,
                                current_stream(q)));
    return {dq, dk, dqw, dkw};
}

// The autograd node of rotary, in C++: a Python one's backward takes the interpreter's
// lock on the engine's thread (64 tokens, forward and gradients: 85 us with that, 72
// here, of which the engine takes 45). Without norms the backward is the rotation back
// and needs nothing of the forward; with them it recomputes the norms from q and k.
struct RotaryFunction : public torch::autograd::Function<RotaryFunction> {
    static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const at::Tensor& q,
                                                  const at::Tensor& k, const at::Tensor& positions,
                                                  const at::Tensor& inv_freq, bool interleaved, double scale,
                                                  const c10::optional<at::Tensor>& q_weight,
                                                  const c10::optional<at::Tensor>& k_weight, double eps) {
        const bool normed = q_weight.has_value();
        ctx->saved_data["interleaved"] = interleaved;
        ctx->saved_data["scale"] = scale;
        ctx->saved_data["eps"] = eps;
        if (normed) ctx->save_for_backward({positions, inv_freq, q, k, *q_weight, *k_weight});
        else ctx->save_for_backward({positions, inv_freq});
        at::AutoDispatchBelowADInplaceOrView below;
        auto [qo, ko] = rotary(q, k, positions, inv_freq, interleaved, scale, q_weight, k_weight, eps);
        return {qo, ko};
    }

    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                   torch::autograd::variable_list grads) {
        const auto saved = ctx->get_saved_variables();
        const bool normed = saved.size() > 2;
        const at::Tensor &dq = grads[0], &dk = grads[1];
        c10::optional<at::Tensor> qw, kw;
        if (normed) {
            qw = saved[4];
            kw = saved[5];
        }
        torch::autograd::variable_list out(9);
        const bool again = at::GradMode::is_enabled();
        {
            at::AutoGradMode off(false);
            auto [gq, gk, gqw, gkw] = rotary_bwd(normed ? saved[2] : dq, normed ? saved[3] : dk, dq, dk, saved[0], saved[1],
                                                 ctx->saved_data["interleaved"].toBool(),
                                                 ctx->saved_data["scale"].toDouble(), qw, kw,
                                                 ctx->saved_data["eps"].toDouble());
            out[0] = gq;
            out[1] = gk;
            if (gqw) out[6] = *gqw;
            if (gkw) out[7] = *gkw;
        }
        if (again) {                    // (gradients of these would be wrong without a word: they raise)
            torch::autograd::variable_list some;
            for (auto& t : out)
                if (t.defined()) some.push_back(t.detach().set_requires_grad(true));
            const auto node = std::make_shared<torch::autograd::DelayedError>(
                "mtlattn: rotary is once_differentiable: gradients of its gradients are not supported", (int)some.size());
            some = (*node)(std::move(some));
            size_t i = 0;
            for (auto& t : out)
                if (t.defined()) t = some[i++];
        }
        return out;
    }
};

// _C.rotary_grad: rotary as a differentiable operation of q, k and the weights.
std::tuple<at::Tensor, at::Tensor> rotary_grad(const at::Tensor& q, const at::Tensor& k, const at::Tensor& positions,
                                               const at::Tensor& inv_freq, bool interleaved, double scale,
                                               c10::optional<at::Tensor> q_weight, c10::optional<at::Tensor> k_weight,
                                               double eps) {
    TORCH_CHECK(q_weight.has_value() == k_weight.has_value(), "mtlattn: q_weight and k_weight go together");
    auto out = RotaryFunction::apply(q, k, positions, inv_freq, interleaved, scale, q_weight, k_weight, eps);
    return {out[0], out[1]};
}

// _C.paged_cache_append: rows k, v [M, Hkv, D] into a 16-bit paged cache, k (and q, whose
// rows are returned) normed and rotated on the way.
c10::optional<at::Tensor> paged_cache_append(const at::Tensor& k_, const at::Tensor& v_, const at::Tensor& k_cache,
                                             const at::Tensor& v_cache, const at::Tensor& cu_seqlens,
                                             const at::Tensor& cu_seqlens_kv, const at::Tensor& block_table,
                                             c10::optional<at::Tensor> q_, c10::optional<at::Tensor> positions,
                                             c10::optional<at::Tensor> inv_freq, bool interleaved, double scale,
                                             c10::optional<at::Tensor> q_weight, c10::optional<at::Tensor> k_weight,
                                             double eps) {
    check_qkv(k_, k_, v_);
    check_cu(cu_seqlens, cu_seqlens_kv, k_);
    const bool has_q = q_.has_value() && q_->defined();
    if (has_q) check_rotated(*q_, k_);
    const c10::OptionalDeviceGuard guard(k_.device());
    const auto k = laid_out(k_), v = laid_out(v_);
    const auto q = has_q ? c10::optional<at::Tensor>(laid_out(*q_)) : c10::nullopt;
    check_cache16(k_cache, v_cache, k);
    TORCH_CHECK(k.size(1) == k_cache.size(2) && k.size(2) == k_cache.size(3),
                "mtlattn: k/v heads and head dim must be the cache's");
    TORCH_CHECK(block_table.is_cuda() && block_table.get_device() == k.get_device() &&
                    block_table.scalar_type() == at::kInt && block_table.dim() == 2 &&
                    block_table.size(0) == cu_seqlens.numel() - 1 && block_table.size(1) > 0,
                "mtlattn: block_table must be an int32 [B, max_pages] GPU tensor");
    std::vector<at::Tensor> keep;
    const mtlattn_rotary r = make_rotary(k, has_q ? q->size(1) : 0, positions, inv_freq, interleaved, scale, q_weight,
                                         k_weight, eps, keep);
    auto cu = cu_seqlens.contiguous(), cu_kv = cu_seqlens_kv.contiguous(), bt = block_table.contiguous();
    c10::optional<at::Tensor> qo;
    if (has_q) qo = at::empty(q->sizes(), q->options());
    const int64_t row = k.size(1) * k.size(2);
    check_rc(mtlattn_cache_append(&r, has_q ? q->data_ptr() : nullptr, has_q ? row_stride(*q) : 0,
                                  qo ? qo->data_ptr() : nullptr, qo ? row_stride(*qo) : 0, k.data_ptr(), row_stride(k),
                                  v.data_ptr(), row_stride(v), k_cache.data_ptr(),
                                  k_cache.size(1) > 1 ? k_cache.stride(1) : k_cache.size(0) > 1 ? k_cache.stride(0) : row,
                                  v_cache.data_ptr(),
                                  v_cache.size(1) > 1 ? v_cache.stride(1) : v_cache.size(0) > 1 ? v_cache.stride(0) : row,
                                  (int32_t)std::min<int64_t>(k_cache.size(1), 0x7fffffff), k_cache.size(0),
                                  bt.data_ptr<int32_t>(), bt.size(1), (int32_t)(cu.numel() - 1), cu.data_ptr<int32_t>(),
                                  cu_kv.data_ptr<int32_t>(), current_stream(k)));
    return qo;
}

// _C.paged_tree_decode: attention of drafted tokens' trees over a 16-bit paged cache.
at::Tensor paged_tree_decode(const at::Tensor& q, const at::Tensor& k_cache, const at::Tensor& v_cache,
                             const at::Tensor& cu_seqlens_q, const at::Tensor& cu_seqlens_kv,
                             const at::Tensor& block_table, const at::Tensor& tree_mask, int64_t max_seqlen_q,
                             int64_t max_seqlen_kv, double scale, c10::optional<at::Tensor> lse_out) {
    check_rows3(q, "q");
    check_cache16(k_cache, v_cache, q);
    const int64_t D = q.size(2), Hkv = k_cache.size(2), page_size = k_cache.size(1);
    TORCH_CHECK(k_cache.size(3) == D, "mtlattn: k_cache head dim must match q");
    TORCH_CHECK(q.size(1) % Hkv == 0, "mtlattn: query heads must be a multiple of kv heads");
    check_cu(cu_seqlens_q, cu_seqlens_kv, q);
    TORCH_CHECK(block_table.is_cuda() && block_table.get_device() == q.get_device() &&
                    block_table.scalar_type() == at::kInt && block_table.dim() == 2 &&
                    block_table.size(0) == cu_seqlens_q.numel() - 1,
                "mtlattn: block_table must be an int32 [B, max_pages] GPU tensor");
    TORCH_CHECK(max_seqlen_kv >= 0 && block_table.size(1) * page_size >= max_seqlen_kv,
                "mtlattn: block_table has ", block_table.size(1), " pages of ", page_size,
                " tokens per sequence, fewer than max_seqlen_kv (", max_seqlen_kv, ")");
    TORCH_CHECK(tree_mask.is_cuda() && tree_mask.get_device() == q.get_device() &&
                    tree_mask.scalar_type() == at::kBool && tree_mask.dim() == 2 && tree_mask.size(0) == q.size(0) &&
                    tree_mask.size(1) >= 1,
                "mtlattn: tree_mask must be a bool [total_q, T] GPU tensor");
    const c10::OptionalDeviceGuard guard(q.device());
    auto cu_q = cu_seqlens_q.contiguous(), cu_kv = cu_seqlens_kv.contiguous(), bt = block_table.contiguous();
    const auto qr = laid_out(q);
    const auto mask = tree_mask.size(1) == 1 || tree_mask.stride(1) == 1 ? tree_mask : tree_mask.contiguous();
    auto out = at::empty({q.size(0), q.size(1), D}, q.options());
    float* lse = nullptr;
    if (defined(lse_out)) {
        const at::Tensor& l = *lse_out;
        TORCH_CHECK(l.is_cuda() && l.get_device() == q.get_device() && l.scalar_type() == at::kFloat && l.is_contiguous() &&
                        l.dim() == 2 && l.size(0) == q.size(0) && l.size(1) == q.size(1),
                    "mtlattn: lse_out must be a contiguous fp32 [total_q, H] GPU tensor");
        lse = l.data_ptr<float>();
    }
    mtlattn_problem p;
    std::memset(&p, 0, sizeof(p));
    p.dtype = dtype_code(q.scalar_type());
    p.num_seqs = (int32_t)(cu_q.numel() - 1);
    p.total_q = q.size(0);
    p.num_heads_q = (int32_t)q.size(1);
    p.num_heads_kv = (int32_t)Hkv;
    p.head_dim = (int32_t)D;
    p.max_seqlen_q = (int32_t)std::max<int64_t>(std::min<int64_t>(max_seqlen_q, 0x7fffffff), -1);
    p.scale = (float)scale;
    p.cu_seqlens_q = cu_q.data_ptr<int32_t>();
    p.cu_seqlens_kv = cu_kv.data_ptr<int32_t>();
    const size_t ws_bytes = mtlattn_tree_decode_workspace_size(&p, max_seqlen_kv);
    at::Tensor ws = workspace((int64_t)ws_bytes, q);
    const int64_t row = Hkv * D;
    const int64_t krs = k_cache.size(1) > 1 ? k_cache.stride(1) : row, vrs = v_cache.size(1) > 1 ? v_cache.stride(1) : row;
    check_rc(mtlattn_tree_decode(&p, qr.data_ptr(), row_stride(qr), k_cache.data_ptr(), krs, v_cache.data_ptr(), vrs,
                                 (int32_t)std::min<int64_t>(page_size, 0x7fffffff), k_cache.size(0), bt.data_ptr<int32_t>(),
                                 bt.size(1), max_seqlen_kv, (const uint8_t*)mask.data_ptr(),
                                 mask.size(0) > 1 ? mask.stride(0) : mask.size(1),
                                 (int32_t)std::min<int64_t>(mask.size(1), 0x7fffffff), out.data_ptr(), lse, ws.data_ptr(),
                                 ws_bytes, current_stream(q)));
    return out;
}

// _C.paged_decode8: paged_decode over an 8-bit cache.
at::Tensor paged_decode8(const at::Tensor& q, const at::Tensor& k_cache, const at::Tensor& v_cache,
                         const at::Tensor& k_scale, const at::Tensor& v_scale, const at::Tensor& cu_seqlens_q,
                         const at::Tensor& cu_seqlens_kv, const at::Tensor& block_table, int64_t max_seqlen_q,
                         int64_t max_seqlen_kv, double scale, bool causal, int64_t window,
                         c10::optional<at::Tensor> lse_out, c10::optional<at::Tensor> attn_bias) {
    TORCH_CHECK(q.is_cuda(), "mtlattn: q must be a GPU tensor");
    TORCH_CHECK(q.dim() == 3, "mtlattn: q must be [M, H, D]");
    check_cu(cu_seqlens_q, cu_seqlens_kv, q);
    at::Tensor table;
    const mtlattn_cache8 c =
        make_cache8(k_cache, v_cache, k_scale, v_scale, block_table, cu_seqlens_q.numel() - 1, table);
    const int64_t D = q.size(2), Hkv = k_cache.size(2), page_size = k_cache.size(1);
    TORCH_CHECK(k_cache.size(3) == D, "mtlattn: k_cache head dim must match q");
    TORCH_CHECK(q.size(1) > 0 && q.size(1) % Hkv == 0, "mtlattn: query heads must be a multiple of kv heads");
    TORCH_CHECK((q.size(2) == 1 || q.stride(2) == 1) && (q.size(1) == 1 || q.stride(1) == D),
                "mtlattn: q inner dims must be contiguous");
    TORCH_CHECK(k_cache.get_device() == q.get_device(), "mtlattn: q and the caches must be on the same device");
    const c10::OptionalDeviceGuard guard(q.device());
    auto cu_q = cu_seqlens_q.contiguous(), cu_kv = cu_seqlens_kv.contiguous();
    TORCH_CHECK(max_seqlen_kv >= 0 && block_table.size(1) * page_size >= max_seqlen_kv,
                "mtlattn: block_table has ", block_table.size(1), " pages of ", page_size,
                " tokens per sequence, fewer than max_seqlen_kv (", max_seqlen_kv, ")");
    auto out = at::empty({q.size(0), q.size(1), D}, q.options());
    float* lse = nullptr;
    if (defined(lse_out)) {
        const at::Tensor& l = *lse_out;
        TORCH_CHECK(l.is_cuda() && l.get_device() == q.get_device() && l.scalar_type() == at::kFloat &&
                        l.is_contiguous() && l.dim() == 2 && l.size(0) == q.size(0) && l.size(1) == q.size(1),
                    "mtlattn: lse_out must be a contiguous fp32 [total_q, H] GPU tensor");
        lse = l.data_ptr<float>();
    }
    mtlattn_problem p;
    std::memset(&p, 0, sizeof(p));
    p.dtype = dtype_code(q.scalar_type());
    if (q.size(0) == 0) return out;
    p.num_seqs = (int32_t)(cu_q.numel() - 1);
    p.total_q = q.size(0);
    // What the tables hold bounds the logical KV total: a max_seqlen_kv that is too
    // small (a captured graph's, of lengths that grew) shapes the launch, no more.
    p.total_kv = std::min<int64_t>((int64_t)p.num_seqs * block_table.size(1), 0x7fffffff / page_size) * page_size;
    p.num_heads_q = (int32_t)q.size(1);
    p.num_heads_kv = (int32_t)Hkv;
    p.head_dim = (int32_t)D;
    p.max_seqlen_q = (int32_t)std::min<int64_t>(max_seqlen_q, 0x7fffffff);
    p.scale = (float)scale;
    p.causal = causal ? 1 : 0;
    p.window = window > 0 ? (int32_t)std::min<int64_t>(window, 0x7fffffff) : 0;
    p.cu_seqlens_q = cu_q.data_ptr<int32_t>();
    p.cu_seqlens_kv = cu_kv.data_ptr<int32_t>();
    at::Tensor bias_keep;
    fill_bias(p, attn_bias, q, bias_keep);
    const size_t ws_bytes = mtlattn_decode8_workspace_size(&p, max_seqlen_kv);
    at::Tensor ws = workspace((int64_t)ws_bytes, q);
    check_rc(mtlattn_decode8(&p, q.data_ptr(), row_stride(q), &c, max_seqlen_kv, out.data_ptr(), lse, ws.data_ptr(),
                             ws_bytes, current_stream(q)));
    return out;
}

// _C.mpp_bwd_dq (src/ext.mm:656-711): fp32 dQ.
at::Tensor mpp_bwd_dq(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& dO,
                      const at::Tensor& lse, const at::Tensor& delta, const at::Tensor& cu_q_in,
                      const at::Tensor& cu_kv_in, int64_t max_seqlen_q, double scale, bool causal, int64_t window,
                      c10::optional<at::Tensor> attn_bias) {
    check_qkv(q, k, v);
    check_cu(cu_q_in, cu_kv_in, q);
    TORCH_CHECK(dO.sizes() == q.sizes() && dO.scalar_type() == q.scalar_type(), "mtlattn: dO must match q");
    const c10::OptionalDeviceGuard guard(q.device());
    auto cu_q = cu_q_in.contiguous(), cu_kv = cu_kv_in.contiguous();
    auto dOc = dO.contiguous();
    check_rowhead(lse, q, "lse");
    check_rowhead(delta, q, "delta");
    auto lsec = lse.to(at::kFloat).contiguous(), deltac = delta.to(at::kFloat).contiguous();
    auto dQ = at::zeros({q.size(0), q.size(1), q.size(2)}, q.options().dtype(at::kFloat));
    mtlattn_problem p = make_problem(q, k, cu_q, cu_kv, max_seqlen_q, scale, causal, window);
    at::Tensor bias_keep;
    fill_bias(p, attn_bias, q, bias_keep);
    check_rc(mtlattn_bwd_dq(&p, q.data_ptr(), row_stride(q), k.data_ptr(), row_stride(k), v.data_ptr(),
                            row_stride(v), dOc.data_ptr(), row_stride(dOc), lsec.data_ptr<float>(),
                            deltac.data_ptr<float>(), dQ.data_ptr(), MTLATTN_DTYPE_F32, current_stream(q)));
    return dQ;
}

// _C.mpp_bwd_dkv (src/ext.mm:597-653): fp32 (dK, dV).
std::tuple<at::Tensor, at::Tensor> mpp_bwd_dkv(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                                               const at::Tensor& dO, const at::Tensor& lse, const at::Tensor& delta,
                                               const at::Tensor& cu_q_in, const at::Tensor& cu_kv_in,
                                               int64_t max_seqlen_kv, double scale, bool causal, int64_t window,
                                               c10::optional<at::Tensor> attn_bias) {
    (void)max_seqlen_kv;   // grids are sized from tensor shapes; no host sync needed
    check_qkv(q, k, v);
    check_cu(cu_q_in, cu_kv_in, q);
    TORCH_CHECK(dO.sizes() == q.sizes() && dO.scalar_type() == q.scalar_type(), "mtlattn: dO must match q");
    const c10::OptionalDeviceGuard guard(q.device());
    auto cu_q = cu_q_in.contiguous(), cu_kv = cu_kv_in.contiguous();
    auto dOc = dO.contiguous();
    check_rowhead(lse, q, "lse");
    check_rowhead(delta, q, "delta");
    auto lsec = lse.to(at::kFloat).contiguous(), deltac = delta.to(at::kFloat).contiguous();
    auto dK = at::zeros({k.size(0), k.size(1), k.size(2)}, k.options().dtype(at::kFloat));
    auto dV = at::zeros_like(dK);
    mtlattn_problem p = make_problem(q, k, cu_q, cu_kv, q.size(0), scale, causal, window);
    at::Tensor bias_keep;
    fill_bias(p, attn_bias, q, bias_keep);
    check_rc(mtlattn_bwd_dkv(&p, q.data_ptr(), row_stride(q), k.data_ptr(), row_stride(k), v.data_ptr(),
                             row_stride(v), dOc.data_ptr(), row_stride(dOc), lsec.data_ptr<float>(),
                             deltac.data_ptr<float>(), dK.data_ptr(), dV.data_ptr(), MTLATTN_DTYPE_F32,
                             current_stream(q)));
    return {dK, dV};
}

// The reference's "is the fast path usable here" probe (src/ext.mm:780-782):
// the MFMA kernels are compiled into this build for gfx950.
// SDPA key-padding adapter on the device (see mtlattn_pack_padded): x is
// dense [B, H, N, D] with D contiguous, lens int32 [B] on x's device. Returns
// the packed rows [B * N, H, D] and cu_seqlens [B + 1].
std::tuple<at::Tensor, at::Tensor> pack_padded(const at::Tensor& x_in, const at::Tensor& lens) {
    TORCH_CHECK(x_in.is_cuda() && x_in.dim() == 4, "mtlattn: pack_padded expects a [B, H, N, D] GPU tensor");
    const at::Tensor x = (x_in.size(3) == 1 || x_in.stride(3) == 1) ? x_in : x_in.contiguous();
    TORCH_CHECK(lens.is_cuda() && lens.scalar_type() == at::kInt && lens.dim() == 1 && lens.size(0) == x.size(0) &&
                    lens.get_device() == x.get_device(),
                "mtlattn: lens must be int32 [B] on the device of x");
    const c10::DeviceGuard guard(x.device());
    const auto B = x.size(0), H = x.size(1), N = x.size(2), D = x.size(3);
    auto lc = lens.contiguous();
    auto packed = at::empty({B * N, H, D}, x.options());
    auto cu = at::empty({B + 1}, lens.options());
    check_rc(mtlattn_pack_padded(dtype_code(x.scalar_type()), (int32_t)B, (int32_t)N, (int32_t)H, (int32_t)D,
                                 x.data_ptr(), x.stride(0), x.stride(1), x.stride(2), lc.data_ptr<int32_t>(),
                                 cu.data_ptr<int32_t>(), packed.data_ptr(), current_stream(x)));
    return {packed, cu};
}

// Inverse of pack_padded: packed rows [B * N, H, D] -> dense contiguous
// [B, H, N, D], zeros for padded tokens.
at::Tensor unpack_padded(const at::Tensor& packed, const at::Tensor& cu, const at::Tensor& lens, int64_t B,
                         int64_t N) {
    TORCH_CHECK(packed.is_cuda() && packed.dim() == 3 && packed.size(0) == B * N,
                "mtlattn: unpack_padded expects packed rows [B * N, H, D]");
    TORCH_CHECK(cu.scalar_type() == at::kInt && cu.numel() == B + 1 && lens.scalar_type() == at::kInt &&
                    lens.numel() == B && cu.is_cuda() && lens.is_cuda(),
                "mtlattn: cu_seqlens [B + 1] and lens [B] must be int32 GPU tensors");
    const c10::DeviceGuard guard(packed.device());
    auto pc = packed.contiguous();
    const auto H = pc.size(1), D = pc.size(2);
    auto out = at::empty({B, H, N, D}, pc.options());
    auto lc = lens.contiguous();
    auto cc = cu.contiguous();
    check_rc(mtlattn_unpack_padded(dtype_code(pc.scalar_type()), (int32_t)B, (int32_t)N, (int32_t)H, (int32_t)D,
                                   pc.data_ptr(), lc.data_ptr<int32_t>(), cc.data_ptr<int32_t>(), out.data_ptr(),
                                   out.stride(0), out.stride(1), out.stride(2), current_stream(pc)));
    return out;
}

// Whether two contiguous GPU tensors differ in any byte, into a cleared int32
// in pinned host memory, to be read after the current stream has come here.
void content_differs(const at::Tensor& a, const at::Tensor& b, const at::Tensor& flag) {
    TORCH_CHECK(a.is_cuda() && b.is_cuda() && a.get_device() == b.get_device() && a.is_contiguous() &&
                    b.is_contiguous() && a.nbytes() == b.nbytes(),
                "mtlattn: content_differs expects two contiguous tensors of one size on one GPU");
    TORCH_CHECK(flag.is_cpu() && flag.is_pinned() && flag.scalar_type() == at::kInt && flag.numel() == 1,
                "mtlattn: flag must be a pinned int32");
    const c10::DeviceGuard guard(a.device());
    check_rc(mtlattn_content_differs(a.data_ptr(), b.data_ptr(), (int64_t)a.nbytes(), flag.data_ptr<int32_t>(),
                                     current_stream(a)));
}

bool mpp_available() { return true; }

int64_t gpu_core_count() {
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess) return 0;
    return mtlattn_gpu_core_count(dev);
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
    m.def("mpp_available", &mpp_available, "True: the MFMA fast path is compiled in for gfx950");
    m.def("pack_padded", &pack_padded, "SDPA key-padding adapter: dense [B,H,N,D] -> packed rows + cu_seqlens",
          py::arg("x"), py::arg("lens"));
    m.def("unpack_padded", &unpack_padded, "Inverse of pack_padded (zeros for padded tokens)", py::arg("packed"),
          py::arg("cu_seqlens"), py::arg("lens"), py::arg("B"), py::arg("N"));
    m.def("content_differs", &content_differs, "a pinned flag set where two GPU tensors differ", py::arg("a"),
          py::arg("b"), py::arg("flag"));
    m.def("gpu_core_count", &gpu_core_count, "Compute-unit count of the current device (0 if unknown)");
    m.def("abi_version", [] { return mtlattn_abi_version(); }, "C ABI version of libmtlattn_hip.so");
    m.def("attn_splitkv", &attn_splitkv, "split-KV decode with an explicit split count (test entry)", py::arg("q"),
          py::arg("k"), py::arg("v"), py::arg("cu_q"), py::arg("cu_kv"), py::arg("max_seqlen_q"), py::arg("scale"),
          py::arg("causal"), py::arg("num_splits"), py::arg("window") = 0, py::arg("attn_bias") = c10::nullopt);
    m.def("paged_decode", &paged_decode, "decode (max_seqlen_q <= 16) over a paged KV cache", py::arg("q"),
          py::arg("k_cache"), py::arg("v_cache"), py::arg("cu_seqlens_q"), py::arg("cu_seqlens_kv"),
          py::arg("block_table"), py::arg("max_seqlen_q"), py::arg("max_seqlen_kv"), py::arg("scale"),
          py::arg("causal") = false, py::arg("window") = 0, py::arg("lse_out") = c10::nullopt,
          py::arg("attn_bias") = c10::nullopt);
    m.def("paged_cache_write", &paged_cache_write, "rows into a paged KV cache of 8-bit codes", py::arg("k"),
          py::arg("v"), py::arg("k_cache"), py::arg("v_cache"), py::arg("k_scale"), py::arg("v_scale"),
          py::arg("cu_seqlens"), py::arg("cu_seqlens_kv"), py::arg("block_table"));
    m.def("paged_cache_read", &paged_cache_read, "the last tokens of each sequence out of an 8-bit cache",
          py::arg("k_cache"), py::arg("v_cache"), py::arg("k_scale"), py::arg("v_scale"), py::arg("cu_seqlens"),
          py::arg("cu_seqlens_kv"), py::arg("block_table"), py::arg("total"), py::arg("dtype"));
    m.def("rotary", &rotary, "q and k with their heads normed and rotated", py::arg("q"), py::arg("k"),
          py::arg("positions"), py::arg("inv_freq"), py::arg("interleaved") = false, py::arg("scale") = 1.0,
          py::arg("q_weight") = py::none(), py::arg("k_weight") = py::none(), py::arg("eps") = 1e-6);
    m.def("rotary_grad", &rotary_grad, "rotary, differentiable in q, k and the weights", py::arg("q"), py::arg("k"),
          py::arg("positions"), py::arg("inv_freq"), py::arg("interleaved") = false, py::arg("scale") = 1.0,
          py::arg("q_weight") = py::none(), py::arg("k_weight") = py::none(), py::arg("eps") = 1e-6);
    m.def("rotary_bwd", &rotary_bwd, "gradients of rotary", py::arg("q"), py::arg("k"), py::arg("dq_out"),
          py::arg("dk_out"), py::arg("positions"), py::arg("inv_freq"), py::arg("interleaved") = false,
          py::arg("scale") = 1.0, py::arg("q_weight") = py::none(), py::arg("k_weight") = py::none(),
          py::arg("eps") = 1e-6);
    m.def("paged_cache_append", &paged_cache_append, "rows into a 16-bit paged KV cache, normed and rotated on the way",
          py::arg("k"), py::arg("v"), py::arg("k_cache"), py::arg("v_cache"), py::arg("cu_seqlens"),
          py::arg("cu_seqlens_kv"), py::arg("block_table"), py::arg("q") = py::none(), py::arg("positions") = py::none(),
          py::arg("inv_freq") = py::none(), py::arg("interleaved") = false, py::arg("scale") = 1.0,
          py::arg("q_weight") = py::none(), py::arg("k_weight") = py::none(), py::arg("eps") = 1e-6);
    m.def("paged_tree_decode", &paged_tree_decode, "attention of drafted tokens' trees over a paged KV cache", py::arg("q"),
          py::arg("k_cache"), py::arg("v_cache"), py::arg("cu_seqlens_q"), py::arg("cu_seqlens_kv"), py::arg("block_table"),
          py::arg("tree_mask"), py::arg("max_seqlen_q"), py::arg("max_seqlen_kv"), py::arg("scale"),
          py::arg("lse_out") = py::none());
    m.def("paged_decode8", &paged_decode8, "paged_decode over an 8-bit cache", py::arg("q"), py::arg("k_cache"),
          py::arg("v_cache"), py::arg("k_scale"), py::arg("v_scale"), py::arg("cu_seqlens_q"),
          py::arg("cu_seqlens_kv"), py::arg("block_table"), py::arg("max_seqlen_q"), py::arg("max_seqlen_kv"),
          py::arg("scale"), py::arg("causal") = false, py::arg("window") = 0, py::arg("lse_out") = c10::nullopt,
          py::arg("attn_bias") = c10::nullopt);
    m.def("mpp_bwd_dkv", &mpp_bwd_dkv, "dK/dV backward kernel, fp32 outputs (test entry)", py::arg("q"), py::arg("k"),
          py::arg("v"), py::arg("dO"), py::arg("lse"), py::arg("delta"), py::arg("cu_q"), py::arg("cu_kv"),
          py::arg("max_seqlen_kv"), py::arg("scale"), py::arg("causal") = false, py::arg("window") = 0,
          py::arg("attn_bias") = c10::nullopt);
    m.def("mpp_bwd_dq", &mpp_bwd_dq, "dQ backward kernel, fp32 output (test entry)", py::arg("q"), py::arg("k"),
          py::arg("v"), py::arg("dO"), py::arg("lse"), py::arg("delta"), py::arg("cu_q"), py::arg("cu_kv"),
          py::arg("max_seqlen_q"), py::arg("scale"), py::arg("causal") = false, py::arg("window") = 0,
          py::arg("attn_bias") = c10::nullopt);
    m.def("varlen_attention", &varlen_attention, "Fused varlen attention forward (MI355X)", py::arg("q"),
          py::arg("k"), py::arg("v"), py::arg("cu_seqlens_q"), py::arg("cu_seqlens_kv"), py::arg("max_seqlen_q"),
          py::arg("scale"), py::arg("causal") = false, py::arg("window") = 0, py::arg("lse_out") = c10::nullopt,
          py::arg("attn_bias") = c10::nullopt);
    m.def("varlen_attention_bwd", &varlen_attention_bwd, "Varlen attention backward (dQ, dK, dV)", py::arg("q"),
          py::arg("k"), py::arg("v"), py::arg("o"), py::arg("dout"), py::arg("lse"), py::arg("cu_seqlens_q"),
          py::arg("cu_seqlens_kv"), py::arg("scale"), py::arg("causal") = false, py::arg("window") = 0,
          py::arg("attn_bias") = c10::nullopt);
    m.def("varlen_attention_bwd_qkvpacked", &varlen_attention_bwd_qkvpacked, "Backward into a packed qkv gradient",
          py::arg("qkv"), py::arg("o"), py::arg("dout"), py::arg("lse"), py::arg("cu_seqlens"), py::arg("scale"),
          py::arg("causal") = false, py::arg("window") = 0);
    m.def("varlen_attention_bwd_kvpacked", &varlen_attention_bwd_kvpacked, "Backward into dq and a packed kv gradient",
          py::arg("q"), py::arg("kv"), py::arg("o"), py::arg("dout"), py::arg("lse"), py::arg("cu_seqlens_q"),
          py::arg("cu_seqlens_kv"), py::arg("scale"), py::arg("causal") = false, py::arg("window") = 0);
    m.def("dense_attention", &dense_attention, "dense [B,H,N,D] forward in place, or None (pack the rows)",
          py::arg("q"), py::arg("k"), py::arg("v"), py::arg("scale"), py::arg("causal") = false,
          py::arg("lens") = c10::nullopt, py::arg("attn_bias") = c10::nullopt);
}
