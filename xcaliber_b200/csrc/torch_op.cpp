// PyTorch custom-op registration of the fused MoE operator: `torch.ops.xmoe_b200.{forward, repack_gptq,
// prep_nvfp4_sf, build_info}`, and of the operators around FP8 experts (permute .. fp8_grouped_matmul below: they write
// into tensors of the caller, ops.py and fp8.py allocate). This is the vLLM-facing counterpart of the reference's torch extension module
// (xFused-XXXX-Kernels/xMoE/xW4A16/sm75/xR64/vllm/csrc/xr64_abs_bridge.cu:61-242: `_C.forward`,
// `_C.repack_gptq`, `_C.build_info`), registered through TORCH_LIBRARY instead of pybind11 so that the
// dispatcher, torch.compile (through the Meta kernels below) and CUDA-graph capture see a real operator
// rather than an opaque Python call. It contains no compute: every op checks its tensors the way the
// reference's bridge does (device, dtype, contiguity, shapes), allocates output and scratch with torch's
// allocator (as xr64_abs_bridge.cu:160-173 does; the caching allocator makes that capture-safe) and calls
// the C ABI of libxmoe_b200.so on the current stream.
#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/library.h>

#include <string>
#include <vector>

#include "../../include/xmoe_b200.h"

namespace {

void check_cuda_contig(const at::Tensor& t, const at::Tensor& like, const char* name) {
    TORCH_CHECK(t.is_cuda() && t.is_contiguous(), name, " must be a contiguous CUDA tensor");
    TORCH_CHECK(t.device() == like.device(), name, " must live on the same device as x");
}

// cfg_ints: hidden, inter, num_experts, top_k, num_shared_experts, scoring, renormalize, n_group, topk_group,
//           activation, act_topk_keep, token_tile (the int fields of xmoe_config, in order)
// cfg_floats: routed_scale, swiglu_alpha, swiglu_limit
xmoe_config make_cfg(at::IntArrayRef ci, at::ArrayRef<double> cf) {
    TORCH_CHECK(ci.size() == 12 && cf.size() == 3, "cfg_ints needs 12 entries and cfg_floats 3");
    xmoe_config c;
    int32_t* p = &c.hidden;
    for (int i = 0; i < 12; ++i) p[i] = (int32_t)ci[i];
    c.routed_scale = (float)cf[0];
    c.swiglu_alpha = (float)cf[1];
    c.swiglu_limit = (float)cf[2];
    return c;
}

const void* opt_ptr(const c10::optional<at::Tensor>& t) { return t.has_value() && t->defined() ? t->data_ptr() : nullptr; }

at::Tensor forward_cuda(const at::Tensor& x, const at::Tensor& router_logits,
                        const c10::optional<at::Tensor>& per_expert_scale, const at::Tensor& w13_packed,
                        const at::Tensor& w13_sf, const at::Tensor& w13_gs, const at::Tensor& w2_q,
                        const at::Tensor& w2_scale, const c10::optional<at::Tensor>& router_bias,
                        const c10::optional<at::Tensor>& sigmoid_lut, at::IntArrayRef cfg_ints,
                        at::ArrayRef<double> cfg_floats) {
    TORCH_CHECK(x.is_cuda() && x.is_contiguous() && x.dim() == 2, "x must be a contiguous CUDA tensor [N, H]");
    TORCH_CHECK(x.scalar_type() == at::kBFloat16 || x.scalar_type() == at::kHalf, "x must be bf16 or fp16");
    c10::cuda::CUDAGuard guard(x.device());
    const xmoe_config cfg = make_cfg(cfg_ints, cfg_floats);
    check_cuda_contig(router_logits, x, "router_logits");
    check_cuda_contig(w13_packed, x, "w13_packed");
    check_cuda_contig(w13_sf, x, "w13_sf");
    check_cuda_contig(w13_gs, x, "w13_gs");
    check_cuda_contig(w2_q, x, "w2_q");
    check_cuda_contig(w2_scale, x, "w2_scale");
    const int64_t n = x.size(0), h = x.size(1);
    const int64_t e_tot = (int64_t)cfg.num_experts + cfg.num_shared_experts;
    TORCH_CHECK(h == cfg.hidden, "x must be [N, hidden]");
    TORCH_CHECK(router_logits.dim() == 2 && router_logits.size(0) == n && router_logits.size(1) == cfg.num_experts,
                "router_logits must be [N, num_experts]");
    TORCH_CHECK(w13_packed.scalar_type() == at::kByte && w13_packed.dim() == 3 && w13_packed.size(0) == e_tot &&
                    w13_packed.size(1) == 2 * (int64_t)cfg.inter && w13_packed.size(2) == h / 2,
                "w13_packed must be u8 [E_tot, 2I, H/2]");
    TORCH_CHECK(w13_gs.scalar_type() == at::kFloat && w13_gs.numel() == 2 * e_tot, "w13_gs must be f32 [E_tot, 2]");
    TORCH_CHECK(w2_q.scalar_type() == at::kInt && w2_q.dim() == 3 && w2_q.size(0) == e_tot && w2_q.size(1) == h &&
                    w2_q.size(2) == cfg.inter / 8,
                "w2_q must be i32 [E_tot, H, I/8] (repack_gptq output)");
    TORCH_CHECK(w2_scale.scalar_type() == at::kBFloat16 && w2_scale.dim() == 3 && w2_scale.size(0) == e_tot &&
                    w2_scale.size(1) == (cfg.inter + 127) / 128 && w2_scale.size(2) == h,
                "w2_scale must be bf16 [E_tot, ceil(I/128), H]");
    TORCH_CHECK((int64_t)w13_sf.numel() * (int64_t)w13_sf.element_size() ==
                    (int64_t)xmoe_nvfp4_sf_bytes((int32_t)(2 * e_tot), cfg.inter, cfg.hidden),
                "w13_sf must be the output of prep_nvfp4_sf");
    if (per_expert_scale.has_value() && per_expert_scale->defined()) {
        check_cuda_contig(*per_expert_scale, x, "per_expert_scale");
        TORCH_CHECK(per_expert_scale->scalar_type() == at::kBFloat16 && per_expert_scale->numel() == cfg.num_experts,
                    "per_expert_scale must be bf16 [num_experts]");
    }
    if (router_bias.has_value() && router_bias->defined()) {
        check_cuda_contig(*router_bias, x, "router_bias");
        TORCH_CHECK(router_bias->scalar_type() == at::kFloat && router_bias->numel() == cfg.num_experts,
                    "router_bias must be f32 [num_experts]");
    }
    if (sigmoid_lut.has_value() && sigmoid_lut->defined()) {
        check_cuda_contig(*sigmoid_lut, x, "sigmoid_lut");
        TORCH_CHECK(sigmoid_lut->scalar_type() == at::kFloat && sigmoid_lut->numel() == 65536,
                    "sigmoid_lut must be f32 [65536]");
    }
    if (n == 0) return at::empty_like(x);
    // fp16 callers are served in bf16 like the reference's bridge (xr64_abs_bridge.cu:127-137)
    const at::Tensor xb = x.scalar_type() == at::kBFloat16 ? x : x.to(at::kBFloat16);
    const at::Tensor lb =
        router_logits.scalar_type() == at::kBFloat16 ? router_logits : router_logits.to(at::kBFloat16).contiguous();
    const size_t ws_bytes = xmoe_workspace_bytes(&cfg, (int32_t)n);
    TORCH_CHECK(ws_bytes > 0, "unsupported MoE configuration");
    at::Tensor raw = at::empty({(int64_t)ws_bytes + 1024}, x.options().dtype(at::kByte));
    uint8_t* ws = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw.data_ptr()) + 1023) & ~(uintptr_t)1023);
    at::Tensor y = at::empty_like(xb);
    xmoe_weights w;
    w.w13_packed = w13_packed.data_ptr();
    w.w13_sf = w13_sf.data_ptr();
    w.w13_gs = w13_gs.data_ptr<float>();
    w.w2_q = w2_q.data_ptr();
    w.w2_scale = w2_scale.data_ptr();
    w.router_bias = static_cast<const float*>(opt_ptr(router_bias));
    w.expert_scale = opt_ptr(per_expert_scale);
    w.sigmoid_lut = static_cast<const float*>(opt_ptr(sigmoid_lut));
    const int rc = xmoe_forward(&cfg, &w, xb.data_ptr(), lb.data_ptr(), (int32_t)n, y.data_ptr(), ws, ws_bytes,
                                c10::cuda::getCurrentCUDAStream(x.get_device()).stream());
    TORCH_CHECK(rc == XMOE_OK, "xmoe_forward: ", xmoe_status_string(rc));
    return x.scalar_type() == at::kBFloat16 ? y : y.to(x.scalar_type());
}

at::Tensor forward_meta(const at::Tensor& x, const at::Tensor&, const c10::optional<at::Tensor>&, const at::Tensor&,
                        const at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&,
                        const c10::optional<at::Tensor>&, const c10::optional<at::Tensor>&, at::IntArrayRef,
                        at::ArrayRef<double>) {
    return at::empty_like(x);
}

at::Tensor repack_gptq_cuda(const at::Tensor& qweight) {
    TORCH_CHECK(qweight.is_cuda() && qweight.is_contiguous() && qweight.scalar_type() == at::kInt && qweight.dim() == 3,
                "qweight must be a contiguous CUDA int32 tensor [E, K/8, O]");
    c10::cuda::CUDAGuard guard(qweight.device());
    const int64_t e = qweight.size(0), k8 = qweight.size(1), o = qweight.size(2);
    at::Tensor out = at::empty({e, o, k8}, qweight.options());
    const int rc = xmoe_repack_gptq(qweight.data_ptr(), out.data_ptr(), (int32_t)e, (int32_t)(k8 * 8), (int32_t)o,
                                    c10::cuda::getCurrentCUDAStream(qweight.get_device()).stream());
    TORCH_CHECK(rc == XMOE_OK, "xmoe_repack_gptq: ", xmoe_status_string(rc));
    return out;
}
at::Tensor repack_gptq_meta(const at::Tensor& q) { return at::empty({q.size(0), q.size(2), q.size(1)}, q.options()); }

at::Tensor prep_nvfp4_sf_cuda(const at::Tensor& scale, int64_t rows_per_mat) {
    TORCH_CHECK(scale.is_cuda() && scale.is_contiguous() && scale.element_size() == 1 && scale.dim() >= 2,
                "scale must be a contiguous CUDA tensor of E4M3 bytes [..., rows, K/16]");
    c10::cuda::CUDAGuard guard(scale.device());
    const int64_t k = scale.size(-1) * 16;
    TORCH_CHECK(rows_per_mat > 0 && scale.numel() % (rows_per_mat * scale.size(-1)) == 0, "rows_per_mat does not divide the tensor");
    const int64_t n_mats = scale.numel() / (rows_per_mat * scale.size(-1));
    const size_t bytes = xmoe_nvfp4_sf_bytes((int32_t)n_mats, (int32_t)rows_per_mat, (int32_t)k);
    at::Tensor out = at::empty({(int64_t)bytes}, scale.options().dtype(at::kByte));
    const int rc = xmoe_prep_nvfp4_sf(scale.data_ptr(), out.data_ptr(), (int32_t)n_mats, (int32_t)rows_per_mat, (int32_t)k,
                                      c10::cuda::getCurrentCUDAStream(scale.get_device()).stream());
    TORCH_CHECK(rc == XMOE_OK, "xmoe_prep_nvfp4_sf: ", xmoe_status_string(rc));
    return out;
}
at::Tensor prep_nvfp4_sf_meta(const at::Tensor& scale, int64_t rows_per_mat) {
    const int64_t n_mats = scale.numel() / (rows_per_mat * scale.size(-1));
    return at::empty({(int64_t)xmoe_nvfp4_sf_bytes((int32_t)n_mats, (int32_t)rows_per_mat, (int32_t)(scale.size(-1) * 16))},
                     scale.options().dtype(at::kByte));
}

std::string build_info() { return xmoe_build_info(); }

// ---- operators around FP8 experts: each checks its tensors, makes their device current and enqueues on its stream ----
int32_t elem_type(const at::Tensor& t, const char* name) {
    switch (t.scalar_type()) {
        case at::kBFloat16: return XMOE_BF16;
        case at::kHalf: return XMOE_FP16;
        case at::kFloat: return XMOE_FP32;
        default: TORCH_CHECK(false, name, " must be bf16, fp16 or fp32");
    }
}
void check_matrix(const at::Tensor& t, const at::Tensor& like, const char* name) {
    check_cuda_contig(t, like, name);
    TORCH_CHECK(t.dim() == 2, name, " must be a matrix");
}
int32_t i32(int64_t v, const char* name) {
    TORCH_CHECK(v >= 0 && v <= 0x7fffffff, name, " is beyond 32 bits");
    return (int32_t)v;
}
void check_rc(int rc, const char* what) { TORCH_CHECK(rc == XMOE_OK, what, ": ", xmoe_status_string(rc)); }
// Marks a tensor of the caller as changed, so that autograd refuses a backward pass through a value saved before the write.
void written(const at::Tensor& t) {
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}
xmoe_stream_t stream_of(const at::Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.get_device()).stream(); }

// topk_row i32 [N, k], rows of any stride
int32_t check_plan(const at::Tensor& plan, int64_t n, const at::Tensor& like) {
    TORCH_CHECK(plan.is_cuda() && plan.device() == like.device() && plan.scalar_type() == at::kInt && plan.dim() == 2 &&
                    plan.size(0) == n && (plan.size(1) <= 1 || plan.stride(1) == 1),
                "topk_row must be an int32 CUDA tensor [N, k] with contiguous rows, on the device of the other tensors");
    return i32(n > 1 ? plan.stride(0) : plan.size(1), "topk_row's stride");
}
struct SlotWeights { const void* p = nullptr; int32_t type = 0, stride = 0; };
SlotWeights check_weights(const c10::optional<at::Tensor>& w, const at::Tensor& plan) {
    SlotWeights r;
    if (!w.has_value() || !w->defined()) return r;
    TORCH_CHECK(w->is_cuda() && w->device() == plan.device() && w->sizes() == plan.sizes() &&
                    (w->size(1) <= 1 || w->stride(1) == 1) &&
                    (w->scalar_type() == at::kBFloat16 || w->scalar_type() == at::kFloat),
                "weights must be a bf16 or fp32 CUDA tensor of topk_row's shape with contiguous rows");
    r.p = w->data_ptr();
    r.type = elem_type(*w, "weights");
    r.stride = i32(w->size(0) > 1 ? w->stride(0) : w->size(1), "the weights' stride");
    return r;
}

void permute_cuda(const at::Tensor& x, const at::Tensor& topk_row, at::Tensor& rows) {
    check_matrix(x, x, "x");
    check_matrix(rows, x, "rows");
    const int32_t ld = check_plan(topk_row, x.size(0), x);
    TORCH_CHECK(rows.scalar_type() == x.scalar_type() && rows.size(1) == x.size(1), "rows must have x's type and width");
    written(rows);
    if (x.numel() == 0 || rows.numel() == 0 || topk_row.numel() == 0) return;
    c10::cuda::CUDAGuard guard(x.device());
    check_rc(xmoe_permute(x.data_ptr(), topk_row.data_ptr<int32_t>(), i32(x.size(0), "N"), i32(x.size(1), "hidden"),
                          i32(topk_row.size(1), "k"), ld, i32(rows.size(0), "rows"), elem_type(x, "x"), rows.data_ptr(),
                          stream_of(x)),
             "xmoe_permute");
}

void unpermute_cuda(const at::Tensor& rows, const at::Tensor& topk_row, const c10::optional<at::Tensor>& weights,
                    at::Tensor& y) {
    check_matrix(rows, rows, "rows");
    check_matrix(y, rows, "y");
    const int32_t ld = check_plan(topk_row, y.size(0), rows);
    const SlotWeights w = check_weights(weights, topk_row);
    TORCH_CHECK(rows.scalar_type() == y.scalar_type() && rows.size(1) == y.size(1), "y must have the rows' type and width");
    written(y);
    if (y.numel() == 0) return;
    c10::cuda::CUDAGuard guard(rows.device());
    check_rc(xmoe_unpermute(rows.data_ptr(), topk_row.data_ptr<int32_t>(), w.p, w.type, w.stride, i32(y.size(0), "N"),
                            i32(y.size(1), "hidden"), i32(topk_row.size(1), "k"), ld, i32(rows.size(0), "rows"),
                            elem_type(rows, "rows"), y.data_ptr(), stream_of(rows)),
             "xmoe_unpermute");
}

// Forms that allocate their result: for decode-sized calls the allocation in Python costs as much as the kernel.
at::Tensor unpermute_new_cuda(const at::Tensor& rows, const at::Tensor& topk_row, const c10::optional<at::Tensor>& weights) {
    TORCH_CHECK(rows.dim() == 2 && topk_row.dim() == 2, "rows and topk_row must be matrices");
    at::Tensor y = at::empty({topk_row.size(0), rows.size(1)}, rows.options());
    unpermute_cuda(rows, topk_row, weights, y);
    return y;
}

void unpermute_backward_cuda(const at::Tensor& dy, const at::Tensor& rows, const at::Tensor& topk_row,
                             const c10::optional<at::Tensor>& weights, at::Tensor& drows, at::Tensor& dw) {
    check_matrix(dy, dy, "dy");
    check_matrix(rows, dy, "rows");
    check_matrix(drows, dy, "drows");
    check_matrix(dw, dy, "dw");
    const int32_t ld = check_plan(topk_row, dy.size(0), dy);
    const SlotWeights w = check_weights(weights, topk_row);
    TORCH_CHECK(rows.scalar_type() == dy.scalar_type() && rows.size(1) == dy.size(1), "rows must have dy's type and width");
    TORCH_CHECK(drows.scalar_type() == dy.scalar_type() && drows.sizes() == rows.sizes(), "drows must be like rows");
    TORCH_CHECK(dw.scalar_type() == at::kFloat && dw.sizes() == topk_row.sizes(), "dw must be fp32 [N, k]");
    written(drows);
    written(dw);
    if (dw.numel() == 0) return;
    if (dy.size(1) == 0) {
        dw.zero_();
        return;
    }
    c10::cuda::CUDAGuard guard(dy.device());
    check_rc(xmoe_unpermute_backward(dy.data_ptr(), rows.data_ptr(), topk_row.data_ptr<int32_t>(), w.p, w.type, w.stride,
                                     i32(dy.size(0), "N"), i32(dy.size(1), "hidden"), i32(topk_row.size(1), "k"), ld,
                                     i32(rows.size(0), "rows"), elem_type(dy, "dy"), drows.data_ptr(), dw.data_ptr<float>(),
                                     stream_of(dy)),
             "xmoe_unpermute_backward");
}

// Codes [rows, cols] whose rows start at multiples of 16 bytes; returns the distance of two rows.
int32_t check_codes(const at::Tensor& q, const at::Tensor& like, const char* name) {
    const int64_t d = q.dim(), cols = q.size(d - 1), rows = q.size(d - 2);
    TORCH_CHECK(q.is_cuda() && q.device() == like.device() && q.scalar_type() == at::kFloat8_e4m3fn, name,
                " must be a float8_e4m3fn CUDA tensor on the device of the other tensors");
    TORCH_CHECK((cols <= 1 || q.stride(d - 1) == 1) && (rows <= 1 || (q.stride(d - 2) % 16 == 0 && q.stride(d - 2) >= cols)) &&
                    (reinterpret_cast<uintptr_t>(q.data_ptr()) & 15u) == 0,
                name, "'s rows must be contiguous and start at multiples of 16 bytes (as fp8.quant lays them out)");
    return i32(rows > 1 ? q.stride(d - 2) : (cols + 15) / 16 * 16, "the codes' row stride");
}
// Scales [rows, blocks] laid out block-major (stride (1, ld), ld a multiple of 4); returns ld, or -1 for another layout.
int64_t scale_ld(const at::Tensor& s) {
    const int64_t rows = s.size(0), blocks = s.size(1);
    if (reinterpret_cast<uintptr_t>(s.data_ptr()) & 15u) return -1;
    if (rows > 1 && s.stride(0) != 1) return -1;
    // each block's row is read to a multiple of 4: the last one's end must still belong to the storage
    const int64_t up = (rows + 3) / 4 * 4, ld = blocks <= 1 ? up : s.stride(1);
    if (ld % 4 || ld < rows) return -1;
    const int64_t end = s.storage_offset() + (blocks - 1) * ld + up;
    return end * 4 <= (int64_t)s.storage().nbytes() ? ld : -1;
}
at::Tensor block_major(const at::Tensor& s) {
    at::Tensor room = at::empty({s.size(1), (s.size(0) + 3) / 4 * 4}, s.options());
    at::Tensor t = room.narrow(1, 0, s.size(0)).t();
    t.copy_(s);
    return room;
}
int64_t blocks_of(int64_t cols) { return (cols + 127) / 128; }

int32_t check_scale_out(const at::Tensor& s, int64_t rows, int64_t cols, const at::Tensor& like) {
    TORCH_CHECK(s.is_cuda() && s.device() == like.device() && s.scalar_type() == at::kFloat && s.dim() == 2 &&
                    s.size(0) == rows && s.size(1) == blocks_of(cols),
                "scale must be fp32 [rows, ceil(cols / 128)]");
    if (rows == 0) return 0;  // nothing will be written
    const int64_t ld = scale_ld(s);
    TORCH_CHECK(ld >= 0, "scale must be laid out block-major: strides (1, multiple of 4), 16-byte aligned (as fp8.quant lays it out)");
    return i32(ld, "the scales' stride");
}

void fp8_quant_cuda(const at::Tensor& x, const c10::optional<at::Tensor>& topk_row, at::Tensor& q, at::Tensor& scale) {
    TORCH_CHECK(x.is_cuda() && x.dim() == 2 && x.size(1) > 0 && (x.size(1) == 1 || x.stride(1) == 1) &&
                    (x.size(0) <= 1 || x.stride(0) >= x.size(1)),
                "x must be a CUDA matrix with contiguous rows");
    const bool sorted = topk_row.has_value() && topk_row->defined();
    TORCH_CHECK(q.dim() == 2 && q.size(1) == x.size(1) && (sorted || q.size(0) == x.size(0)), "codes must be [rows, cols] like x");
    const int32_t ldq = check_codes(q, x, "codes");
    const int32_t lds = check_scale_out(scale, q.size(0), x.size(1), x);
    const int32_t ldp = sorted ? check_plan(*topk_row, x.size(0), x) : 0;
    written(q);
    written(scale);
    if (x.numel() == 0 || q.numel() == 0 || (sorted && topk_row->numel() == 0)) return;
    c10::cuda::CUDAGuard guard(x.device());
    check_rc(xmoe_fp8_quant(x.data_ptr(), elem_type(x, "x"), i32(x.size(0), "rows"), i32(x.size(1), "cols"),
                            i32(x.size(0) > 1 ? x.stride(0) : x.size(1), "x's stride"),
                            sorted ? topk_row->data_ptr<int32_t>() : nullptr, sorted ? i32(topk_row->size(1), "k") : 0, ldp,
                            i32(q.size(0), "rows"), q.data_ptr(), ldq, scale.data_ptr<float>(), lds, stream_of(x)),
             "xmoe_fp8_quant");
}

void fp8_quant_weight_cuda(const at::Tensor& w, at::Tensor& q, at::Tensor& scale) {
    check_cuda_contig(w, w, "w");
    check_cuda_contig(scale, w, "scale");
    TORCH_CHECK(w.dim() == 3 && w.size(1) > 0 && w.size(2) > 0 && q.sizes() == w.sizes(), "w and codes must be [mats, n, k]");
    const int32_t ldq = check_codes(q, w, "codes");
    TORCH_CHECK(w.size(0) <= 1 || q.stride(0) == (int64_t)ldq * w.size(1), "the codes' matrices must follow one another");
    TORCH_CHECK(scale.scalar_type() == at::kFloat && scale.dim() == 3 && scale.size(0) == w.size(0) &&
                    scale.size(1) == blocks_of(w.size(1)) && scale.size(2) == blocks_of(w.size(2)),
                "scale must be fp32 [mats, ceil(n / 128), ceil(k / 128)]");
    written(q);
    written(scale);
    if (w.numel() == 0) return;
    c10::cuda::CUDAGuard guard(w.device());
    check_rc(xmoe_fp8_quant_weight(w.data_ptr(), elem_type(w, "w"), i32(w.size(0), "mats"), i32(w.size(1), "n"),
                                   i32(w.size(2), "k"), q.data_ptr(), ldq, scale.data_ptr<float>(), stream_of(w)),
             "xmoe_fp8_quant_weight");
}

struct Segments { const int32_t* counts = nullptr; const int32_t* offsets = nullptr; int32_t mats = 0; };
Segments check_segments(const c10::optional<at::Tensor>& counts, const c10::optional<at::Tensor>& offsets, const at::Tensor& like) {
    Segments g;
    const bool have = counts.has_value() && counts->defined();
    TORCH_CHECK(have == (offsets.has_value() && offsets->defined()), "counts and offsets come together");
    if (!have) return g;
    for (const at::Tensor* t : {&*counts, &*offsets}) {
        check_cuda_contig(*t, like, "counts / offsets");
        TORCH_CHECK(t->scalar_type() == at::kInt && t->dim() == 1, "counts and offsets must be int32 vectors");
    }
    TORCH_CHECK(counts->size(0) > 0 && offsets->size(0) >= counts->size(0), "offsets must have an entry for every expert");
    g.counts = counts->data_ptr<int32_t>();
    g.offsets = offsets->data_ptr<int32_t>();
    g.mats = i32(counts->size(0), "experts");
    return g;
}

void glu_fp8_quant_cuda(const at::Tensor& h, int64_t activation, double alpha, double limit,
                        const c10::optional<at::Tensor>& counts, const c10::optional<at::Tensor>& offsets, at::Tensor& q,
                        at::Tensor& scale) {
    check_matrix(h, h, "h");
    TORCH_CHECK(h.size(1) > 0 && h.size(1) % 2 == 0, "h must be [rows, 2 * inter] (gate | up)");
    TORCH_CHECK(q.dim() == 2 && q.size(0) == h.size(0) && q.size(1) == h.size(1) / 2, "codes must be [rows, inter]");
    const int32_t ldq = check_codes(q, h, "codes");
    const int32_t lds = check_scale_out(scale, q.size(0), q.size(1), h);
    const Segments g = check_segments(counts, offsets, h);
    written(q);
    written(scale);
    if (h.numel() == 0) return;
    c10::cuda::CUDAGuard guard(h.device());
    check_rc(xmoe_glu_fp8_quant(h.data_ptr(), elem_type(h, "h"), i32(h.size(0), "rows"), i32(h.size(1) / 2, "inter"),
                                (int32_t)activation, (float)alpha, (float)limit, g.counts, g.offsets, g.mats, q.data_ptr(), ldq,
                                scale.data_ptr<float>(), lds, stream_of(h)),
             "xmoe_glu_fp8_quant");
}

void glu_backward_cuda(const at::Tensor& da, const at::Tensor& h, int64_t activation, double alpha, double limit,
                       const c10::optional<at::Tensor>& counts, const c10::optional<at::Tensor>& offsets, at::Tensor& dh) {
    check_matrix(h, h, "h");
    check_matrix(da, h, "da");
    check_matrix(dh, h, "dh");
    TORCH_CHECK(h.size(1) > 0 && h.size(1) % 2 == 0, "h must be [rows, 2 * inter] (gate | up)");
    TORCH_CHECK(da.scalar_type() == h.scalar_type() && da.size(0) == h.size(0) && da.size(1) == h.size(1) / 2,
                "da must be [rows, inter] of h's type");
    TORCH_CHECK(dh.scalar_type() == h.scalar_type() && dh.sizes() == h.sizes(), "dh must be like h");
    const Segments g = check_segments(counts, offsets, h);
    written(dh);
    if (h.numel() == 0) return;
    c10::cuda::CUDAGuard guard(h.device());
    check_rc(xmoe_glu_backward(da.data_ptr(), h.data_ptr(), elem_type(h, "h"), i32(h.size(0), "rows"), i32(h.size(1) / 2, "inter"),
                               (int32_t)activation, (float)alpha, (float)limit, g.counts, g.offsets, g.mats, dh.data_ptr(),
                               stream_of(h)),
             "xmoe_glu_backward");
}

// One product, grouped (counts given, w [mats, n, k]) or not (w [n, k]).
void fp8_product(const at::Tensor& x, const at::Tensor& x_scale, const at::Tensor& w, const at::Tensor& w_scale,
                 const Segments* g, bool transpose, int64_t rows_in_use, at::Tensor& out) {
    TORCH_CHECK(x.dim() == 2 && w.dim() == (g ? 3 : 2), g ? "x must be a matrix and w [experts, n, k]" : "x and w must be matrices");
    const int64_t n = w.size(w.dim() - 2), k = w.size(w.dim() - 1), rows = x.size(0);
    const int64_t in = transpose ? n : k, features = transpose ? k : n;
    TORCH_CHECK(n > 0 && k > 0, "w must not be empty");
    const int32_t ldx = check_codes(x, x, "x");
    const int32_t ldw = check_codes(w, x, "w");
    // numbers go through std::to_string: a compiler whose libstdc++ is linked in statically has stream facets of its own,
    // and an integer written to a stream that torch made then looks one up that is not there
    TORCH_CHECK(x.size(1) == in, "x has ", std::to_string(x.size(1)), " columns, the product contracts over ", std::to_string(in));
    TORCH_CHECK(x_scale.is_cuda() && x_scale.device() == x.device() && x_scale.scalar_type() == at::kFloat && x_scale.dim() == 2 &&
                    x_scale.size(0) == rows && x_scale.size(1) == blocks_of(in),
                "x_scale must be fp32 [rows, ceil(columns / 128)]");
    check_cuda_contig(w_scale, x, "w_scale");
    TORCH_CHECK(w_scale.scalar_type() == at::kFloat && w_scale.dim() == w.dim() && w_scale.size(-2) == blocks_of(n) &&
                    w_scale.size(-1) == blocks_of(k) && (!g || w_scale.size(0) == w.size(0)),
                "w_scale must be fp32 [.., ceil(n / 128), ceil(k / 128)]");
    check_matrix(out, x, "out");
    TORCH_CHECK(out.size(0) == rows && out.size(1) == features, "out must be [rows, ", std::to_string(features), "]");
    const int32_t out_type = elem_type(out, "out");
    if (g) {
        TORCH_CHECK(g->counts && g->mats == w.size(0), "counts must have an entry for every expert of w");
        TORCH_CHECK(w.size(0) == 1 || w.stride(0) % 16 == 0, "w's matrices must start at multiples of 16 bytes");
    }
    TORCH_CHECK(rows_in_use >= 0, "rows_in_use must not be negative");
    written(out);
    if (rows == 0) return;
    c10::cuda::CUDAGuard guard(x.device());
    int64_t lds = scale_ld(x_scale);
    at::Tensor relaid;
    if (lds < 0) {
        relaid = block_major(x_scale);
        lds = relaid.size(1);
    }
    const float* xs = lds >= 0 && relaid.defined() ? relaid.data_ptr<float>() : x_scale.data_ptr<float>();
    const int rc =
        g ? xmoe_fp8_grouped_gemm(x.data_ptr(), ldx, xs, i32(lds, "the scales' stride"), w.data_ptr(), ldw,
                                  w.size(0) > 1 ? w.stride(0) : 0, w_scale.data_ptr<float>(), g->counts, g->offsets, g->mats,
                                  i32(rows, "rows"), i32(rows_in_use, "rows_in_use"), i32(n, "n"), i32(k, "k"), transpose,
                                  out.data_ptr(), out_type, i32(features, "features"), stream_of(x))
          : xmoe_fp8_gemm(x.data_ptr(), ldx, xs, i32(lds, "the scales' stride"), w.data_ptr(), ldw, w_scale.data_ptr<float>(),
                          i32(rows, "rows"), i32(n, "n"), i32(k, "k"), transpose, out.data_ptr(), out_type,
                          i32(features, "features"), stream_of(x));
    check_rc(rc, g ? "xmoe_fp8_grouped_gemm" : "xmoe_fp8_gemm");
}
void fp8_matmul_cuda(const at::Tensor& x, const at::Tensor& x_scale, const at::Tensor& w, const at::Tensor& w_scale,
                     bool transpose, at::Tensor& out) {
    fp8_product(x, x_scale, w, w_scale, nullptr, transpose, 0, out);
}
at::Tensor fp8_matmul_new_cuda(const at::Tensor& x, const at::Tensor& x_scale, const at::Tensor& w, const at::Tensor& w_scale,
                               bool transpose, at::ScalarType out_dtype) {
    TORCH_CHECK(x.dim() == 2 && w.dim() == 2, "x and w must be matrices");
    at::Tensor out = at::empty({x.size(0), w.size(transpose ? 1 : 0)}, x.options().dtype(out_dtype));
    fp8_product(x, x_scale, w, w_scale, nullptr, transpose, 0, out);
    return out;
}
void fp8_grouped_matmul_cuda(const at::Tensor& x, const at::Tensor& x_scale, const at::Tensor& w, const at::Tensor& w_scale,
                             const at::Tensor& counts, const at::Tensor& offsets, bool transpose, int64_t rows_in_use,
                             at::Tensor& out) {
    const Segments g = check_segments(counts, offsets, x);
    fp8_product(x, x_scale, w, w_scale, &g, transpose, rows_in_use, out);
}

// Fake tensors: where every result is a tensor of the caller there is nothing to shape.
at::Tensor unpermute_new_meta(const at::Tensor& rows, const at::Tensor& topk_row, const c10::optional<at::Tensor>&) {
    return at::empty({topk_row.size(0), rows.size(1)}, rows.options());
}
at::Tensor fp8_matmul_new_meta(const at::Tensor& x, const at::Tensor&, const at::Tensor& w, const at::Tensor&, bool transpose,
                               at::ScalarType out_dtype) {
    return at::empty({x.size(0), w.size(transpose ? 1 : 0)}, x.options().dtype(out_dtype));
}
void permute_meta(const at::Tensor&, const at::Tensor&, at::Tensor& rows) { written(rows); }
void unpermute_meta(const at::Tensor&, const at::Tensor&, const c10::optional<at::Tensor>&, at::Tensor& y) { written(y); }
void unpermute_backward_meta(const at::Tensor&, const at::Tensor&, const at::Tensor&, const c10::optional<at::Tensor>&,
                             at::Tensor& drows, at::Tensor& dw) {
    written(drows);
    written(dw);
}
void fp8_quant_meta(const at::Tensor&, const c10::optional<at::Tensor>&, at::Tensor& codes, at::Tensor& scale) {
    written(codes);
    written(scale);
}
void fp8_quant_weight_meta(const at::Tensor&, at::Tensor& codes, at::Tensor& scale) {
    written(codes);
    written(scale);
}
void glu_fp8_quant_meta(const at::Tensor&, int64_t, double, double, const c10::optional<at::Tensor>&,
                        const c10::optional<at::Tensor>&, at::Tensor& codes, at::Tensor& scale) {
    written(codes);
    written(scale);
}
void glu_backward_meta(const at::Tensor&, const at::Tensor&, int64_t, double, double, const c10::optional<at::Tensor>&,
                       const c10::optional<at::Tensor>&, at::Tensor& dh) {
    written(dh);
}
void fp8_matmul_meta(const at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&, bool, at::Tensor& out) {
    written(out);
}
void fp8_grouped_matmul_meta(const at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&,
                             const at::Tensor&, bool, int64_t, at::Tensor& out) {
    written(out);
}

}  // namespace

TORCH_LIBRARY(xmoe_b200, m) {
    m.def(
        "forward(Tensor x, Tensor router_logits, Tensor? per_expert_scale, Tensor w13_packed, Tensor w13_sf, "
        "Tensor w13_gs, Tensor w2_q, Tensor w2_scale, Tensor? router_bias, Tensor? sigmoid_lut, int[] cfg_ints, "
        "float[] cfg_floats) -> Tensor");
    m.def("repack_gptq(Tensor qweight) -> Tensor");
    m.def("prep_nvfp4_sf(Tensor scale_e4m3, int rows_per_mat) -> Tensor");
    m.def("build_info() -> str", &build_info);
    m.def("permute(Tensor x, Tensor topk_row, Tensor(a!) rows) -> ()");
    m.def("unpermute(Tensor rows, Tensor topk_row, Tensor? weights, Tensor(a!) y) -> ()");
    m.def("unpermute_new(Tensor rows, Tensor topk_row, Tensor? weights) -> Tensor");
    m.def(
        "fp8_matmul_new(Tensor x, Tensor x_scale, Tensor w, Tensor w_scale, bool transpose, ScalarType out_dtype) -> Tensor");
    m.def(
        "unpermute_backward(Tensor dy, Tensor rows, Tensor topk_row, Tensor? weights, Tensor(a!) drows, Tensor(b!) dw) "
        "-> ()");
    m.def("fp8_quant(Tensor x, Tensor? topk_row, Tensor(a!) codes, Tensor(b!) scale) -> ()");
    m.def("fp8_quant_weight(Tensor w, Tensor(a!) codes, Tensor(b!) scale) -> ()");
    m.def(
        "glu_fp8_quant(Tensor h, int activation, float alpha, float limit, Tensor? counts, Tensor? offsets, Tensor(a!) "
        "codes, Tensor(b!) scale) -> ()");
    m.def(
        "glu_backward(Tensor da, Tensor h, int activation, float alpha, float limit, Tensor? counts, Tensor? offsets, "
        "Tensor(a!) dh) -> ()");
    m.def("fp8_matmul(Tensor x, Tensor x_scale, Tensor w, Tensor w_scale, bool transpose, Tensor(a!) out) -> ()");
    m.def(
        "fp8_grouped_matmul(Tensor x, Tensor x_scale, Tensor w, Tensor w_scale, Tensor counts, Tensor offsets, bool "
        "transpose, int rows_in_use, Tensor(a!) out) -> ()");
}

TORCH_LIBRARY_IMPL(xmoe_b200, CUDA, m) {
    m.impl("forward", &forward_cuda);
    m.impl("repack_gptq", &repack_gptq_cuda);
    m.impl("prep_nvfp4_sf", &prep_nvfp4_sf_cuda);
    m.impl("permute", &permute_cuda);
    m.impl("unpermute_new", &unpermute_new_cuda);
    m.impl("fp8_matmul_new", &fp8_matmul_new_cuda);
    m.impl("unpermute", &unpermute_cuda);
    m.impl("unpermute_backward", &unpermute_backward_cuda);
    m.impl("fp8_quant", &fp8_quant_cuda);
    m.impl("fp8_quant_weight", &fp8_quant_weight_cuda);
    m.impl("glu_fp8_quant", &glu_fp8_quant_cuda);
    m.impl("glu_backward", &glu_backward_cuda);
    m.impl("fp8_matmul", &fp8_matmul_cuda);
    m.impl("fp8_grouped_matmul", &fp8_grouped_matmul_cuda);
}

TORCH_LIBRARY_IMPL(xmoe_b200, Meta, m) {
    m.impl("forward", &forward_meta);
    m.impl("repack_gptq", &repack_gptq_meta);
    m.impl("prep_nvfp4_sf", &prep_nvfp4_sf_meta);
    m.impl("permute", &permute_meta);
    m.impl("unpermute_new", &unpermute_new_meta);
    m.impl("fp8_matmul_new", &fp8_matmul_new_meta);
    m.impl("unpermute", &unpermute_meta);
    m.impl("unpermute_backward", &unpermute_backward_meta);
    m.impl("fp8_quant", &fp8_quant_meta);
    m.impl("fp8_quant_weight", &fp8_quant_weight_meta);
    m.impl("glu_fp8_quant", &glu_fp8_quant_meta);
    m.impl("glu_backward", &glu_backward_meta);
    m.impl("fp8_matmul", &fp8_matmul_meta);
    m.impl("fp8_grouped_matmul", &fp8_grouped_matmul_meta);
}
