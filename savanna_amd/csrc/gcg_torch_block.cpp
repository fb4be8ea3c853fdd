// PyTorch binding of the operators around the convolution (include/gcg.h): 8-bit activation checkpoints and layer norm.
// As in gcg_torch.cpp: device and meta implementations of torch.ops.gcg.*, and C++ autograd nodes around them for eager
// training steps.
#include <optional>
#include <tuple>

#include "gcg_torch_common.h"

namespace {

using OptTensor = std::optional<Tensor>;

void *ptr(const OptTensor &t) { return t.has_value() && t->defined() ? t->data_ptr() : nullptr; }
bool given(const OptTensor &t) { return t.has_value() && t->defined(); }

// ---- 8-bit activation checkpoints ---------------------------------------------------------------

std::vector<int64_t> scale_sizes(const Tensor &x)
{
    std::vector<int64_t> s = x.sizes().vec();
    s.back() = (s.back() + GCG_BLOCK8 - 1) / GCG_BLOCK8;
    return s;
}

void check_rows(const Tensor &x)
{
    TORCH_CHECK(x.dim() >= 1 && x.is_contiguous(), "gcg: x must be a contiguous tensor of at least one dimension");
    (void)dtype_code(x.scalar_type());
}

std::tuple<Tensor, Tensor> pack8(const Tensor &x)
{
    require_gpu(x, "x");
    check_rows(x);
    DeviceGuard guard(x.device());
    Tensor codes = at::empty(x.sizes(), x.options().dtype(at::kChar));
    Tensor scales = at::empty(scale_sizes(x), x.options().dtype(at::kFloat));
    if (x.numel() == 0) return {codes, scales};
    const int64_t D = x.size(-1);
    check_rc(gcg_pack8(x.data_ptr(), (int8_t *)codes.data_ptr(), (float *)scales.data_ptr(), x.numel() / D, D,
                       dtype_code(x.scalar_type()), stream_of(x)),
             "gcg_pack8");
    return {codes, scales};
}

void check_codes(const Tensor &codes, const Tensor &scales)
{
    TORCH_CHECK(codes.dim() >= 1 && codes.scalar_type() == at::kChar && codes.is_contiguous(),
                "gcg: codes must be a contiguous int8 tensor");
    TORCH_CHECK(scales.scalar_type() == at::kFloat && scales.is_contiguous() && scales.sizes() == at::IntArrayRef(scale_sizes(codes)),
                "gcg: scales must be contiguous float32 with one element for every ", (int)GCG_BLOCK8, " codes of a row");
    TORCH_CHECK(scales.device() == codes.device(), "gcg: codes and scales must be on one device");
}

Tensor unpack8(const Tensor &codes, const Tensor &scales, at::ScalarType dtype)
{
    require_gpu(codes, "codes");
    check_codes(codes, scales);
    const int code = dtype_code(dtype);
    DeviceGuard guard(codes.device());
    Tensor x = at::empty(codes.sizes(), codes.options().dtype(dtype));
    if (x.numel() == 0) return x;
    const int64_t D = x.size(-1);
    check_rc(gcg_unpack8((const int8_t *)codes.data_ptr(), (const float *)scales.data_ptr(), x.data_ptr(), x.numel() / D, D, code,
                         stream_of(codes)),
             "gcg_unpack8");
    return x;
}

std::tuple<Tensor, Tensor> pack8_meta(const Tensor &x)
{
    check_rows(x);
    return {at::empty(x.sizes(), x.options().dtype(at::kChar)), at::empty(scale_sizes(x), x.options().dtype(at::kFloat))};
}
Tensor unpack8_meta(const Tensor &codes, const Tensor &scales, at::ScalarType dtype)
{
    check_codes(codes, scales);
    (void)dtype_code(dtype);
    return at::empty(codes.sizes(), codes.options().dtype(dtype));
}

// ---- layer norm ---------------------------------------------------------------------------------

// the library's code for x with these parameters; also checks both
int norm_code(const Tensor &x, const OptTensor &w, const OptTensor &b)
{
    check_rows(x);
    TORCH_CHECK(x.size(-1) > 0, "gcg: layer norm over an empty dimension");
    const int code = dtype_code(x.scalar_type());
    bool wide = false;
    for (const OptTensor *p : {&w, &b}) {
        if (!given(*p)) continue;
        const Tensor &t = **p;
        TORCH_CHECK(t.dim() == 1 && t.size(0) == x.size(-1) && t.is_contiguous(),
                    "gcg: weight and bias must be contiguous and have the size of x's last dimension");
        TORCH_CHECK(t.device() == x.device(), "gcg: x, weight and bias must be on one device");
        TORCH_CHECK(t.scalar_type() == x.scalar_type() || t.scalar_type() == at::kFloat,
                    "gcg: weight and bias must have x's dtype or be float32; got ", t.scalar_type(), " with ", x.scalar_type());
        wide = t.scalar_type() != x.scalar_type();
    }
    TORCH_CHECK(!given(w) || !given(b) || w->scalar_type() == b->scalar_type(), "gcg: weight and bias must share one dtype");
    if (!wide) return code;
    return code == GCG_BF16 ? GCG_BF16_F32 : GCG_F16_F32;
}

std::vector<int64_t> stats_sizes(const Tensor &x)
{
    std::vector<int64_t> s = x.sizes().vec();
    s.back() = 2;
    return s;
}

// (y, stats, codes, scales); what is not asked for is empty
std::tuple<Tensor, Tensor, Tensor, Tensor> norm_outputs(const Tensor &x, bool stats, bool save_8bit)
{
    const auto f32 = x.options().dtype(at::kFloat), i8 = x.options().dtype(at::kChar);
    return {at::empty_like(x), stats ? at::empty(stats_sizes(x), f32) : at::empty({0}, f32),
            save_8bit ? at::empty(x.sizes(), i8) : at::empty({0}, i8), save_8bit ? at::empty(scale_sizes(x), f32) : at::empty({0}, f32)};
}

void norm_fwd_launch(const Tensor &x, const OptTensor &w, const OptTensor &b, double eps, int code, Tensor &y, float *stats,
                     int8_t *codes, float *scales)
{
    if (x.numel() == 0) return;
    const int64_t D = x.size(-1);
    TORCH_CHECK(D <= GCG_NORM_MAX_WIDTH, "gcg: layer norm over ", D, " elements; at most ", (int)GCG_NORM_MAX_WIDTH, " are supported");
    check_rc(gcg_layer_norm_fwd(x.data_ptr(), ptr(w), ptr(b), y.data_ptr(), stats, codes, scales, x.numel() / D, (int32_t)D, (float)eps,
                                code, stream_of(x)),
             "gcg_layer_norm_fwd");
}

std::tuple<Tensor, Tensor, Tensor, Tensor> layer_norm_fwd(const Tensor &x, const OptTensor &w, const OptTensor &b, double eps,
                                                          bool save_8bit)
{
    require_gpu(x, "x");
    const int code = norm_code(x, w, b);
    DeviceGuard guard(x.device());
    auto out = norm_outputs(x, true, save_8bit);
    auto &[y, stats, codes, scales] = out;
    norm_fwd_launch(x, w, b, eps, code, y, (float *)stats.data_ptr(), save_8bit ? (int8_t *)codes.data_ptr() : nullptr,
                    save_8bit ? (float *)scales.data_ptr() : nullptr);
    return out;
}

// the result alone, for calls whose backward nobody asks for
Tensor layer_norm_infer(const Tensor &x, const OptTensor &w, const OptTensor &b, double eps)
{
    require_gpu(x, "x");
    const int code = norm_code(x, w, b);
    DeviceGuard guard(x.device());
    Tensor y = at::empty_like(x);
    norm_fwd_launch(x, w, b, eps, code, y, nullptr, nullptr, nullptr);
    return y;
}

void check_norm_bwd(const Tensor &dy, const OptTensor &x, const OptTensor &codes, const OptTensor &scales, const Tensor &stats)
{
    TORCH_CHECK(given(codes) == given(scales) && given(x) != given(codes), "gcg: the backward takes either x, or its codes and scales");
    check_rows(dy);
    if (given(x)) {
        TORCH_CHECK(x->sizes() == dy.sizes() && x->scalar_type() == dy.scalar_type() && x->device() == dy.device() && x->is_contiguous(),
                    "gcg: dy must be a contiguous tensor with the shape, dtype and device of x");
    } else {
        check_codes(*codes, *scales);
        TORCH_CHECK(codes->sizes() == dy.sizes() && codes->device() == dy.device(), "gcg: dy must have the shape and device of the codes");
    }
    TORCH_CHECK(stats.sizes() == at::IntArrayRef(stats_sizes(dy)) && stats.scalar_type() == at::kFloat && stats.is_contiguous() &&
                    stats.device() == dy.device(),
                "gcg: stats must be the forward's");
}

// (dx, dw, db); dw and db are empty without w and b
std::tuple<Tensor, Tensor, Tensor> layer_norm_bwd(const Tensor &dy, const OptTensor &x, const OptTensor &codes, const OptTensor &scales,
                                                  const Tensor &stats, const OptTensor &w, const OptTensor &b)
{
    require_gpu(dy, "dy");
    check_norm_bwd(dy, x, codes, scales, stats);
    const int code = norm_code(dy, w, b);
    DeviceGuard guard(dy.device());
    const int64_t D = dy.size(-1), rows = dy.numel() / D;
    Tensor dx = at::empty_like(dy);
    Tensor dw = given(w) ? at::empty_like(*w) : at::empty({0}, dy.options());
    Tensor db = given(b) ? at::empty_like(*b) : at::empty({0}, dy.options());
    if (rows == 0) return {dx, dw.zero_(), db.zero_()};
    Tensor ws;
    size_t bytes = 0;
    if (given(w) || given(b)) {
        bytes = gcg_layer_norm_bwd_workspace_bytes(rows, (int32_t)std::min<int64_t>(D, INT32_MAX), code);
        ws = workspace(bytes, dy, "gcg_layer_norm_bwd_workspace_bytes");
    }
    check_rc(gcg_layer_norm_bwd(dy.data_ptr(), ptr(x), (const int8_t *)ptr(codes), (const float *)ptr(scales),
                                (const float *)stats.data_ptr(), ptr(w), dx.data_ptr(), given(w) ? dw.data_ptr() : nullptr,
                                given(b) ? db.data_ptr() : nullptr, bytes ? ws.data_ptr() : nullptr, bytes, rows, (int32_t)D, code,
                                stream_of(dy)),
             "gcg_layer_norm_bwd");
    return {dx, dw, db};
}

std::tuple<Tensor, Tensor, Tensor, Tensor> layer_norm_fwd_meta(const Tensor &x, const OptTensor &w, const OptTensor &b, double,
                                                               bool save_8bit)
{
    (void)norm_code(x, w, b);
    return norm_outputs(x, true, save_8bit);
}
Tensor layer_norm_infer_meta(const Tensor &x, const OptTensor &w, const OptTensor &b, double)
{
    (void)norm_code(x, w, b);
    return at::empty_like(x);
}
std::tuple<Tensor, Tensor, Tensor> layer_norm_bwd_meta(const Tensor &dy, const OptTensor &x, const OptTensor &codes,
                                                       const OptTensor &scales, const Tensor &stats, const OptTensor &w,
                                                       const OptTensor &b)
{
    check_norm_bwd(dy, x, codes, scales, stats);
    (void)norm_code(dy, w, b);
    return {at::empty_like(dy), given(w) ? at::empty_like(*w) : at::empty({0}, dy.options()),
            given(b) ? at::empty_like(*b) : at::empty({0}, dy.options())};
}

Tensor or_empty(const OptTensor &t) { return given(t) ? *t : Tensor(); }
OptTensor opt(const Tensor &t) { return t.defined() ? OptTensor(t) : OptTensor(); }

struct LayerNormNode : torch::autograd::Function<LayerNormNode> {
    static Tensor forward(AutogradContext *ctx, const Tensor &x, const OptTensor &w, const OptTensor &b, double eps, bool save_8bit)
    {
        static const auto f = op<std::tuple<Tensor, Tensor, Tensor, Tensor>(const Tensor &, const OptTensor &, const OptTensor &, double,
                                                                           bool)>("gcg::layer_norm_fwd");
        at::AutoDispatchBelowADInplaceOrView below;
        auto [y, stats, codes, scales] = f.call(x, w, b, eps, save_8bit);
        if (save_8bit) ctx->save_for_backward({Tensor(), codes, scales, stats, or_empty(w), or_empty(b)});
        else ctx->save_for_backward({x, Tensor(), Tensor(), stats, or_empty(w), or_empty(b)});
        return y;
    }
    static variable_list backward(AutogradContext *ctx, variable_list dy)
    {
        static const auto f = op<std::tuple<Tensor, Tensor, Tensor>(const Tensor &, const OptTensor &, const OptTensor &,
                                                                   const OptTensor &, const Tensor &, const OptTensor &,
                                                                   const OptTensor &)>("gcg::layer_norm_bwd");
        const variable_list s = ctx->get_saved_variables();
        auto [dx, dw, db] = f.call(dy[0].contiguous(), opt(s[0]), opt(s[1]), opt(s[2]), s[3], opt(s[4]), opt(s[5]));
        return {dx, s[4].defined() ? dw : Tensor(), s[5].defined() ? db : Tensor(), Tensor(), Tensor()};
    }
};

Tensor layer_norm(const Tensor &x, const OptTensor &w, const OptTensor &b, double eps, bool save_8bit)
{
    return LayerNormNode::apply(x, w, b, eps, save_8bit);
}

} // namespace

TORCH_LIBRARY_FRAGMENT(gcg, m)
{
    m.def("pack8(Tensor x) -> (Tensor, Tensor)");
    m.def("unpack8(Tensor codes, Tensor scales, ScalarType dtype) -> Tensor");
    m.def("layer_norm_fwd(Tensor x, Tensor? w, Tensor? b, float eps, bool save_8bit) -> (Tensor, Tensor, Tensor, Tensor)");
    m.def("layer_norm_infer(Tensor x, Tensor? w, Tensor? b, float eps) -> Tensor");
    m.def("layer_norm_bwd(Tensor dy, Tensor? x, Tensor? codes, Tensor? scales, Tensor stats, Tensor? w, Tensor? b)"
          " -> (Tensor, Tensor, Tensor)");
    m.def("layer_norm(Tensor x, Tensor? w, Tensor? b, float eps, bool save_8bit) -> Tensor", &layer_norm);
}

TORCH_LIBRARY_IMPL(gcg, CUDA, m)
{
    m.impl("pack8", &pack8);
    m.impl("unpack8", &unpack8);
    m.impl("layer_norm_fwd", &layer_norm_fwd);
    m.impl("layer_norm_infer", &layer_norm_infer);
    m.impl("layer_norm_bwd", &layer_norm_bwd);
}

TORCH_LIBRARY_IMPL(gcg, Meta, m)
{
    m.impl("pack8", &pack8_meta);
    m.impl("unpack8", &unpack8_meta);
    m.impl("layer_norm_fwd", &layer_norm_fwd_meta);
    m.impl("layer_norm_infer", &layer_norm_infer_meta);
    m.impl("layer_norm_bwd", &layer_norm_bwd_meta);
}
