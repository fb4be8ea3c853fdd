// PyTorch binding of the operators around the convolution (include/gcg.h): 8-bit activation checkpoints, layer norm, linear
// attention with a decay for each head.
// As in gcg_torch.cpp: device and meta implementations of torch.ops.gcg.*, and C++ autograd nodes around them for eager
// training steps.
#include <algorithm>
#include <array>
#include <optional>
#include <tuple>
#include <vector>

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
    TORCH_CHECK(x.size(-1) <= GCG_NORM_MAX_WIDTH, "gcg: layer norm over ", x.size(-1), " elements; at most ", (int)GCG_NORM_MAX_WIDTH,
                " are supported");
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

Tensor norm_gradient(const OptTensor &p, bool need, const Tensor &dy) { return given(p) && need ? at::empty_like(*p) : at::empty({0}, dy.options()); }

// (dx, dw, db); dw and db are empty without w and b, or where they are not needed
std::tuple<Tensor, Tensor, Tensor> layer_norm_bwd(const Tensor &dy, const OptTensor &x, const OptTensor &codes, const OptTensor &scales,
                                                  const Tensor &stats, const OptTensor &w, const OptTensor &b, bool need_dw, bool need_db)
{
    require_gpu(dy, "dy");
    check_norm_bwd(dy, x, codes, scales, stats);
    const int code = norm_code(dy, w, b);
    DeviceGuard guard(dy.device());
    const int64_t D = dy.size(-1), rows = dy.numel() / D;
    Tensor dx = at::empty_like(dy);
    need_dw = need_dw && given(w);
    need_db = need_db && given(b);
    Tensor dw = norm_gradient(w, need_dw, dy), db = norm_gradient(b, need_db, dy);
    if (rows == 0) return {dx, dw.zero_(), db.zero_()};
    Tensor ws;
    size_t bytes = 0;
    if (need_dw || need_db) {
        bytes = gcg_layer_norm_bwd_workspace_bytes(rows, (int32_t)D, code);
        ws = workspace(bytes, dy, "gcg_layer_norm_bwd_workspace_bytes");
    }
    check_rc(gcg_layer_norm_bwd(dy.data_ptr(), ptr(x), (const int8_t *)ptr(codes), (const float *)ptr(scales),
                                (const float *)stats.data_ptr(), ptr(w), dx.data_ptr(), need_dw ? dw.data_ptr() : nullptr,
                                need_db ? db.data_ptr() : nullptr, bytes ? ws.data_ptr() : nullptr, bytes, rows, (int32_t)D, code,
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
                                                       const OptTensor &b, bool need_dw, bool need_db)
{
    check_norm_bwd(dy, x, codes, scales, stats);
    (void)norm_code(dy, w, b);
    return {at::empty_like(dy), norm_gradient(w, need_dw, dy), norm_gradient(b, need_db, dy)};
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
        ctx->saved_data["dw"] = given(w) && w->requires_grad();
        ctx->saved_data["db"] = given(b) && b->requires_grad();
        return y;
    }
    static variable_list backward(AutogradContext *ctx, variable_list dy)
    {
        static const auto f = op<std::tuple<Tensor, Tensor, Tensor>(const Tensor &, const OptTensor &, const OptTensor &,
                                                                   const OptTensor &, const Tensor &, const OptTensor &,
                                                                   const OptTensor &, bool, bool)>("gcg::layer_norm_bwd");
        const variable_list s = ctx->get_saved_variables();
        const bool need_dw = ctx->saved_data["dw"].toBool(), need_db = ctx->saved_data["db"].toBool();
        auto [dx, dw, db] = f.call(dy[0].contiguous(), opt(s[0]), opt(s[1]), opt(s[2]), s[3], opt(s[4]), opt(s[5]), need_dw, need_db);
        return {dx, need_dw ? dw : Tensor(), need_db ? db : Tensor(), Tensor(), Tensor()};
    }
};

Tensor layer_norm(const Tensor &x, const OptTensor &w, const OptTensor &b, double eps, bool save_8bit)
{
    return LayerNormNode::apply(x, w, b, eps, save_8bit);
}

// ---- linear attention with a decay for each head ------------------------------------------------------

void add_strides(std::vector<int64_t> &s, const Tensor &t) { s.insert(s.end(), {t.stride(0), t.stride(1), t.stride(2)}); }

// a tensor whose last dimension is contiguous and whose rows are near enough to each other, as the kernels read it
Tensor rows_of(const Tensor &t)
{
    const bool in_place = (t.size(-1) == 1 || t.stride(-1) == 1) && (t.dim() < 4 || t.stride(1) <= GCG_LINEAR_MAX_TIME_STRIDE);
    return in_place ? t : t.contiguous();
}

void check_heads(const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &log_decay, int64_t dim)
{
    TORCH_CHECK(q.dim() == dim && k.dim() == dim && v.dim() == dim && q.sizes() == k.sizes() &&
                    v.sizes().slice(0, dim - 1) == q.sizes().slice(0, dim - 1),
                dim == 4 ? "gcg: q and k must be (bs, L, H, dk), v (bs, L, H, dv)" : "gcg: q and k must be (bs, H, dk), v (bs, H, dv)");
    TORCH_CHECK(k.scalar_type() == q.scalar_type() && v.scalar_type() == q.scalar_type() && k.device() == q.device() &&
                    v.device() == q.device(),
                "gcg: q, k and v must share dtype and device");
    (void)dtype_code(q.scalar_type());
    TORCH_CHECK(log_decay.dim() == 1 && log_decay.size(0) == q.size(dim - 2) && log_decay.scalar_type() == at::kFloat &&
                    log_decay.is_contiguous() && log_decay.device() == q.device(),
                "gcg: log_decay must be a contiguous float32 tensor of one element a head on q's device");
    TORCH_CHECK(q.size(dim - 2) <= INT32_MAX, "gcg: ", q.size(dim - 2), " heads; at most ", INT32_MAX, " are supported");
    TORCH_CHECK(q.size(-1) <= GCG_LINEAR_MAX_DIM && v.size(-1) <= GCG_LINEAR_MAX_DIM && q.size(-1) > 0 && v.size(-1) > 0,
                "gcg: head dimensions are 1 to ", (int)GCG_LINEAR_MAX_DIM);
}

void check_state(const OptTensor &t, const Tensor &q, const Tensor &v, const char *name)
{
    if (!given(t)) return;
    TORCH_CHECK(t->dim() == 4 && t->size(0) == q.size(0) && t->size(1) == q.size(-2) && t->size(2) == q.size(-1) &&
                    t->size(3) == v.size(-1) && t->scalar_type() == at::kFloat && t->is_contiguous() && t->device() == q.device(),
                "gcg: ", name, " must be a contiguous (bs, H, dk, dv) float32 tensor on q's device");
}

void check_lengths(const OptTensor &t, const Tensor &q)
{
    if (!given(t)) return;
    TORCH_CHECK(t->dim() == 1 && t->size(0) == q.size(0) && t->scalar_type() == at::kInt && t->is_contiguous() && t->device() == q.device(),
                "gcg: lengths must be a contiguous int32 tensor of one element a batch entry on q's device");
}

Tensor new_state(const Tensor &q, const Tensor &v, bool wanted)
{
    const auto f32 = q.options().dtype(at::kFloat);
    return wanted ? at::empty({q.size(0), q.size(-2), q.size(-1), v.size(-1)}, f32) : at::empty({0}, f32);
}

Tensor linear_workspace(const Tensor &q, const Tensor &v, bool backward, size_t *bytes)
{
    *bytes = gcg_linear_attn_workspace_bytes(q.size(0), q.size(1), (int32_t)q.size(2), (int32_t)q.size(3), (int32_t)v.size(3), backward);
    return *bytes ? at::empty({(int64_t)*bytes}, q.options().dtype(at::kByte)) : Tensor();
}

// a sequence of no rows: the state is the one given
Tensor passed_on(const OptTensor &from, Tensor to) { return to.numel() == 0 ? to : given(from) ? to.copy_(*from) : to.zero_(); }

// Head dimensions that the kernels' vectors do not divide: the tensors with zeros up to the next multiple of 8, which add nothing
// to any product, and the results without them.
int64_t to_whole(const Tensor &q, int64_t d) { return q.scalar_type() == at::kFloat && d % 4 == 0 ? 0 : (8 - d % 8) % 8; }
bool odd_heads(const Tensor &q, const Tensor &v) { return to_whole(q, q.size(-1)) || to_whole(q, v.size(-1)); }
Tensor padded(const Tensor &t, int64_t n) { return n ? at::constant_pad_nd(t, {0, n}) : t; }
OptTensor padded_state(const OptTensor &t, int64_t dk, int64_t dv) { return given(t) ? OptTensor(at::constant_pad_nd(*t, {0, dv, 0, dk})) : t; }
Tensor cut(const Tensor &t, int64_t d) { return t.size(-1) == d ? t : t.slice(-1, 0, d).contiguous(); }
Tensor cut_state(const Tensor &t, int64_t dk, int64_t dv) { return t.numel() ? t.slice(2, 0, dk).slice(3, 0, dv).contiguous() : t; }

// The batch at once, or, with more heads in it than a launch takes, some entries after the others.
template <typename Part, typename Whole> void for_entries(const Tensor &q, Part part, Whole whole)
{
    const int64_t bs = q.size(0), H = q.size(2), n = std::max<int64_t>(1, GCG_LINEAR_MAX_HEADS / H);
    if (bs <= n) return whole();
    for (int64_t at = 0; at < bs; at += n) part(at, std::min(n, bs - at));
}
OptTensor entries(const OptTensor &t, int64_t at, int64_t n) { return given(t) ? OptTensor(t->narrow(0, at, n)) : t; }

void linear_fwd_launch(const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &log_decay, const OptTensor &initial,
                       const OptTensor &lengths, double scale, const Tensor &o, const Tensor &last)
{
    const Tensor a = rows_of(q), b = rows_of(k), c = rows_of(v);
    std::vector<int64_t> s;
    for (const Tensor *t : {&a, &b, &c, &o}) add_strides(s, *t);
    size_t bytes;
    Tensor ws = linear_workspace(q, v, false, &bytes);
    check_rc(gcg_linear_attn_fwd(a.data_ptr(), b.data_ptr(), c.data_ptr(), s.data(), (const float *)log_decay.data_ptr(),
                                 (const float *)ptr(initial), (const int32_t *)ptr(lengths), o.data_ptr(),
                                 last.defined() ? (float *)last.data_ptr() : nullptr, bytes ? ws.data_ptr() : nullptr, bytes, q.size(0),
                                 q.size(1), (int32_t)q.size(2), (int32_t)q.size(3), (int32_t)v.size(3), (float)scale,
                                 dtype_code(q.scalar_type()), stream_of(q)),
             "gcg_linear_attn_fwd");
}

std::tuple<Tensor, Tensor> linear_attn_fwd(const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &log_decay,
                                           const OptTensor &initial, const OptTensor &lengths, double scale, bool final)
{
    require_gpu(q, "q");
    check_heads(q, k, v, log_decay, 4);
    check_state(initial, q, v, "initial_state");
    check_lengths(lengths, q);
    DeviceGuard guard(q.device());
    Tensor o = at::empty({v.size(0), v.size(1), v.size(2), v.size(3)}, v.options());
    Tensor last = new_state(q, v, final);
    if (o.numel() == 0) return {o, passed_on(initial, last)};
    if (odd_heads(q, v)) {
        const int64_t dk = q.size(-1), dv = v.size(-1), pk = to_whole(q, dk), pv = to_whole(q, dv);
        const auto [po, pl] = linear_attn_fwd(padded(q, pk), padded(k, pk), padded(v, pv), log_decay, padded_state(initial, pk, pv), lengths,
                                              scale, final);
        return {cut(po, dv), cut_state(pl, dk, dv)};
    }
    for_entries(q, [&](int64_t at, int64_t n) {
        linear_fwd_launch(q.narrow(0, at, n), k.narrow(0, at, n), v.narrow(0, at, n), log_decay, entries(initial, at, n),
                          entries(lengths, at, n), scale, o.narrow(0, at, n), final ? last.narrow(0, at, n) : Tensor());
    }, [&] { linear_fwd_launch(q, k, v, log_decay, initial, lengths, scale, o, final ? last : Tensor()); });
    return {o, last};
}

void linear_bwd_launch(const Tensor &d_o, const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &log_decay,
                       const OptTensor &initial, const OptTensor &lengths, const OptTensor &dfinal, double scale, const Tensor &dq,
                       const Tensor &d_k, const Tensor &d_v, const Tensor &dinitial)
{
    const Tensor g = rows_of(d_o), a = rows_of(q), b = rows_of(k), c = rows_of(v);
    std::vector<int64_t> s;
    for (const Tensor *t : {&g, &a, &b, &c, &dq, &d_k, &d_v}) add_strides(s, *t);
    size_t bytes;
    Tensor ws = linear_workspace(q, v, true, &bytes);
    check_rc(gcg_linear_attn_bwd(g.data_ptr(), a.data_ptr(), b.data_ptr(), c.data_ptr(), s.data(), (const float *)log_decay.data_ptr(),
                                 (const float *)ptr(initial), (const int32_t *)ptr(lengths), (const float *)ptr(dfinal), dq.data_ptr(),
                                 d_k.data_ptr(), d_v.data_ptr(), dinitial.defined() ? (float *)dinitial.data_ptr() : nullptr,
                                 bytes ? ws.data_ptr() : nullptr, bytes, q.size(0), q.size(1), (int32_t)q.size(2), (int32_t)q.size(3),
                                 (int32_t)v.size(3), (float)scale, dtype_code(q.scalar_type()), stream_of(q)),
             "gcg_linear_attn_bwd");
}

void linear_bwd_all(const Tensor &d_o, const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &log_decay, const OptTensor &initial,
                    const OptTensor &lengths, const OptTensor &dfinal, double scale, const Tensor &dq, const Tensor &d_k, const Tensor &d_v,
                    const Tensor &dinitial)
{
    for_entries(q, [&](int64_t at, int64_t n) {
        const auto of = [&](const Tensor &t) { return t.narrow(0, at, n); };
        linear_bwd_launch(of(d_o), of(q), of(k), of(v), log_decay, entries(initial, at, n), entries(lengths, at, n), entries(dfinal, at, n),
                          scale, of(dq), of(d_k), of(d_v), dinitial.defined() ? of(dinitial) : Tensor());
    }, [&] { linear_bwd_launch(d_o, q, k, v, log_decay, initial, lengths, dfinal, scale, dq, d_k, d_v, dinitial); });
}

void check_do(const Tensor &d_o, const Tensor &v)
{
    TORCH_CHECK(d_o.sizes() == v.sizes() && d_o.scalar_type() == v.scalar_type() && d_o.device() == v.device(),
                "gcg: do must have the shape, dtype and device of v");
}

std::tuple<Tensor, Tensor, Tensor, Tensor> linear_attn_bwd(const Tensor &d_o, const Tensor &q, const Tensor &k, const Tensor &v,
                                                           const Tensor &log_decay, const OptTensor &initial, const OptTensor &lengths,
                                                           const OptTensor &dfinal, double scale, bool need_dinitial)
{
    require_gpu(q, "q");
    check_heads(q, k, v, log_decay, 4);
    check_do(d_o, v);
    check_state(initial, q, v, "initial_state");
    check_state(dfinal, q, v, "the final state's gradient");
    check_lengths(lengths, q);
    DeviceGuard guard(q.device());
    Tensor dq = at::empty(q.sizes(), q.options()), d_k = at::empty(k.sizes(), k.options()), d_v = at::empty(v.sizes(), v.options());
    Tensor dinitial = new_state(q, v, need_dinitial);
    if (d_o.numel() == 0) return {dq, d_k, d_v, passed_on(dfinal, dinitial)};
    if (odd_heads(q, v)) {
        const int64_t dk = q.size(-1), dv = v.size(-1), pk = to_whole(q, dk), pv = to_whole(q, dv);
        const auto [pq, pkk, pvv, pi] = linear_attn_bwd(padded(d_o, pv), padded(q, pk), padded(k, pk), padded(v, pv), log_decay,
                                                        padded_state(initial, pk, pv), lengths, padded_state(dfinal, pk, pv), scale,
                                                        need_dinitial);
        return {cut(pq, dk), cut(pkk, dk), cut(pvv, dv), cut_state(pi, dk, dv)};
    }
    linear_bwd_all(d_o, q, k, v, log_decay, initial, lengths, dfinal, scale, dq, d_k, d_v, need_dinitial ? dinitial : Tensor());
    return {dq, d_k, d_v, dinitial};
}

// the projected features (bs, L, 3 * H * d), laid out "(p h d)" with p = q, k, v
std::array<Tensor, 3> split_features(const Tensor &features, int64_t H)
{
    TORCH_CHECK(features.dim() == 3 && features.is_contiguous() && H > 0 && features.size(2) % (3 * H) == 0,
                "gcg: features must be a contiguous (bs, L, 3 * H * d) tensor");
    const Tensor f = features.view({features.size(0), features.size(1), 3, H, features.size(2) / (3 * H)});
    return {f.select(2, 0), f.select(2, 1), f.select(2, 2)};
}

Tensor linear_attn_packed_fwd(const Tensor &features, int64_t H, const Tensor &log_decay, double scale)
{
    const auto [q, k, v] = split_features(features, H);
    return std::get<0>(linear_attn_fwd(q, k, v, log_decay, OptTensor(), OptTensor(), scale, false));
}

Tensor linear_attn_packed_bwd(const Tensor &d_o, const Tensor &features, int64_t H, const Tensor &log_decay, double scale)
{
    require_gpu(features, "features");
    const auto [q, k, v] = split_features(features, H);
    check_heads(q, k, v, log_decay, 4);
    check_do(d_o, v);
    DeviceGuard guard(q.device());
    Tensor df = at::empty_like(features);
    if (df.numel() == 0) return df;
    const auto [dq, d_k, d_v] = split_features(df, H);
    // (the kernels write no rows further apart; the forward copies such an input)
    if (odd_heads(q, v) || features.size(2) > GCG_LINEAR_MAX_TIME_STRIDE) {
        const auto [pq, pk, pv, pi] = linear_attn_bwd(d_o, q, k, v, log_decay, OptTensor(), OptTensor(), OptTensor(), scale, false);
        dq.copy_(pq);
        d_k.copy_(pk);
        d_v.copy_(pv);
        return df;
    }
    linear_bwd_all(d_o, q, k, v, log_decay, OptTensor(), OptTensor(), OptTensor(), scale, dq, d_k, d_v, Tensor());
    return df;
}

Tensor linear_attn_step(const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &log_decay, Tensor &state, double scale)
{
    require_gpu(q, "q");
    check_heads(q, k, v, log_decay, 3);
    check_state(state, q, v, "state");
    DeviceGuard guard(q.device());
    Tensor o = at::empty(v.sizes(), v.options());
    if (o.numel() == 0) return o;
    const Tensor a = rows_of(q), b = rows_of(k), c = rows_of(v);
    const int64_t s[8] = {a.stride(0), a.stride(1), b.stride(0), b.stride(1), c.stride(0), c.stride(1), o.stride(0), o.stride(1)};
    check_rc(gcg_linear_attn_step(a.data_ptr(), b.data_ptr(), c.data_ptr(), o.data_ptr(), s, (const float *)log_decay.data_ptr(),
                                  (float *)state.data_ptr(), q.size(0), (int32_t)q.size(1), (int32_t)q.size(2), (int32_t)v.size(2),
                                  (float)scale, dtype_code(q.scalar_type()), stream_of(q)),
             "gcg_linear_attn_step");
    return o;
}

// The step as in-place operators of torch are: whatever saved the state for a backward pass finds it modified.  (An inference tensor
// has no such count, and nothing can have saved it.)
Tensor linear_attn_step_in_place(const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &log_decay, Tensor &state, double scale)
{
    static const auto f = op<Tensor(const Tensor &, const Tensor &, const Tensor &, const Tensor &, Tensor &, double)>("gcg::linear_attn_step");
    Tensor o;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        o = f.call(q, k, v, log_decay, state, scale);
    }
    if (!state.is_inference()) torch::autograd::impl::bump_version(state);
    return o;
}

std::tuple<Tensor, Tensor> linear_attn_fwd_meta(const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &log_decay,
                                                const OptTensor &initial, const OptTensor &lengths, double, bool final)
{
    check_heads(q, k, v, log_decay, 4);
    check_state(initial, q, v, "initial_state");
    check_lengths(lengths, q);
    return {at::empty(v.sizes(), v.options()), new_state(q, v, final)};
}
std::tuple<Tensor, Tensor, Tensor, Tensor> linear_attn_bwd_meta(const Tensor &d_o, const Tensor &q, const Tensor &k, const Tensor &v,
                                                                const Tensor &log_decay, const OptTensor &, const OptTensor &,
                                                                const OptTensor &, double, bool need_dinitial)
{
    check_heads(q, k, v, log_decay, 4);
    check_do(d_o, v);
    return {at::empty(q.sizes(), q.options()), at::empty(k.sizes(), k.options()), at::empty(v.sizes(), v.options()),
            new_state(q, v, need_dinitial)};
}
Tensor linear_attn_packed_fwd_meta(const Tensor &features, int64_t H, const Tensor &log_decay, double)
{
    const auto [q, k, v] = split_features(features, H);
    check_heads(q, k, v, log_decay, 4);
    return at::empty({features.size(0), features.size(1), H, features.size(2) / (3 * H)}, features.options());
}
Tensor linear_attn_packed_bwd_meta(const Tensor &, const Tensor &features, int64_t H, const Tensor &, double)
{
    (void)split_features(features, H);
    return at::empty_like(features);
}
Tensor linear_attn_step_meta(const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &log_decay, Tensor &state, double)
{
    check_heads(q, k, v, log_decay, 3);
    check_state(state, q, v, "state");
    return at::empty(v.sizes(), v.options());
}

struct LinearAttnNode : torch::autograd::Function<LinearAttnNode> {
    static variable_list forward(AutogradContext *ctx, const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &log_decay,
                                 const OptTensor &initial, const OptTensor &lengths, double scale, bool final)
    {
        static const auto f = op<std::tuple<Tensor, Tensor>(const Tensor &, const Tensor &, const Tensor &, const Tensor &,
                                                           const OptTensor &, const OptTensor &, double, bool)>("gcg::linear_attn_fwd");
        at::AutoDispatchBelowADInplaceOrView below;
        ctx->set_materialize_grads(false);
        ctx->save_for_backward({q, k, v, log_decay, or_empty(initial), or_empty(lengths)});
        ctx->saved_data["scale"] = scale;
        ctx->saved_data["dinitial"] = given(initial) && initial->requires_grad();
        auto [o, last] = f.call(q, k, v, log_decay, initial, lengths, scale, final);
        if (final) return {o, last};
        return {o};
    }
    static variable_list backward(AutogradContext *ctx, variable_list g)
    {
        static const auto f = op<std::tuple<Tensor, Tensor, Tensor, Tensor>(const Tensor &, const Tensor &, const Tensor &, const Tensor &,
                                                                           const Tensor &, const OptTensor &, const OptTensor &,
                                                                           const OptTensor &, double, bool)>("gcg::linear_attn_bwd");
        const variable_list s = ctx->get_saved_variables();
        const Tensor d_o = g[0].defined() ? g[0] : at::zeros(s[2].sizes(), s[2].options());
        const Tensor dfinal = g.size() > 1 && g[1].defined() ? g[1].contiguous() : Tensor();
        const bool need = ctx->saved_data["dinitial"].toBool();
        auto [dq, d_k, d_v, dinitial] = f.call(d_o, s[0], s[1], s[2], s[3], opt(s[4]), opt(s[5]), opt(dfinal),
                                               ctx->saved_data["scale"].toDouble(), need);
        return {dq, d_k, d_v, Tensor(), need ? dinitial : Tensor(), Tensor(), Tensor(), Tensor()};
    }
};

struct PackedLinearAttnNode : torch::autograd::Function<PackedLinearAttnNode> {
    static Tensor forward(AutogradContext *ctx, const Tensor &features, int64_t H, const Tensor &log_decay, double scale, bool save_8bit)
    {
        static const auto f = op<Tensor(const Tensor &, int64_t, const Tensor &, double)>("gcg::linear_attn_packed_fwd");
        static const auto pack = op<std::tuple<Tensor, Tensor>(const Tensor &)>("gcg::pack8");
        at::AutoDispatchBelowADInplaceOrView below;
        Tensor codes, scales;
        if (save_8bit) std::tie(codes, scales) = pack.call(features);
        ctx->save_for_backward({save_8bit ? Tensor() : features, codes, scales, log_decay});
        ctx->saved_data["H"] = H;
        ctx->saved_data["scale"] = scale;
        ctx->saved_data["dtype"] = (int64_t)features.scalar_type();
        return f.call(features, H, log_decay, scale);
    }
    static variable_list backward(AutogradContext *ctx, variable_list g)
    {
        static const auto f = op<Tensor(const Tensor &, const Tensor &, int64_t, const Tensor &, double)>("gcg::linear_attn_packed_bwd");
        static const auto unpack = op<Tensor(const Tensor &, const Tensor &, at::ScalarType)>("gcg::unpack8");
        const variable_list s = ctx->get_saved_variables();
        const Tensor features = s[0].defined() ? s[0] : unpack.call(s[1], s[2], (at::ScalarType)ctx->saved_data["dtype"].toInt());
        return {f.call(g[0], features, ctx->saved_data["H"].toInt(), s[3], ctx->saved_data["scale"].toDouble()), Tensor(), Tensor(),
                Tensor(), Tensor()};
    }
};

// the decays' gradient is none of the operator's: asked for, it is refused rather than left out
void check_constant(const Tensor &log_decay)
{
    TORCH_CHECK(!(at::GradMode::is_enabled() && log_decay.requires_grad()),
                "gcg: log_decay is a constant of the heads and has no gradient; pass log_decay.detach()");
}

std::vector<Tensor> linear_attn(const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &log_decay, const OptTensor &initial,
                                const OptTensor &lengths, double scale, bool final)
{
    check_constant(log_decay);
    return LinearAttnNode::apply(q, k, v, log_decay, initial, lengths, scale, final);
}
Tensor linear_attn_packed(const Tensor &features, int64_t H, const Tensor &log_decay, double scale, bool save_8bit)
{
    check_constant(log_decay);
    return PackedLinearAttnNode::apply(features, H, log_decay, scale, save_8bit);
}

} // namespace

TORCH_LIBRARY_FRAGMENT(gcg, m)
{
    m.def("pack8(Tensor x) -> (Tensor, Tensor)");
    m.def("unpack8(Tensor codes, Tensor scales, ScalarType dtype) -> Tensor");
    m.def("layer_norm_fwd(Tensor x, Tensor? w, Tensor? b, float eps, bool save_8bit) -> (Tensor, Tensor, Tensor, Tensor)");
    m.def("layer_norm_infer(Tensor x, Tensor? w, Tensor? b, float eps) -> Tensor");
    m.def("layer_norm_bwd(Tensor dy, Tensor? x, Tensor? codes, Tensor? scales, Tensor stats, Tensor? w, Tensor? b,"
          " bool need_dw=True, bool need_db=True) -> (Tensor, Tensor, Tensor)");
    m.def("layer_norm(Tensor x, Tensor? w, Tensor? b, float eps, bool save_8bit) -> Tensor", &layer_norm);
    m.def("linear_attn_fwd(Tensor q, Tensor k, Tensor v, Tensor log_decay, Tensor? initial, Tensor? lengths, float scale, bool final)"
          " -> (Tensor, Tensor)");
    m.def("linear_attn_bwd(Tensor d_o, Tensor q, Tensor k, Tensor v, Tensor log_decay, Tensor? initial, Tensor? lengths, Tensor? dfinal,"
          " float scale, bool need_dinitial) -> (Tensor, Tensor, Tensor, Tensor)");
    m.def("linear_attn_packed_fwd(Tensor features, int H, Tensor log_decay, float scale) -> Tensor");
    m.def("linear_attn_packed_bwd(Tensor d_o, Tensor features, int H, Tensor log_decay, float scale) -> Tensor");
    m.def("linear_attn_step(Tensor q, Tensor k, Tensor v, Tensor log_decay, Tensor(a!) state, float scale) -> Tensor");
    m.def("linear_attn(Tensor q, Tensor k, Tensor v, Tensor log_decay, Tensor? initial, Tensor? lengths, float scale, bool final)"
          " -> Tensor[]", &linear_attn);
    m.def("linear_attn_packed(Tensor features, int H, Tensor log_decay, float scale, bool save_8bit) -> Tensor", &linear_attn_packed);
}

TORCH_LIBRARY_IMPL(gcg, CUDA, m)
{
    m.impl("pack8", &pack8);
    m.impl("unpack8", &unpack8);
    m.impl("layer_norm_fwd", &layer_norm_fwd);
    m.impl("layer_norm_infer", &layer_norm_infer);
    m.impl("layer_norm_bwd", &layer_norm_bwd);
    m.impl("linear_attn_fwd", &linear_attn_fwd);
    m.impl("linear_attn_bwd", &linear_attn_bwd);
    m.impl("linear_attn_packed_fwd", &linear_attn_packed_fwd);
    m.impl("linear_attn_packed_bwd", &linear_attn_packed_bwd);
    m.impl("linear_attn_step", &linear_attn_step);
}

TORCH_LIBRARY_IMPL(gcg, ADInplaceOrView, m)
{
    m.impl("linear_attn_step", &linear_attn_step_in_place);
}

TORCH_LIBRARY_IMPL(gcg, Meta, m)
{
    m.impl("pack8", &pack8_meta);
    m.impl("unpack8", &unpack8_meta);
    m.impl("layer_norm_fwd", &layer_norm_fwd_meta);
    m.impl("layer_norm_infer", &layer_norm_infer_meta);
    m.impl("layer_norm_bwd", &layer_norm_bwd_meta);
    m.impl("linear_attn_fwd", &linear_attn_fwd_meta);
    m.impl("linear_attn_bwd", &linear_attn_bwd_meta);
    m.impl("linear_attn_packed_fwd", &linear_attn_packed_fwd_meta);
    m.impl("linear_attn_packed_bwd", &linear_attn_packed_bwd_meta);
    m.impl("linear_attn_step", &linear_attn_step_meta);
}
