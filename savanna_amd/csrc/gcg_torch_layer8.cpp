// PyTorch binding of the operators of a layer in 8-bit floating point around a recurrent mixer (include/gcg.h): root-mean-square
// norm, 8-bit tensors and their products, gated linear recurrence.
// As in gcg_torch.cpp: device and meta implementations of torch.ops.gcg.*, and C++ autograd nodes around them for eager
// training steps.
#include <optional>
#include <tuple>
#include <vector>

#include "gcg_torch_common.h"

namespace {

using OptTensor = std::optional<Tensor>;
using Two = std::tuple<Tensor, Tensor>;
using Three = std::tuple<Tensor, Tensor, Tensor>;
using Four = std::tuple<Tensor, Tensor, Tensor, Tensor>;
using Five = std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor>;

bool given(const OptTensor &t) { return t.has_value() && t->defined(); }
void *ptr(const OptTensor &t) { return given(t) ? t->data_ptr() : nullptr; }
Tensor or_empty(const OptTensor &t) { return given(t) ? *t : Tensor(); }
OptTensor opt(const Tensor &t) { return t.defined() ? OptTensor(t) : OptTensor(); }
Tensor none_like(const Tensor &t) { return at::empty({0}, t.options()); }

void check_rows(const Tensor &x, const char *name = "x")
{
    TORCH_CHECK(x.dim() >= 1 && x.is_contiguous(), "gcg: ", name, " must be a contiguous tensor of at least one dimension");
    (void)dtype_code(x.scalar_type());
}
int64_t rows_of(const Tensor &x) { return x.size(-1) ? x.numel() / x.size(-1) : 0; }
std::vector<int64_t> with_last(const Tensor &x, int64_t n)
{
    std::vector<int64_t> s = x.sizes().vec();
    s.back() = n;
    return s;
}

// ---- tensors in 8-bit floating point ----------------------------------------------------------------

int format_code(at::ScalarType t)
{
    TORCH_CHECK(t == at::kFloat8_e4m3fn || t == at::kFloat8_e5m2, "gcg: 8-bit tensors are float8_e4m3fn or float8_e5m2; got ", t);
    return t == at::kFloat8_e5m2 ? GCG_E5M2 : GCG_E4M3;
}
int64_t code_columns(int64_t D) { return (D + 127) / 128 * 128; }
int64_t scale_columns(int64_t D) { return (D + 511) / 512 * 4; }
uint8_t *bytes(const Tensor &t) { return (uint8_t *)t.data_ptr(); }

Two empty_float8(const Tensor &like, std::vector<int64_t> sizes, at::ScalarType format)
{
    const int64_t D = sizes.back();
    sizes.back() = code_columns(D);
    Tensor codes = at::empty(sizes, like.options().dtype(format));
    sizes.back() = scale_columns(D);
    return {codes, at::empty(sizes, like.options().dtype(at::kFloat8_e8m0fnu))};
}
void check_float8(const Tensor &codes, const Tensor &scales, int64_t columns)
{
    (void)format_code(codes.scalar_type());
    TORCH_CHECK(columns >= 0 && codes.dim() >= 1 && codes.is_contiguous() && codes.size(-1) == code_columns(columns),
                "gcg: the codes of ", columns, " columns must be contiguous rows of ", code_columns(columns));
    TORCH_CHECK(scales.scalar_type() == at::kFloat8_e8m0fnu && scales.is_contiguous() &&
                    scales.sizes() == at::IntArrayRef(with_last(codes, scale_columns(columns))),
                "gcg: the scales of ", columns, " columns must be contiguous float8_e8m0fnu rows of ", scale_columns(columns));
    TORCH_CHECK(scales.device() == codes.device(), "gcg: codes and scales must be on one device");
}

Two to_float8(const Tensor &x, at::ScalarType format)
{
    require_gpu(x, "x");
    check_rows(x);
    const int f = format_code(format);
    DeviceGuard guard(x.device());
    auto [codes, scales] = empty_float8(x, x.sizes().vec(), format);
    if (x.numel() == 0) return {codes, scales};
    check_rc(gcg_to_float8(x.data_ptr(), bytes(codes), bytes(scales), rows_of(x), x.size(-1), dtype_code(x.scalar_type()), f, stream_of(x)),
             "gcg_to_float8");
    return {codes, scales};
}

Tensor from_float8(const Tensor &codes, const Tensor &scales, int64_t columns, at::ScalarType dtype)
{
    require_gpu(codes, "codes");
    check_float8(codes, scales, columns);
    const int code = dtype_code(dtype);
    DeviceGuard guard(codes.device());
    Tensor x = at::empty(with_last(codes, columns), codes.options().dtype(dtype));
    if (x.numel() == 0) return x;
    check_rc(gcg_from_float8(bytes(codes), bytes(scales), x.data_ptr(), rows_of(x), columns, code, format_code(codes.scalar_type()),
                             stream_of(codes)),
             "gcg_from_float8");
    return x;
}

void check_matrix(const Tensor &x)
{
    check_rows(x);
    TORCH_CHECK(x.dim() == 2, "gcg: x must be a matrix");
}
// (codes, scales) of x along its rows, empty without `rows`, and of its columns
Four columns_outputs(const Tensor &x, int64_t R, int64_t D, at::ScalarType format, bool rows)
{
    auto [ct, st] = empty_float8(x, {D, R}, format);
    if (!rows) return {at::empty({0}, ct.options()), at::empty({0}, st.options()), ct, st};
    auto [c, s] = empty_float8(x, {R, D}, format);
    return {c, s, ct, st};
}
Four quantised_columns(const Tensor &x, at::ScalarType format, bool rows)
{
    require_gpu(x, "x");
    check_matrix(x);
    const int f = format_code(format);
    DeviceGuard guard(x.device());
    auto out = columns_outputs(x, x.size(0), x.size(1), format, rows);
    auto &[c, s, ct, st] = out;
    if (x.numel() == 0) return out;
    check_rc(gcg_to_float8_columns(x.data_ptr(), nullptr, rows ? bytes(c) : nullptr, rows ? bytes(s) : nullptr, bytes(ct), bytes(st), x.size(0),
                                   x.size(1), dtype_code(x.scalar_type()), f, stream_of(x)),
             "gcg_to_float8_columns");
    return out;
}
Four to_float8_both(const Tensor &x, at::ScalarType format) { return quantised_columns(x, format, true); }
Two to_float8_columns(const Tensor &x, at::ScalarType format)
{
    auto [c, s, ct, st] = quantised_columns(x, format, false);
    return {ct, st};
}
Two float8_columns(const Tensor &codes, const Tensor &scales, int64_t columns, at::ScalarType format)
{
    require_gpu(codes, "codes");
    check_float8(codes, scales, columns);
    TORCH_CHECK(codes.dim() == 2, "gcg: codes must be a matrix");
    const int f = format_code(format);
    DeviceGuard guard(codes.device());
    auto [ct, st] = empty_float8(codes, {columns, codes.size(0)}, format);
    if (ct.numel() == 0) return {ct, st};
    check_rc(gcg_to_float8_columns(codes.data_ptr(), bytes(scales), nullptr, nullptr, bytes(ct), bytes(st), codes.size(0), columns,
                                   format_code(codes.scalar_type()), f, stream_of(codes)),
             "gcg_to_float8_columns");
    return {ct, st};
}

int product_dtype(at::ScalarType t)
{
    TORCH_CHECK(t == at::kBFloat16 || t == at::kHalf, "gcg: products of 8-bit tensors are bfloat16 or float16; got ", t,
                " (the matrix instructions' own sums do not hold float32's bits)");
    return dtype_code(t);
}
void check_product(const Tensor &a, const Tensor &a_scales, const Tensor &b, const Tensor &b_scales, int64_t columns)
{
    check_float8(a, a_scales, columns);
    check_float8(b, b_scales, columns);
    TORCH_CHECK(b.dim() == 2 && b.device() == a.device(), "gcg: b must be a matrix on a's device");
    TORCH_CHECK(columns <= GCG_PRODUCT8_MAX_K, "gcg: a product over ", columns, " columns; at most ", (int)GCG_PRODUCT8_MAX_K, " are supported");
}
Tensor matmul_float8(const Tensor &a, const Tensor &a_scales, const Tensor &b, const Tensor &b_scales, int64_t columns, at::ScalarType dtype)
{
    require_gpu(a, "a");
    check_product(a, a_scales, b, b_scales, columns);
    const int code = product_dtype(dtype);
    DeviceGuard guard(a.device());
    const int64_t N = b.size(0);
    Tensor y = at::empty(with_last(a, N), a.options().dtype(dtype));
    if (y.numel() == 0) return y;
    if (columns == 0) return y.zero_();
    const int64_t M = y.numel() / N;
    const size_t need = gcg_product8_workspace_bytes(M, N, columns);
    const Tensor ws = need ? at::empty({(int64_t)need}, a.options().dtype(at::kByte)) : Tensor();
    check_rc(gcg_product8(bytes(a), bytes(a_scales), bytes(b), bytes(b_scales), y.data_ptr(), need ? ws.data_ptr() : nullptr, need, M, N,
                          columns, format_code(a.scalar_type()), format_code(b.scalar_type()), code, stream_of(a)),
             "gcg_product8");
    return y;
}

void check_linear(const Tensor &x, const Tensor &codes, const Tensor &scales, int64_t columns)
{
    check_rows(x);
    (void)product_dtype(x.scalar_type());
    check_float8(codes, scales, columns);
    TORCH_CHECK(codes.dim() == 2 && codes.device() == x.device() && x.size(-1) == columns,
                "gcg: the weight must be a matrix on x's device with as many columns as x");
}
Tensor linear_float8_infer(const Tensor &x, const Tensor &codes, const Tensor &scales, int64_t columns)
{
    require_gpu(x, "x");
    check_linear(x, codes, scales, columns);
    const int64_t M = rows_of(x), N = codes.size(0);
    if (!gcg_linear8_supported(M, N, columns)) {
        auto [c, s] = to_float8(x, at::kFloat8_e4m3fn);
        return matmul_float8(c, s, codes, scales, columns, x.scalar_type());
    }
    DeviceGuard guard(x.device());
    Tensor y = at::empty(with_last(x, N), x.options());
    check_rc(gcg_linear8(x.data_ptr(), bytes(codes), bytes(scales), y.data_ptr(), M, N, columns, format_code(codes.scalar_type()),
                         dtype_code(x.scalar_type()), stream_of(x)),
             "gcg_linear8");
    return y;
}

Two to_float8_meta(const Tensor &x, at::ScalarType format)
{
    check_rows(x);
    (void)format_code(format);
    return empty_float8(x, x.sizes().vec(), format);
}
Tensor from_float8_meta(const Tensor &codes, const Tensor &scales, int64_t columns, at::ScalarType dtype)
{
    check_float8(codes, scales, columns);
    (void)dtype_code(dtype);
    return at::empty(with_last(codes, columns), codes.options().dtype(dtype));
}
Four to_float8_both_meta(const Tensor &x, at::ScalarType format)
{
    check_matrix(x);
    (void)format_code(format);
    return columns_outputs(x, x.size(0), x.size(1), format, true);
}
Two to_float8_columns_meta(const Tensor &x, at::ScalarType format)
{
    check_matrix(x);
    (void)format_code(format);
    return empty_float8(x, {x.size(1), x.size(0)}, format);
}
Two float8_columns_meta(const Tensor &codes, const Tensor &scales, int64_t columns, at::ScalarType format)
{
    check_float8(codes, scales, columns);
    (void)format_code(format);
    return empty_float8(codes, {columns, codes.size(0)}, format);
}
Tensor matmul_float8_meta(const Tensor &a, const Tensor &a_scales, const Tensor &b, const Tensor &b_scales, int64_t columns, at::ScalarType dtype)
{
    check_product(a, a_scales, b, b_scales, columns);
    (void)product_dtype(dtype);
    return at::empty(with_last(a, b.size(0)), a.options().dtype(dtype));
}
Tensor linear_float8_infer_meta(const Tensor &x, const Tensor &codes, const Tensor &scales, int64_t columns)
{
    check_linear(x, codes, scales, columns);
    return at::empty(with_last(x, codes.size(0)), x.options());
}

// ---- root-mean-square norm ------------------------------------------------------------------------------

// the library's code for x with this weight; also checks them and the residual
int rms_code(const Tensor &x, const OptTensor &residual, const OptTensor &w)
{
    check_rows(x);
    TORCH_CHECK(x.size(-1) > 0, "gcg: norm over an empty dimension");
    TORCH_CHECK(x.size(-1) <= GCG_NORM_MAX_WIDTH, "gcg: norm over ", x.size(-1), " elements; at most ", (int)GCG_NORM_MAX_WIDTH,
                " are supported");
    if (given(residual))
        TORCH_CHECK(residual->sizes() == x.sizes() && residual->scalar_type() == x.scalar_type() && residual->device() == x.device() &&
                        residual->is_contiguous(),
                    "gcg: the residual must be a contiguous tensor with the shape, dtype and device of x");
    const int code = dtype_code(x.scalar_type());
    if (!given(w)) return code;
    TORCH_CHECK(w->dim() == 1 && w->size(0) == x.size(-1) && w->is_contiguous() && w->device() == x.device(),
                "gcg: the weight must be contiguous, on x's device and of the size of x's last dimension");
    TORCH_CHECK(w->scalar_type() == x.scalar_type() || w->scalar_type() == at::kFloat,
                "gcg: the weight must have x's dtype or be float32; got ", w->scalar_type(), " with ", x.scalar_type());
    if (w->scalar_type() == x.scalar_type()) return code;
    return code == GCG_BF16 ? GCG_BF16_F32 : GCG_F16_F32;
}
std::vector<int64_t> rstd_sizes(const Tensor &x) { return x.sizes().slice(0, x.dim() - 1).vec(); }

void rms_launch(const Tensor &x, const OptTensor &residual, const OptTensor &w, double eps, int code, void *y, const Tensor &r, uint8_t *codes,
                uint8_t *scales, float *rstd)
{
    if (x.numel() == 0) return;
    check_rc(gcg_rms_norm_fwd(x.data_ptr(), ptr(residual), ptr(w), y, given(residual) ? r.data_ptr() : nullptr, codes, scales, rstd, rows_of(x),
                              (int32_t)x.size(-1), (float)eps, code, stream_of(x)),
             "gcg_rms_norm_fwd");
}
Tensor new_sum(const Tensor &x, const OptTensor &residual) { return given(residual) ? at::empty_like(x) : none_like(x); }

Three rms_norm_fwd(const Tensor &x, const OptTensor &residual, const OptTensor &w, double eps)
{
    require_gpu(x, "x");
    const int code = rms_code(x, residual, w);
    DeviceGuard guard(x.device());
    Tensor y = at::empty_like(x), r = new_sum(x, residual), rstd = at::empty(rstd_sizes(x), x.options().dtype(at::kFloat));
    rms_launch(x, residual, w, eps, code, y.data_ptr(), r, nullptr, nullptr, (float *)rstd.data_ptr());
    return {y, r, rstd};
}
// without what only a backward asks for
Two rms_norm_infer(const Tensor &x, const OptTensor &residual, const OptTensor &w, double eps)
{
    require_gpu(x, "x");
    const int code = rms_code(x, residual, w);
    DeviceGuard guard(x.device());
    Tensor y = at::empty_like(x), r = new_sum(x, residual);
    rms_launch(x, residual, w, eps, code, y.data_ptr(), r, nullptr, nullptr, nullptr);
    return {y, r};
}
Four rms_norm_float8(const Tensor &x, const OptTensor &residual, const OptTensor &w, double eps)
{
    require_gpu(x, "x");
    const int code = rms_code(x, residual, w);
    DeviceGuard guard(x.device());
    auto [codes, scales] = empty_float8(x, x.sizes().vec(), at::kFloat8_e4m3fn);
    Tensor r = new_sum(x, residual), rstd = at::empty(rstd_sizes(x), x.options().dtype(at::kFloat));
    rms_launch(x, residual, w, eps, code, nullptr, r, bytes(codes), bytes(scales), (float *)rstd.data_ptr());
    return {codes, scales, r, rstd};
}

// the norm and a product with a weight in 8 bits: (y, r)
Two norm_linear_float8_infer(const Tensor &x, const OptTensor &residual, const OptTensor &gain, const Tensor &codes, const Tensor &scales,
                             int64_t columns, double eps)
{
    require_gpu(x, "x");
    const int code = rms_code(x, residual, gain);
    check_linear(x, codes, scales, columns);
    DeviceGuard guard(x.device());
    auto [c, s] = empty_float8(x, x.sizes().vec(), at::kFloat8_e4m3fn);
    Tensor r = new_sum(x, residual);
    rms_launch(x, residual, gain, eps, code, nullptr, r, bytes(c), bytes(s), nullptr);
    return {matmul_float8(c, s, codes, scales, columns, x.scalar_type()), r};
}

void check_rms_bwd(const Tensor &dy, const Tensor &r, const OptTensor &dr, const Tensor &rstd)
{
    check_rows(dy, "dy");
    for (const Tensor *t : {&r, given(dr) ? &*dr : &dy})
        TORCH_CHECK(t->sizes() == dy.sizes() && t->scalar_type() == dy.scalar_type() && t->device() == dy.device() && t->is_contiguous(),
                    "gcg: dy and dr must be contiguous tensors with the shape, dtype and device of r");
    TORCH_CHECK(rstd.sizes() == at::IntArrayRef(rstd_sizes(dy)) && rstd.scalar_type() == at::kFloat && rstd.is_contiguous() &&
                    rstd.device() == dy.device(),
                "gcg: rstd must be the forward's");
}
// (dx, dw); dw is empty without w, or where it is not needed
Two rms_norm_bwd(const Tensor &dy, const Tensor &r, const OptTensor &dr, const Tensor &rstd, const OptTensor &w, bool need_dw)
{
    require_gpu(dy, "dy");
    check_rms_bwd(dy, r, dr, rstd);
    const int code = rms_code(dy, OptTensor(), w);
    DeviceGuard guard(dy.device());
    const int64_t rows = rows_of(dy);
    need_dw = need_dw && given(w);
    Tensor dx = at::empty_like(dy), dw = need_dw ? at::empty_like(*w) : none_like(dy);
    if (rows == 0) return {dx, dw.zero_()};
    const size_t need = need_dw ? gcg_rms_norm_bwd_workspace_bytes(rows, (int32_t)dy.size(-1), code) : 0;
    const Tensor ws = need_dw ? workspace(need, dy, "gcg_rms_norm_bwd_workspace_bytes") : Tensor();
    check_rc(gcg_rms_norm_bwd(dy.data_ptr(), r.data_ptr(), ptr(dr), (const float *)rstd.data_ptr(), ptr(w), dx.data_ptr(),
                              need_dw ? dw.data_ptr() : nullptr, need ? ws.data_ptr() : nullptr, need, rows, (int32_t)dy.size(-1), code,
                              stream_of(dy)),
             "gcg_rms_norm_bwd");
    return {dx, dw};
}

Three rms_norm_fwd_meta(const Tensor &x, const OptTensor &residual, const OptTensor &w, double)
{
    (void)rms_code(x, residual, w);
    return {at::empty_like(x), new_sum(x, residual), at::empty(rstd_sizes(x), x.options().dtype(at::kFloat))};
}
Two rms_norm_infer_meta(const Tensor &x, const OptTensor &residual, const OptTensor &w, double)
{
    (void)rms_code(x, residual, w);
    return {at::empty_like(x), new_sum(x, residual)};
}
Four rms_norm_float8_meta(const Tensor &x, const OptTensor &residual, const OptTensor &w, double)
{
    (void)rms_code(x, residual, w);
    auto [codes, scales] = empty_float8(x, x.sizes().vec(), at::kFloat8_e4m3fn);
    return {codes, scales, new_sum(x, residual), at::empty(rstd_sizes(x), x.options().dtype(at::kFloat))};
}
Two norm_linear_float8_infer_meta(const Tensor &x, const OptTensor &residual, const OptTensor &gain, const Tensor &codes, const Tensor &scales,
                                  int64_t columns, double)
{
    (void)rms_code(x, residual, gain);
    check_linear(x, codes, scales, columns);
    return {at::empty(with_last(x, codes.size(0)), x.options()), new_sum(x, residual)};
}
Two rms_norm_bwd_meta(const Tensor &dy, const Tensor &r, const OptTensor &dr, const Tensor &rstd, const OptTensor &w, bool need_dw)
{
    check_rms_bwd(dy, r, dr, rstd);
    (void)rms_code(dy, OptTensor(), w);
    return {at::empty_like(dy), need_dw && given(w) ? at::empty_like(*w) : none_like(dy)};
}

// ---- gated linear recurrence ------------------------------------------------------------------------------

// a tensor whose last dimension is contiguous and whose rows are near enough to each other, as the kernels read it
Tensor read_rows(const Tensor &t)
{
    const bool in_place = (t.size(-1) == 1 || t.stride(-1) == 1) && (t.dim() < 3 || t.stride(1) <= GCG_SCAN_MAX_TIME_STRIDE);
    return in_place ? t : t.contiguous();
}
void check_scan(const Tensor &x, const Tensor &f, const OptTensor &gate, const OptTensor &bias, int64_t dim)
{
    TORCH_CHECK(x.dim() == dim && f.sizes() == x.sizes() && (!given(gate) || gate->sizes() == x.sizes()),
                dim == 3 ? "gcg: x, f and gate must be (bs, L, D)" : "gcg: x, f and gate must be (bs, D)");
    TORCH_CHECK(f.scalar_type() == x.scalar_type() && f.device() == x.device() &&
                    (!given(gate) || (gate->scalar_type() == x.scalar_type() && gate->device() == x.device())),
                "gcg: x, f and gate must share dtype and device");
    (void)dtype_code(x.scalar_type());
    if (given(bias))
        TORCH_CHECK(bias->dim() == 1 && bias->size(0) == x.size(-1) && bias->scalar_type() == at::kFloat && bias->is_contiguous() &&
                        bias->device() == x.device(),
                    "gcg: bias must be a contiguous float32 tensor of one element a channel on x's device");
    TORCH_CHECK(x.size(-1) > 0 && x.size(-1) <= GCG_SCAN_MAX_WIDTH, "gcg: ", x.size(-1), " channels; 1 to ", (int)GCG_SCAN_MAX_WIDTH,
                " are supported");
    TORCH_CHECK(dim == 2 || x.size(1) <= GCG_SCAN_MAX_ROWS, "gcg: ", x.size(1), " rows; at most ", (int)GCG_SCAN_MAX_ROWS, " are supported");
}
void check_scan_state(const OptTensor &t, const Tensor &x, const char *name)
{
    if (!given(t)) return;
    TORCH_CHECK(t->dim() == 2 && t->size(0) == x.size(0) && t->size(1) == x.size(-1) && t->scalar_type() == at::kFloat && t->is_contiguous() &&
                    t->device() == x.device(),
                "gcg: ", name, " must be a contiguous (bs, D) float32 tensor on x's device");
}
void check_scan_lengths(const OptTensor &t, const Tensor &x)
{
    if (!given(t)) return;
    TORCH_CHECK(t->dim() == 1 && t->size(0) == x.size(0) && t->scalar_type() == at::kInt && t->is_contiguous() && t->device() == x.device(),
                "gcg: lengths must be a contiguous int32 tensor of one element a batch entry on x's device");
}
std::vector<int64_t> state_sizes(const Tensor &x, bool wanted) { return wanted ? std::vector<int64_t>{x.size(0), x.size(-1)} : std::vector<int64_t>{0}; }
std::vector<int64_t> kept_sizes(const Tensor &x, bool wanted)
{
    return wanted ? std::vector<int64_t>{x.size(0), gcg_scan_states(x.size(1)), x.size(2)} : std::vector<int64_t>{0};
}
void add_strides(std::vector<int64_t> &s, const Tensor &t)
{
    s.insert(s.end(), {t.defined() ? t.stride(0) : 0, t.defined() ? t.stride(1) : 0});
}
Tensor scan_workspace(const Tensor &x, bool backward, size_t *n)
{
    *n = gcg_scan_workspace_bytes(x.size(0), x.size(1), (int32_t)x.size(2), backward);
    return *n ? at::empty({(int64_t)*n}, x.options().dtype(at::kByte)) : Tensor();
}
// a sequence of no rows: the state is the one given
Tensor passed_on(const OptTensor &from, Tensor to) { return to.numel() == 0 ? to : given(from) ? to.copy_(*from) : to.zero_(); }

// (y, final state, kept states); what is not asked for is empty
Three scan_fwd(const Tensor &x, const Tensor &f, const OptTensor &gate, const OptTensor &bias, const OptTensor &initial, const OptTensor &lengths,
               bool final, bool keep)
{
    require_gpu(x, "x");
    check_scan(x, f, gate, bias, 3);
    check_scan_state(initial, x, "initial_state");
    check_scan_lengths(lengths, x);
    DeviceGuard guard(x.device());
    const auto f32 = x.options().dtype(at::kFloat);
    Tensor y = at::empty(x.sizes(), x.options()), last = at::empty(state_sizes(x, final), f32), states = at::empty(kept_sizes(x, keep), f32);
    if (y.numel() == 0) return {y, passed_on(initial, last), states};
    const Tensor a = read_rows(x), b = read_rows(f), c = given(gate) ? read_rows(*gate) : Tensor();
    std::vector<int64_t> s;
    for (const Tensor *t : {&a, &b, &c, (const Tensor *)&y}) add_strides(s, *t);
    size_t n;
    const Tensor ws = scan_workspace(x, false, &n);
    check_rc(gcg_scan_fwd(a.data_ptr(), b.data_ptr(), c.defined() ? c.data_ptr() : nullptr, s.data(), (const float *)ptr(bias),
                          (const float *)ptr(initial), (const int32_t *)ptr(lengths), y.data_ptr(), final ? (float *)last.data_ptr() : nullptr,
                          keep ? (float *)states.data_ptr() : nullptr, n ? ws.data_ptr() : nullptr, n, x.size(0), x.size(1), (int32_t)x.size(2),
                          dtype_code(x.scalar_type()), stream_of(x)),
             "gcg_scan_fwd");
    return {y, last, states};
}

void check_scan_bwd(const Tensor &dy, const Tensor &x, const Tensor &states, const OptTensor &dfinal, const OptTensor &lengths)
{
    TORCH_CHECK(dy.sizes() == x.sizes() && dy.scalar_type() == x.scalar_type() && dy.device() == x.device(),
                "gcg: dy must have the shape, dtype and device of x");
    TORCH_CHECK(states.sizes() == at::IntArrayRef(kept_sizes(x, true)) && states.scalar_type() == at::kFloat && states.is_contiguous() &&
                    states.device() == x.device(),
                "gcg: states must be the forward's");
    check_scan_state(dfinal, x, "the final state's gradient");
    check_scan_lengths(lengths, x);
}
void scan_bwd_into(const Tensor &dy, const Tensor &x, const Tensor &f, const OptTensor &gate, const OptTensor &bias, const Tensor &states,
                   const OptTensor &lengths, const OptTensor &dfinal, const Tensor &dx, const Tensor &df, const Tensor &dgate, float *dbias,
                   float *dinitial)
{
    const Tensor d = read_rows(dy), a = read_rows(x), b = read_rows(f), c = given(gate) ? read_rows(*gate) : Tensor();
    const Tensor none, &dg = given(gate) ? dgate : none;
    std::vector<int64_t> s;
    for (const Tensor *t : {&d, &a, &b, &c, &dx, &df, &dg}) add_strides(s, *t);
    size_t n;
    const Tensor ws = scan_workspace(x, true, &n);
    check_rc(gcg_scan_bwd(d.data_ptr(), a.data_ptr(), b.data_ptr(), c.defined() ? c.data_ptr() : nullptr, s.data(), (const float *)ptr(bias),
                          (const float *)states.data_ptr(), (const int32_t *)ptr(lengths), (const float *)ptr(dfinal), dx.data_ptr(),
                          df.data_ptr(), dg.defined() ? dg.data_ptr() : nullptr, dbias, dinitial, n ? ws.data_ptr() : nullptr, n, x.size(0),
                          x.size(1), (int32_t)x.size(2), dtype_code(x.scalar_type()), stream_of(x)),
             "gcg_scan_bwd");
}
Five scan_gradients(const Tensor &x, const OptTensor &gate, bool need_dbias, bool need_dinitial)
{
    const auto f32 = x.options().dtype(at::kFloat);
    return {at::empty(x.sizes(), x.options()), at::empty(x.sizes(), x.options()), given(gate) ? at::empty(x.sizes(), x.options()) : none_like(x),
            need_dbias ? at::empty({x.size(-1)}, f32) : at::empty({0}, f32), at::empty(state_sizes(x, need_dinitial), f32)};
}
// (dx, df, dgate, dbias, dinitial); what is not asked for is empty
Five scan_bwd(const Tensor &dy, const Tensor &x, const Tensor &f, const OptTensor &gate, const OptTensor &bias, const Tensor &states,
              const OptTensor &lengths, const OptTensor &dfinal, bool need_dbias, bool need_dinitial)
{
    require_gpu(x, "x");
    check_scan(x, f, gate, bias, 3);
    check_scan_bwd(dy, x, states, dfinal, lengths);
    DeviceGuard guard(x.device());
    auto out = scan_gradients(x, gate, need_dbias, need_dinitial);
    auto &[dx, df, dg, db, di] = out;
    if (x.numel() == 0) {
        db.zero_();
        passed_on(dfinal, di);
        return out;
    }
    scan_bwd_into(dy, x, f, gate, bias, states, lengths, dfinal, dx, df, dg, need_dbias ? (float *)db.data_ptr() : nullptr,
                  need_dinitial ? (float *)di.data_ptr() : nullptr);
    return out;
}

// the projected features (bs, L, 3 * D), laid out "(p d)" with p = x, f, gate
Three split_features(const Tensor &features)
{
    TORCH_CHECK(features.dim() == 3 && features.is_contiguous() && features.size(2) % 3 == 0,
                "gcg: features must be a contiguous (bs, L, 3 * D) tensor");
    const int64_t D = features.size(2) / 3;
    return {features.slice(2, 0, D), features.slice(2, D, 2 * D), features.slice(2, 2 * D, 3 * D)};
}
Two scan_packed_fwd(const Tensor &features, const OptTensor &bias, bool keep)
{
    require_gpu(features, "features");
    const auto [x, f, gate] = split_features(features);
    auto [y, last, states] = scan_fwd(x, f, gate, bias, OptTensor(), OptTensor(), false, keep);
    return {y, states};
}
Two scan_packed_bwd(const Tensor &dy, const Tensor &features, const OptTensor &bias, const Tensor &states, bool need_dbias)
{
    require_gpu(features, "features");
    const auto [x, f, gate] = split_features(features);
    check_scan(x, f, gate, bias, 3);
    check_scan_bwd(dy, x, states, OptTensor(), OptTensor());
    DeviceGuard guard(features.device());
    Tensor df = at::empty_like(features), db = at::empty({need_dbias ? x.size(2) : 0}, features.options().dtype(at::kFloat));
    if (df.numel() == 0) return {df, db.zero_()};
    const auto [dx, dff, dg] = split_features(df);
    scan_bwd_into(dy, x, f, gate, bias, states, OptTensor(), OptTensor(), dx, dff, dg, need_dbias ? (float *)db.data_ptr() : nullptr, nullptr);
    return {df, db};
}

Tensor scan_step(const Tensor &x, const Tensor &f, const OptTensor &gate, const OptTensor &bias, Tensor &state)
{
    require_gpu(x, "x");
    check_scan(x, f, gate, bias, 2);
    check_scan_state(state, x, "state");
    DeviceGuard guard(x.device());
    Tensor y = at::empty(x.sizes(), x.options());
    if (y.numel() == 0) return y;
    const Tensor a = read_rows(x), b = read_rows(f), c = given(gate) ? read_rows(*gate) : Tensor();
    const int64_t s[3] = {a.stride(0), b.stride(0), c.defined() ? c.stride(0) : 0};
    check_rc(gcg_scan_step(a.data_ptr(), b.data_ptr(), c.defined() ? c.data_ptr() : nullptr, s, (const float *)ptr(bias), (float *)state.data_ptr(),
                           y.data_ptr(), x.size(0), (int32_t)x.size(1), dtype_code(x.scalar_type()), stream_of(x)),
             "gcg_scan_step");
    return y;
}
// As in-place operators of torch are: whatever saved the state for a backward pass finds it modified.  (An inference tensor has no such
// count, and nothing can have saved it.)
Tensor scan_step_in_place(const Tensor &x, const Tensor &f, const OptTensor &gate, const OptTensor &bias, Tensor &state)
{
    static const auto step = op<Tensor(const Tensor &, const Tensor &, const OptTensor &, const OptTensor &, Tensor &)>("gcg::scan_step");
    Tensor y;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        y = step.call(x, f, gate, bias, state);
    }
    if (!state.is_inference()) torch::autograd::impl::bump_version(state);
    return y;
}

Three scan_fwd_meta(const Tensor &x, const Tensor &f, const OptTensor &gate, const OptTensor &bias, const OptTensor &initial,
                    const OptTensor &lengths, bool final, bool keep)
{
    check_scan(x, f, gate, bias, 3);
    check_scan_state(initial, x, "initial_state");
    check_scan_lengths(lengths, x);
    const auto f32 = x.options().dtype(at::kFloat);
    return {at::empty(x.sizes(), x.options()), at::empty(state_sizes(x, final), f32), at::empty(kept_sizes(x, keep), f32)};
}
Five scan_bwd_meta(const Tensor &dy, const Tensor &x, const Tensor &f, const OptTensor &gate, const OptTensor &bias, const Tensor &states,
                   const OptTensor &lengths, const OptTensor &dfinal, bool need_dbias, bool need_dinitial)
{
    check_scan(x, f, gate, bias, 3);
    check_scan_bwd(dy, x, states, dfinal, lengths);
    return scan_gradients(x, gate, need_dbias, need_dinitial);
}
Two scan_packed_fwd_meta(const Tensor &features, const OptTensor &bias, bool keep)
{
    const auto [x, f, gate] = split_features(features);
    check_scan(x, f, gate, bias, 3);
    return {at::empty(x.sizes(), x.options()), at::empty(kept_sizes(x, keep), x.options().dtype(at::kFloat))};
}
Two scan_packed_bwd_meta(const Tensor &dy, const Tensor &features, const OptTensor &bias, const Tensor &states, bool need_dbias)
{
    const auto [x, f, gate] = split_features(features);
    check_scan(x, f, gate, bias, 3);
    check_scan_bwd(dy, x, states, OptTensor(), OptTensor());
    return {at::empty_like(features), at::empty({need_dbias ? x.size(2) : 0}, features.options().dtype(at::kFloat))};
}
Tensor scan_step_meta(const Tensor &x, const Tensor &f, const OptTensor &gate, const OptTensor &bias, Tensor &state)
{
    check_scan(x, f, gate, bias, 2);
    check_scan_state(state, x, "state");
    return at::empty(x.sizes(), x.options());
}

// ---- autograd nodes ------------------------------------------------------------------------------------------
// Each calls the operators above through the dispatcher, below autograd; a backward pass that is recorded itself (create_graph) calls them above it,
// where those without a derivative say so.
struct BelowAutograd {
    std::optional<at::AutoDispatchBelowADInplaceOrView> below;
    BelowAutograd() { if (!at::GradMode::is_enabled()) below.emplace(); }
};

// A leaf whose gradient is still the business of a graph that was recorded on the default stream takes a captured backward pass there, which ends
// the capture, and with it the process: such a call is refused.
void check_leaves(std::initializer_list<const Tensor *> tensors)
{
    if (!(*tensors.begin())->is_cuda() || c10::hip::currentStreamCaptureStatusMayInitCtx() == c10::hip::CaptureStatus::None) return;
    for (const Tensor *t : tensors) {
        if (!t->defined() || !t->requires_grad() || !t->is_leaf()) continue;
        const auto node = torch::autograd::impl::try_get_grad_accumulator(*t);
        const auto stream = node ? node->stream() : std::nullopt;
        TORCH_CHECK(!stream || stream->id() != 0, "gcg: the stream is being captured into a graph, and an argument is a leaf of a graph that was "
                    "recorded on the default stream and still lives; let that graph go before the capture");
    }
}

struct RmsNormNode : torch::autograd::Function<RmsNormNode> {
    static variable_list forward(AutogradContext *ctx, const Tensor &x, const OptTensor &residual, const OptTensor &w, double eps)
    {
        static const auto f = op<Three(const Tensor &, const OptTensor &, const OptTensor &, double)>("gcg::rms_norm_fwd");
        at::AutoDispatchBelowADInplaceOrView below;
        auto [y, r, rstd] = f.call(x, residual, w, eps);
        ctx->set_materialize_grads(false);
        ctx->save_for_backward({given(residual) ? r : x, rstd, or_empty(w)});
        ctx->saved_data["dw"] = given(w) && w->requires_grad();
        if (given(residual)) return {y, r};
        return {y};
    }
    static variable_list backward(AutogradContext *ctx, variable_list g)
    {
        const BelowAutograd below;
        static const auto f = op<Two(const Tensor &, const Tensor &, const OptTensor &, const Tensor &, const OptTensor &, bool)>("gcg::rms_norm_bwd");
        const variable_list s = ctx->get_saved_variables();
        const bool need = ctx->saved_data["dw"].toBool(), added = g.size() > 1;
        const Tensor dy = g[0].defined() ? g[0].contiguous() : at::zeros_like(s[0]);
        const OptTensor dr = added && g[1].defined() ? OptTensor(g[1].contiguous()) : OptTensor();
        auto [dx, dw] = f.call(dy, s[0], dr, s[1], opt(s[2]), need);
        return {dx, added ? dx : Tensor(), need ? dw : Tensor(), Tensor()};
    }
};

// The norm into 8 bits with a residual: (codes, scales, r), of which r, a sum, is differentiable.
struct StreamNode : torch::autograd::Function<StreamNode> {
    static variable_list forward(AutogradContext *ctx, const Tensor &x, const Tensor &residual, const OptTensor &w, double eps)
    {
        static const auto f = op<Four(const Tensor &, const OptTensor &, const OptTensor &, double)>("gcg::rms_norm_float8");
        at::AutoDispatchBelowADInplaceOrView below;
        auto [codes, scales, r, rstd] = f.call(x, residual, w, eps);
        ctx->set_materialize_grads(false);
        ctx->mark_non_differentiable({codes, scales});
        return {codes, scales, r};
    }
    static variable_list backward(AutogradContext *, variable_list g) { return {g[2], g[2], Tensor(), Tensor()}; }
};

// (the rows counted from x's sizes: a matrix of no columns has some)
Tensor as_matrix(const Tensor &t)
{
    int64_t rows = 1;
    for (int64_t i = 0; i + 1 < t.dim(); ++i) rows *= t.size(i);
    return t.reshape({rows, t.size(-1)});
}
// dx and dw of y = x w^T from x in 8 bits, each operand in 8 bits along what it is summed over; dy: (rows, out)
Two linear_gradients(const Tensor &dy, const Tensor &codes, const Tensor &scales, int64_t columns, const Tensor &w, at::ScalarType format,
                     bool need_dx, bool need_dw)
{
    static const auto both = op<Four(const Tensor &, at::ScalarType)>("gcg::to_float8_both");
    static const auto rows = op<Two(const Tensor &, at::ScalarType)>("gcg::to_float8");
    static const auto cols = op<Two(const Tensor &, at::ScalarType)>("gcg::to_float8_columns");
    static const auto again = op<Two(const Tensor &, const Tensor &, int64_t, at::ScalarType)>("gcg::float8_columns");
    static const auto mul = op<Tensor(const Tensor &, const Tensor &, const Tensor &, const Tensor &, int64_t, at::ScalarType)>("gcg::matmul_float8");
    Tensor c, s, ct, st, dx, dw;
    if (need_dx && need_dw) std::tie(c, s, ct, st) = both.call(dy, format);
    else if (need_dx) std::tie(c, s) = rows.call(dy, format);
    else if (need_dw) std::tie(ct, st) = cols.call(dy, format);
    if (need_dx) {
        auto [wc, ws] = cols.call(w, at::kFloat8_e4m3fn);
        dx = mul.call(c, s, wc, ws, dy.size(1), dy.scalar_type());
    }
    if (need_dw) {
        auto [xc, xs] = again.call(codes, scales, columns, at::kFloat8_e4m3fn);
        dw = mul.call(ct, st, xc, xs, dy.size(0), dy.scalar_type());
    }
    return {dx, dw};
}
// checks a weight in the tensors' type; others: the norm's, whose gradients are formed of x's
void check_weight(const Tensor &x, const Tensor &w, const Tensor &residual = {}, const Tensor &gain = {})
{
    (void)product_dtype(x.scalar_type());
    TORCH_CHECK(w.dim() == 2 && w.size(1) == x.size(-1) && w.scalar_type() == x.scalar_type() && w.device() == x.device(),
                "gcg: the weight must be a (out, in) matrix with the dtype and device of x");
    if (!at::GradMode::is_enabled()) return;
    const auto needs = [](const Tensor &t) { return t.defined() && t.requires_grad(); };
    TORCH_CHECK(rows_of(x) <= GCG_PRODUCT8_MAX_K || !needs(w), "gcg: the weight's gradient is a sum over ", rows_of(x), " rows; at most ",
                (int)GCG_PRODUCT8_MAX_K, " are supported");
    TORCH_CHECK(w.size(0) <= GCG_PRODUCT8_MAX_K || !(needs(x) || needs(residual) || needs(gain)), "gcg: x's gradient is a sum over ", w.size(0),
                " outputs; at most ", (int)GCG_PRODUCT8_MAX_K, " are supported");
}

struct LinearFloat8Node : torch::autograd::Function<LinearFloat8Node> {
    static Tensor forward(AutogradContext *ctx, const Tensor &x, const Tensor &w, at::ScalarType format)
    {
        static const auto rows = op<Two(const Tensor &, at::ScalarType)>("gcg::to_float8");
        static const auto mul = op<Tensor(const Tensor &, const Tensor &, const Tensor &, const Tensor &, int64_t, at::ScalarType)>("gcg::matmul_float8");
        at::AutoDispatchBelowADInplaceOrView below;
        const Tensor wc = w.contiguous();
        auto [c, s] = rows.call(x.contiguous(), at::kFloat8_e4m3fn);
        auto [bc, bs] = rows.call(wc, at::kFloat8_e4m3fn);
        const bool need_dw = w.requires_grad();
        ctx->save_for_backward({need_dw ? c : Tensor(), need_dw ? s : Tensor(), wc});
        ctx->saved_data["dx"] = x.requires_grad();
        ctx->saved_data["dw"] = need_dw;
        ctx->saved_data["format"] = (int64_t)format;
        return mul.call(c, s, bc, bs, x.size(-1), x.scalar_type());
    }
    static variable_list backward(AutogradContext *ctx, variable_list g)
    {
        const BelowAutograd below;
        const variable_list s = ctx->get_saved_variables();
        const bool need_dx = ctx->saved_data["dx"].toBool(), need_dw = ctx->saved_data["dw"].toBool();
        const Tensor &w = s[2], dy = g[0].contiguous();
        const Tensor flat = need_dw ? as_matrix(s[0]) : Tensor(), scales = need_dw ? as_matrix(s[1]) : Tensor();
        auto [dx, dw] = linear_gradients(as_matrix(dy), flat, scales, w.size(1), w,
                                         (at::ScalarType)ctx->saved_data["format"].toInt(), need_dx, need_dw);
        if (need_dx) {
            std::vector<int64_t> sizes = dy.sizes().vec();
            sizes.back() = w.size(1);
            dx = dx.reshape(sizes);
        }
        return {dx, dw, Tensor()};
    }
};

struct NormLinearFloat8Node : torch::autograd::Function<NormLinearFloat8Node> {
    static variable_list forward(AutogradContext *ctx, const Tensor &x, const OptTensor &residual, const OptTensor &gain, const Tensor &w, double eps,
                                 at::ScalarType format)
    {
        static const auto norm = op<Four(const Tensor &, const OptTensor &, const OptTensor &, double)>("gcg::rms_norm_float8");
        static const auto rows = op<Two(const Tensor &, at::ScalarType)>("gcg::to_float8");
        static const auto mul = op<Tensor(const Tensor &, const Tensor &, const Tensor &, const Tensor &, int64_t, at::ScalarType)>("gcg::matmul_float8");
        at::AutoDispatchBelowADInplaceOrView below;
        const Tensor wc = w.contiguous();
        auto [c, s, r, rstd] = norm.call(x, residual, gain, eps);
        auto [bc, bs] = rows.call(wc, at::kFloat8_e4m3fn);
        const bool need_dw = w.requires_grad();
        ctx->set_materialize_grads(false);
        ctx->save_for_backward({need_dw ? c : Tensor(), need_dw ? s : Tensor(), wc, given(residual) ? r : x, rstd, or_empty(gain)});
        ctx->saved_data["dx"] = x.requires_grad() || (given(residual) && residual->requires_grad()) || (given(gain) && gain->requires_grad());
        ctx->saved_data["dw"] = need_dw;
        ctx->saved_data["dgain"] = given(gain) && gain->requires_grad();
        ctx->saved_data["format"] = (int64_t)format;
        const Tensor y = mul.call(c, s, bc, bs, x.size(-1), x.scalar_type());
        if (given(residual)) return {y, r};
        return {y};
    }
    static variable_list backward(AutogradContext *ctx, variable_list g)
    {
        const BelowAutograd below;
        static const auto norm = op<Two(const Tensor &, const Tensor &, const OptTensor &, const Tensor &, const OptTensor &, bool)>("gcg::rms_norm_bwd");
        const variable_list s = ctx->get_saved_variables();
        const Tensor &w = s[2], &r = s[3];
        const bool need_dx = ctx->saved_data["dx"].toBool(), need_dw = ctx->saved_data["dw"].toBool(), need_gain = ctx->saved_data["dgain"].toBool();
        const bool added = g.size() > 1;
        std::vector<int64_t> sizes = r.sizes().vec();
        sizes.back() = w.size(0);
        const Tensor dy = g[0].defined() ? g[0].contiguous() : at::zeros(sizes, r.options());
        const Tensor flat = need_dw ? as_matrix(s[0]) : Tensor(), scales = need_dw ? as_matrix(s[1]) : Tensor();
        auto [dn, dw] = linear_gradients(as_matrix(dy), flat, scales, w.size(1), w,
                                         (at::ScalarType)ctx->saved_data["format"].toInt(), need_dx, need_dw);
        Tensor dx, dgain;
        if (need_dx) {
            const OptTensor dr = added && g[1].defined() ? OptTensor(g[1].contiguous()) : OptTensor();
            std::tie(dx, dgain) = norm.call(dn.reshape(r.sizes()), r, dr, s[4], opt(s[5]), need_gain);
        }
        return {dx, added ? dx : Tensor(), need_gain ? dgain : Tensor(), dw, Tensor(), Tensor()};
    }
};

struct ScanNode : torch::autograd::Function<ScanNode> {
    static variable_list forward(AutogradContext *ctx, const Tensor &x, const Tensor &f, const OptTensor &gate, const OptTensor &bias,
                                 const OptTensor &initial, const OptTensor &lengths, bool final)
    {
        static const auto fwd = op<Three(const Tensor &, const Tensor &, const OptTensor &, const OptTensor &, const OptTensor &, const OptTensor &,
                                         bool, bool)>("gcg::scan_fwd");
        at::AutoDispatchBelowADInplaceOrView below;
        auto [y, last, states] = fwd.call(x, f, gate, bias, initial, lengths, final, true);
        ctx->set_materialize_grads(false);
        ctx->save_for_backward({x, f, or_empty(gate), or_empty(bias), states, or_empty(lengths)});
        ctx->saved_data["dbias"] = given(bias) && bias->requires_grad();
        ctx->saved_data["dinitial"] = given(initial) && initial->requires_grad();
        if (final) return {y, last};
        return {y};
    }
    static variable_list backward(AutogradContext *ctx, variable_list g)
    {
        const BelowAutograd below;
        static const auto bwd = op<Five(const Tensor &, const Tensor &, const Tensor &, const OptTensor &, const OptTensor &, const Tensor &,
                                        const OptTensor &, const OptTensor &, bool, bool)>("gcg::scan_bwd");
        const variable_list s = ctx->get_saved_variables();
        const Tensor dy = g[0].defined() ? g[0] : at::zeros(s[0].sizes(), s[0].options());
        const OptTensor dfinal = g.size() > 1 && g[1].defined() ? OptTensor(g[1].contiguous()) : OptTensor();
        const bool nb = ctx->saved_data["dbias"].toBool(), ni = ctx->saved_data["dinitial"].toBool();
        auto [dx, df, dg, db, di] = bwd.call(dy, s[0], s[1], opt(s[2]), opt(s[3]), s[4], opt(s[5]), dfinal, nb, ni);
        return {dx, df, s[2].defined() ? dg : Tensor(), nb ? db : Tensor(), ni ? di : Tensor(), Tensor(), Tensor()};
    }
};

struct PackedScanNode : torch::autograd::Function<PackedScanNode> {
    static Tensor forward(AutogradContext *ctx, const Tensor &features, const OptTensor &bias)
    {
        static const auto fwd = op<Two(const Tensor &, const OptTensor &, bool)>("gcg::scan_packed_fwd");
        at::AutoDispatchBelowADInplaceOrView below;
        auto [y, states] = fwd.call(features, bias, true);
        ctx->save_for_backward({features, or_empty(bias), states});
        ctx->saved_data["dbias"] = given(bias) && bias->requires_grad();
        return y;
    }
    static variable_list backward(AutogradContext *ctx, variable_list g)
    {
        const BelowAutograd below;
        static const auto bwd = op<Two(const Tensor &, const Tensor &, const OptTensor &, const Tensor &, bool)>("gcg::scan_packed_bwd");
        const variable_list s = ctx->get_saved_variables();
        const bool need = ctx->saved_data["dbias"].toBool();
        auto [df, db] = bwd.call(g[0], s[0], opt(s[1]), s[2], need);
        return {df, need ? db : Tensor()};
    }
};

std::vector<Tensor> rms_norm(const Tensor &x, const OptTensor &residual, const OptTensor &w, double eps)
{
    const Tensor a = or_empty(residual), b = or_empty(w);
    check_leaves({&x, &a, &b});
    return RmsNormNode::apply(x, residual, w, eps);
}
std::vector<Tensor> rms_norm_float8_stream(const Tensor &x, const Tensor &residual, const OptTensor &w, double eps)
{
    check_leaves({&x, &residual});
    return StreamNode::apply(x, residual, w, eps);
}
Tensor linear_float8(const Tensor &x, const Tensor &w, at::ScalarType format)
{
    check_weight(x, w);
    check_leaves({&x, &w});
    return LinearFloat8Node::apply(x, w, format);
}
std::vector<Tensor> norm_linear_float8(const Tensor &x, const OptTensor &residual, const OptTensor &gain, const Tensor &w, double eps,
                                       at::ScalarType format)
{
    const Tensor a = or_empty(residual), b = or_empty(gain);
    check_weight(x, w, a, b);
    check_leaves({&x, &a, &b, &w});
    return NormLinearFloat8Node::apply(x, residual, gain, w, eps, format);
}
std::vector<Tensor> scan(const Tensor &x, const Tensor &f, const OptTensor &gate, const OptTensor &bias, const OptTensor &initial,
                         const OptTensor &lengths, bool final)
{
    const Tensor a = or_empty(gate), b = or_empty(bias), c = or_empty(initial);
    check_leaves({&x, &f, &a, &b, &c});
    return ScanNode::apply(x, f, gate, bias, initial, lengths, final);
}
Tensor scan_packed(const Tensor &features, const OptTensor &bias)
{
    const Tensor b = or_empty(bias);
    check_leaves({&features, &b});
    return PackedScanNode::apply(features, bias);
}

} // namespace

TORCH_LIBRARY_FRAGMENT(gcg, m)
{
    m.def("rms_norm_fwd(Tensor x, Tensor? residual, Tensor? w, float eps) -> (Tensor, Tensor, Tensor)");
    m.def("rms_norm_infer(Tensor x, Tensor? residual, Tensor? w, float eps) -> (Tensor, Tensor)");
    m.def("rms_norm_float8(Tensor x, Tensor? residual, Tensor? w, float eps) -> (Tensor, Tensor, Tensor, Tensor)");
    m.def("rms_norm_bwd(Tensor dy, Tensor r, Tensor? dr, Tensor rstd, Tensor? w, bool need_dw=True) -> (Tensor, Tensor)");
    m.def("to_float8(Tensor x, ScalarType format) -> (Tensor, Tensor)");
    m.def("to_float8_both(Tensor x, ScalarType format) -> (Tensor, Tensor, Tensor, Tensor)");
    m.def("to_float8_columns(Tensor x, ScalarType format) -> (Tensor, Tensor)");
    m.def("float8_columns(Tensor codes, Tensor scales, int columns, ScalarType format) -> (Tensor, Tensor)");
    m.def("from_float8(Tensor codes, Tensor scales, int columns, ScalarType dtype) -> Tensor");
    m.def("matmul_float8(Tensor a, Tensor a_scales, Tensor b, Tensor b_scales, int columns, ScalarType dtype) -> Tensor");
    m.def("linear_float8_infer(Tensor x, Tensor codes, Tensor scales, int columns) -> Tensor");
    m.def("norm_linear_float8_infer(Tensor x, Tensor? residual, Tensor? gain, Tensor codes, Tensor scales, int columns, float eps)"
          " -> (Tensor, Tensor)");
    m.def("scan_fwd(Tensor x, Tensor f, Tensor? gate, Tensor? bias, Tensor? initial, Tensor? lengths, bool final, bool keep)"
          " -> (Tensor, Tensor, Tensor)");
    m.def("scan_bwd(Tensor dy, Tensor x, Tensor f, Tensor? gate, Tensor? bias, Tensor states, Tensor? lengths, Tensor? dfinal,"
          " bool need_dbias, bool need_dinitial) -> (Tensor, Tensor, Tensor, Tensor, Tensor)");
    m.def("scan_packed_fwd(Tensor features, Tensor? bias, bool keep) -> (Tensor, Tensor)");
    m.def("scan_packed_bwd(Tensor dy, Tensor features, Tensor? bias, Tensor states, bool need_dbias) -> (Tensor, Tensor)");
    m.def("scan_step(Tensor x, Tensor f, Tensor? gate, Tensor? bias, Tensor(a!) state) -> Tensor");
    m.def("rms_norm(Tensor x, Tensor? residual, Tensor? w, float eps) -> Tensor[]", &rms_norm);
    m.def("rms_norm_float8_stream(Tensor x, Tensor residual, Tensor? w, float eps) -> Tensor[]", &rms_norm_float8_stream);
    m.def("linear_float8(Tensor x, Tensor w, ScalarType format) -> Tensor", &linear_float8);
    m.def("norm_linear_float8(Tensor x, Tensor? residual, Tensor? gain, Tensor w, float eps, ScalarType format) -> Tensor[]", &norm_linear_float8);
    m.def("scan(Tensor x, Tensor f, Tensor? gate, Tensor? bias, Tensor? initial, Tensor? lengths, bool final) -> Tensor[]", &scan);
    m.def("scan_packed(Tensor features, Tensor? bias) -> Tensor", &scan_packed);
}

TORCH_LIBRARY_IMPL(gcg, CUDA, m)
{
    m.impl("rms_norm_fwd", &rms_norm_fwd);
    m.impl("rms_norm_infer", &rms_norm_infer);
    m.impl("rms_norm_float8", &rms_norm_float8);
    m.impl("rms_norm_bwd", &rms_norm_bwd);
    m.impl("to_float8", &to_float8);
    m.impl("to_float8_both", &to_float8_both);
    m.impl("to_float8_columns", &to_float8_columns);
    m.impl("float8_columns", &float8_columns);
    m.impl("from_float8", &from_float8);
    m.impl("matmul_float8", &matmul_float8);
    m.impl("linear_float8_infer", &linear_float8_infer);
    m.impl("norm_linear_float8_infer", &norm_linear_float8_infer);
    m.impl("scan_fwd", &scan_fwd);
    m.impl("scan_bwd", &scan_bwd);
    m.impl("scan_packed_fwd", &scan_packed_fwd);
    m.impl("scan_packed_bwd", &scan_packed_bwd);
    m.impl("scan_step", &scan_step);
}

TORCH_LIBRARY_IMPL(gcg, ADInplaceOrView, m)
{
    m.impl("scan_step", &scan_step_in_place);
}

TORCH_LIBRARY_IMPL(gcg, Meta, m)
{
    m.impl("rms_norm_fwd", &rms_norm_fwd_meta);
    m.impl("rms_norm_infer", &rms_norm_infer_meta);
    m.impl("rms_norm_float8", &rms_norm_float8_meta);
    m.impl("rms_norm_bwd", &rms_norm_bwd_meta);
    m.impl("to_float8", &to_float8_meta);
    m.impl("to_float8_both", &to_float8_both_meta);
    m.impl("to_float8_columns", &to_float8_columns_meta);
    m.impl("float8_columns", &float8_columns_meta);
    m.impl("from_float8", &from_float8_meta);
    m.impl("matmul_float8", &matmul_float8_meta);
    m.impl("linear_float8_infer", &linear_float8_infer_meta);
    m.impl("norm_linear_float8_infer", &norm_linear_float8_infer_meta);
    m.impl("scan_fwd", &scan_fwd_meta);
    m.impl("scan_bwd", &scan_bwd_meta);
    m.impl("scan_packed_fwd", &scan_packed_fwd_meta);
    m.impl("scan_packed_bwd", &scan_packed_bwd_meta);
    m.impl("scan_step", &scan_step_meta);
}
