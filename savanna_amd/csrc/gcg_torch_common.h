// What the translation units of the PyTorch extension share: codes, streams, guards, errors, workspaces.
#pragma once
#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/library.h>
#include <torch/types.h>

#include "../../include/gcg.h"

namespace {

using at::Tensor;
using DeviceGuard = at::hip::OptionalHIPGuardMasqueradingAsCUDA;

inline int dtype_code(at::ScalarType t)
{
    switch (t) {
    case at::kFloat: return GCG_F32;
    case at::kBFloat16: return GCG_BF16;
    case at::kHalf: return GCG_F16;
    default: TORCH_CHECK(false, "gcg: unsupported dtype ", t, "; expected float32, bfloat16 or float16");
    }
}

inline void *stream_of(const Tensor &t)
{
    return (void *)at::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.device().index()).stream();
}

inline void check_rc(int rc, const char *what)
{
    TORCH_CHECK(rc == 0, what, ": ", gcg_strerror(rc), " (code ", rc, ", hipError ", gcg_last_hip_error(), ")");
}

inline void require_gpu(const Tensor &t, const char *name)
{
    TORCH_CHECK(t.is_cuda(), "gcg: ", name, " is on ", t.device(),
                "; the kernels run on an MI355X (gfx950) device only and there is no CPU path");
}

inline Tensor workspace(size_t bytes, const Tensor &like, const char *what)
{
    TORCH_CHECK(bytes > 0, what, ": arguments rejected (shape not supported by the requested kernel family)");
    return at::empty({(int64_t)bytes}, like.options().dtype(at::kByte));
}

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

template <typename F> c10::TypedOperatorHandle<F> op(const char *name)
{
    return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<F>();
}

} // namespace
