// The products by runs of rows as PyTorch operators, in C++: an ordinary call goes from the dispatcher to the launcher
// without touching Python (8 us for a grouped product where marshalling in Python took 21, as long as two small launches).
//
// Everything that is not ordinary (arguments that do not fit, tensors of another device than the current one, a launcher's
// refusal) is handed to the Python function of the same name in ninetoothed_b200._capi, which raises what it always raises.
#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/utils/pybind.h>
#include <torch/library.h>

#include <atomic>

#include "ninetoothed_b200.h"

namespace {

// A tensor as the launchers take it.  (Strides and sizes are the tensor's own arrays, read during the call only.)
NineToothedTensor argument(const at::Tensor &t) {
    static_assert(sizeof(int64_t) == sizeof(uint64_t), "sizes are passed as they are");
    return {t.data_ptr(), reinterpret_cast<uint64_t *>(const_cast<int64_t *>(t.sizes().data())), const_cast<int64_t *>(t.strides().data())};
}

int type_tag(const at::Tensor &t) {
    switch (t.scalar_type()) {
        case at::kHalf:
            return NINETOOTHED_FLOAT16;
        case at::kBFloat16:
            return NINETOOTHED_BFLOAT16;
        case at::kInt:
            return NINETOOTHED_INT32;
        case at::kLong:
            return NINETOOTHED_INT64;
        default:
            return -1;
    }
}

bool is_index(const at::Tensor &t, c10::Device device) {
    return t.dim() == 1 && t.device() == device && (t.scalar_type() == at::kInt || t.scalar_type() == at::kLong);
}

bool is_operand(const at::Tensor &t, const at::Tensor &first, int64_t dim) {
    return t.dim() == dim && t.device() == first.device() && t.scalar_type() == first.scalar_type();
}

// lhs decides: on the current device, of a 16-bit type.
bool ordinary(const at::Tensor &lhs) {
    return lhs.is_cuda() && lhs.dim() == 2 && lhs.device().index() == c10::cuda::current_device() &&
           (lhs.scalar_type() == at::kHalf || lhs.scalar_type() == at::kBFloat16);
}

template <typename... Args>
void in_python(const char *name, const Args &...args) {
    py::gil_scoped_acquire gil;
    py::module_::import("ninetoothed_b200._capi").attr(name)(args...);
}

// A launch on one of the plain kernels warns, as it does from Python.
void warn_of_plain_launches() {
    static std::atomic<long long> seen{0};
    const long long count = ninetoothed_b200_plain_launches(0);
    if (seen.exchange(count) != count) in_python("warn_of_plain_launches");
}

void grouped_matmul(const at::Tensor &lhs, const at::Tensor &rhs, const at::Tensor &offsets, at::Tensor output) {
    if (ordinary(lhs) && is_operand(rhs, lhs, 3) && is_operand(output, lhs, 2) && is_index(offsets, lhs.device()) &&
        launch_grouped_matmul(c10::cuda::getCurrentCUDAStream(lhs.device().index()).stream(), argument(lhs), argument(rhs),
                              argument(offsets), argument(output), type_tag(lhs), type_tag(offsets)) == 0)
        return warn_of_plain_launches();
    in_python("grouped_matmul", lhs, rhs, offsets, output);
}

void grouped_matmul_rhs_grad(const at::Tensor &lhs, const at::Tensor &output_grad, const at::Tensor &offsets, at::Tensor rhs_grad) {
    if (ordinary(lhs) && is_operand(output_grad, lhs, 2) && is_operand(rhs_grad, lhs, 3) && is_index(offsets, lhs.device()) &&
        launch_grouped_matmul_rhs_grad(c10::cuda::getCurrentCUDAStream(lhs.device().index()).stream(), argument(lhs),
                                       argument(output_grad), argument(offsets), argument(rhs_grad), type_tag(lhs),
                                       type_tag(offsets)) == 0)
        return warn_of_plain_launches();
    in_python("grouped_matmul_rhs_grad", lhs, output_grad, offsets, rhs_grad);
}

void lora_matmul(const at::Tensor &lhs, const at::Tensor &rhs, const at::Tensor &down, const at::Tensor &up, const at::Tensor &scales,
                 const at::Tensor &offsets, const at::Tensor &adapters, at::Tensor output) {
    if (ordinary(lhs) && is_operand(rhs, lhs, 2) && is_operand(down, lhs, 3) && is_operand(up, lhs, 3) && is_operand(output, lhs, 2) &&
        is_index(offsets, lhs.device()) && is_index(adapters, lhs.device()) && scales.dim() == 1 && scales.device() == lhs.device() &&
        scales.scalar_type() == at::kFloat) {
        const size_t size = launch_lora_matmul_workspace_size(argument(lhs), argument(down));
        const at::Tensor workspace = at::empty({static_cast<int64_t>(size)}, lhs.options().dtype(at::kByte));
        if (launch_lora_matmul(c10::cuda::getCurrentCUDAStream(lhs.device().index()).stream(), argument(lhs), argument(rhs),
                               argument(down), argument(up), argument(scales), argument(offsets), argument(adapters),
                               argument(output), type_tag(lhs), type_tag(offsets), type_tag(adapters), workspace.data_ptr(),
                               size) == 0)
            return warn_of_plain_launches();
    }
    in_python("lora_matmul", lhs, rhs, down, up, scales, offsets, adapters, output);
}

}  // namespace

TORCH_LIBRARY_IMPL(ninetoothed_b200, CUDA, library) {
    library.impl("grouped_matmul", &grouped_matmul);
    library.impl("grouped_matmul_rhs_grad", &grouped_matmul_rhs_grad);
    library.impl("lora_matmul", &lora_matmul);
}
