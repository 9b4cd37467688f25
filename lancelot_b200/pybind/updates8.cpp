// The 8-bit update calls of cabi.Context on torch tensors: argument checks, results and workspaces, then one lb_* call each.  These
// kernels run in a few microseconds where operands are small; the same checks in Python took longer than the kernels.
// Built by lancelot_b200/pybind/build.py; links liblancelot_b200.so and torch's C++ libraries and launches nothing itself.
#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <c10/cuda/CUDAStream.h>
#include <pybind11/pybind11.h>
#include <torch/csrc/utils/pybind.h>

#include <optional>
#include <string>

#include "lancelot_b200.h"

namespace py = pybind11;
using at::Tensor;
using Maybe = std::optional<Tensor>;

namespace {

struct Refused {
    int code;
    std::string message;
};
[[noreturn]] void refuse(const std::string &message) { throw Refused{LB_ERR_INVALID_ARG, message}; }
void check(int code)
{
    if (code != LB_OK) throw Refused{code, lb_last_error()};
}

int value_type(at::ScalarType t) // as the C ABI numbers them; 0: none
{
    return t == at::kFloat ? 1 : t == at::kBFloat16 ? 3 : t == at::kHalf ? 4 : 0;
}
at::ScalarType scalar_type(int value_type)
{
    if (value_type != 1 && value_type != 3 && value_type != 4) refuse("dtype must be float32, bfloat16 or float16");
    return value_type == 1 ? at::kFloat : value_type == 3 ? at::kBFloat16 : at::kHalf;
}

struct Call {
    lb_context *context;
    int device;

    void tensor(const Tensor &t, int dims, const char *what) const
    {
        if (!t.is_cuda() || t.get_device() != device) refuse(std::string(what) + " must be a tensor on cuda:" + std::to_string(device));
        if (t.dim() != dims) refuse(std::string(what) + " must have " + std::to_string(dims) + " dimension(s)");
        if (t.size(dims - 1) > 1 && t.stride(dims - 1) != 1) refuse(std::string(what) + " must be dense along its rows");
    }
    void tensor(const Tensor &t, int dims, at::ScalarType type, const char *what) const
    {
        tensor(t, dims, what);
        if (t.scalar_type() != type) refuse(std::string(what) + " must be of type " + c10::toString(type));
    }
    void *stream() const { return c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)device).stream(); }
    Tensor empty(at::IntArrayRef size, at::ScalarType type) const
    {
        return at::empty(size, at::TensorOptions().dtype(type).device(at::kCUDA, (c10::DeviceIndex)device));
    }
    // scratch of this call: its own, so that calls on two streams, or captured into two graphs, share none
    Tensor workspace(size_t bytes) const { return bytes ? empty({(int64_t)bytes}, at::kByte) : Tensor(); }
};

// elements from one row to the next; a single row has no next one, and counts as dense wherever it was taken from
int64_t row_stride(const Tensor &t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }
template <typename T> T *address(const Tensor &t) { return t.defined() && t.numel() ? static_cast<T *>(t.data_ptr()) : nullptr; }
template <typename T> T *address(const Maybe &t) { return t ? address<T>(*t) : nullptr; }

struct Cache {
    int8_t *codes;
    float *scales;
    int64_t slots, page, code_stride, scale_stride;
};
Cache cache_of(const Call &c, const Tensor &codes, const Tensor &scales, int64_t group)
{
    c.tensor(codes, 2, at::kChar, "codes");
    c.tensor(scales, 2, at::kFloat, "scales");
    Cache k{address<int8_t>(codes), address<float>(scales), codes.size(0), codes.size(1), row_stride(codes), row_stride(scales)};
    const int64_t groups = group > 0 && group < k.page ? (k.page + group - 1) / group : 1;
    if (scales.size(0) < k.slots || scales.size(1) < groups)
        refuse("scales must hold " + std::to_string(groups) + " scale(s) for each of the " + std::to_string(k.slots) + " slots");
    return k;
}
int64_t pages_of(int64_t n_cols, int64_t page) { return page > 0 ? (n_cols + page - 1) / page : 0; }
const int32_t *slots_of(const Call &c, const Maybe &slots, int64_t n_rows, int64_t pages)
{
    if (!slots) return nullptr;
    const Tensor &t = *slots;
    if (!t.is_cuda() || t.get_device() != c.device || t.scalar_type() != at::kInt || !t.is_contiguous())
        refuse("slots must be a contiguous int32 tensor on cuda:" + std::to_string(c.device));
    if (t.numel() != n_rows * pages) refuse("slots must name " + std::to_string(pages) + " page(s) for each of the " + std::to_string(n_rows) + " row(s)");
    return address<int32_t>(t);
}
Tensor result(const Call &c, const Maybe &out, int64_t rows, int64_t cols, int dtype)
{
    if (!out) return c.empty({rows, cols}, scalar_type(dtype));
    c.tensor(*out, 2, "out");
    if (!value_type(out->scalar_type())) refuse("out must be float32, bfloat16 or float16");
    if (out->size(0) != rows || out->size(1) != cols) refuse("out must be [" + std::to_string(rows) + "][" + std::to_string(cols) + "]");
    return *out;
}
Call call_of(int64_t context, int device) { return Call{reinterpret_cast<lb_context *>(context), device}; }

void quantize_rows(int64_t context, int device, const Tensor &values, const Tensor &codes, const Tensor &scales, int64_t group, const Maybe &slots,
                   const Maybe &lengths, const Maybe &residual, const Maybe &residual_out)
{
    const Call c = call_of(context, device);
    c.tensor(values, 2, "values");
    const int type = value_type(values.scalar_type());
    if (!type) refuse("values must be float32, bfloat16 or float16");
    const int64_t n = values.size(0), cols = values.size(1);
    const Cache k = cache_of(c, codes, scales, group);
    const int32_t *table = slots_of(c, slots, n, pages_of(cols, k.page));
    if (lengths) {
        c.tensor(*lengths, 1, at::kInt, "lengths");
        if (lengths->numel() != n) refuse("lengths must have one entry for each row");
    }
    int64_t stride = 0;
    for (const Maybe *r : {&residual, &residual_out}) {
        if (!*r) continue;
        c.tensor(**r, 2, at::kFloat, "a residual");
        if ((*r)->size(0) != n || (*r)->size(1) != cols) refuse("a residual must have the shape of values");
        if (stride && stride != row_stride(**r)) refuse("residual and residual_out must have the same row stride");
        stride = row_stride(**r);
    }
    const size_t need = lb_quantize_rows_workspace_bytes(n, cols, k.page, group);
    const Tensor ws = c.workspace(need);
    check(lb_quantize_rows(c.context, address<void>(values), type, n, cols, row_stride(values), address<int32_t>(lengths), address<float>(residual),
                           address<float>(residual_out), stride, table, k.slots, k.page, group, k.codes, k.code_stride, k.scales, k.scale_stride,
                           address<void>(ws), need, c.stream()));
}

Tensor dequantize_rows(int64_t context, int device, const Tensor &codes, const Tensor &scales, int64_t n_cols, int64_t group, const Maybe &slots,
                       std::optional<int64_t> n_rows, int dtype, const Maybe &out)
{
    const Call c = call_of(context, device);
    const Cache k = cache_of(c, codes, scales, group);
    if (n_cols < 0) refuse("n_cols is out of range");
    const int64_t pages = pages_of(n_cols, k.page);
    const int64_t n = n_rows ? *n_rows : out ? (out->dim() == 2 ? out->size(0) : 0) : (slots ? slots->numel() : k.slots) / std::max<int64_t>(pages, 1);
    if (n < 0) refuse("n_rows is out of range");
    const int32_t *table = slots_of(c, slots, n, pages);
    const Tensor to = result(c, out, n, n_cols, dtype);
    check(lb_dequantize_rows(c.context, k.codes, k.code_stride, k.scales, k.scale_stride, k.slots, k.page, group, table, n, n_cols, address<void>(to),
                             value_type(to.scalar_type()), row_stride(to), c.stream()));
    return to;
}

Tensor int8_matmul(int64_t context, int device, const Tensor &a, const Tensor &b, const Tensor &a_scale, const Tensor &b_scale, int dtype, const Maybe &out)
{
    const Call c = call_of(context, device);
    c.tensor(a, 2, at::kChar, "a");
    c.tensor(b, 2, at::kChar, "b");
    const int64_t m = a.size(0), n = b.size(0), k = a.size(1);
    if (b.size(1) != k) refuse("a and b must have rows of the same length");
    c.tensor(a_scale, 1, at::kFloat, "a_scale");
    c.tensor(b_scale, 1, at::kFloat, "b_scale");
    if (a_scale.numel() != m || b_scale.numel() != n) refuse("a scale must have one entry for each row of its operand");
    const Tensor to = result(c, out, m, n, dtype);
    const int8_t *pa = address<int8_t>(a), *pb = address<int8_t>(b);
    const int64_t sa = row_stride(a), sb = row_stride(b);
    const size_t need = lb_int8_matmul_workspace_bytes(m, n, k, pa, sa, pb, sb);
    const Tensor ws = c.workspace(need);
    check(lb_int8_matmul(c.context, m, n, k, pa, sa, address<float>(a_scale), pb, sb, address<float>(b_scale), address<void>(to),
                         value_type(to.scalar_type()), row_stride(to), address<void>(ws), need, c.stream()));
    return to;
}

Tensor int8_distances(int64_t context, int device, const Tensor &codes, const Tensor &scales, const Tensor &slots, int64_t group)
{
    const Call c = call_of(context, device);
    const Cache k = cache_of(c, codes, scales, group);
    c.tensor(slots, 2, at::kInt, "slots");
    if (!slots.is_contiguous()) refuse("slots must be contiguous");
    const int64_t n = slots.size(0), pages = slots.size(1);
    const Tensor out = c.empty({n, n}, at::kDouble);
    const size_t need = lb_int8_distances_workspace_bytes(c.context, n, pages, k.page);
    const Tensor ws = c.workspace(need);
    check(lb_int8_distances(c.context, k.codes, k.code_stride, k.scales, k.scale_stride, k.slots, k.page, group, address<int32_t>(slots), n, pages,
                            address<double>(out), address<void>(ws), need, c.stream()));
    return out;
}

} // namespace

PYBIND11_MODULE(_updates8, m)
{
    // the exceptions of the Python layer (lancelot_b200/_lib.py)
    py::register_exception_translator([](std::exception_ptr p) {
        try {
            if (p) std::rethrow_exception(p);
        } catch (const Refused &e) {
            const py::object type = py::module_::import("lancelot_b200._lib").attr(e.code == LB_ERR_INVALID_ARG ? "InvalidArgument" : "LancelotError");
            const py::object exception = type(e.code, e.message);
            PyErr_SetObject(type.ptr(), exception.ptr());
        }
    });
    m.def("quantize_rows", &quantize_rows);
    m.def("dequantize_rows", &dequantize_rows);
    m.def("int8_matmul", &int8_matmul);
    m.def("int8_distances", &int8_distances);
}
