// The 8-bit update calls of cabi.Context (integers, floating point) and its clipping on torch tensors: argument checks, results and workspaces, then one lb_* call each.  These
// kernels run in a few microseconds where operands are small; the same checks in Python took longer than the kernels.
// Built by lancelot_b200/pybind/build.py; links liblancelot_b200.so and torch's C++ libraries and launches nothing itself.
#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <ATen/ops/empty_strided.h>
#include <c10/cuda/CUDAStream.h>
#include <pybind11/pybind11.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/pybind.h>

#include <cmath>
#include <optional>
#include <string>
#include <vector>

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
// a caller's tensor that a call has written: autograd sees from its version that it is no longer what was saved
void written(const Tensor &t)
{
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}
void written(const Maybe &t)
{
    if (t) written(*t);
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
    written(codes);
    written(scales);
    written(residual_out);
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
    written(out);
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
    written(out);
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

// ---- 8-bit floating point -------------------------------------------------------------------------------------------------------
int code_type(const Tensor &t, const char *what) // as the C ABI numbers them
{
    if (t.scalar_type() == at::kFloat8_e4m3fn) return 5;
    if (t.scalar_type() == at::kFloat8_e5m2) return 6;
    refuse(std::string(what) + " must be of type float8_e4m3fn or float8_e5m2");
}
int64_t blocks_of(int64_t n) { return (n + 127) / 128; }

// codes and scales of one kind of blocks: given ones are checked, missing ones made, with rows of codes on 16-byte boundaries
void blocks_into(const Call &c, Maybe &codes, Maybe &scales, int64_t rows, int64_t cols, int64_t scale_rows, int64_t scale_cols, int type)
{
    const at::ScalarType t = type == 5 ? at::kFloat8_e4m3fn : at::kFloat8_e5m2;
    if (!codes) codes = at::empty_strided({rows, cols}, {std::max<int64_t>((cols + 15) / 16 * 16, 16), 1}, at::TensorOptions().dtype(t).device(at::kCUDA, (c10::DeviceIndex)c.device));
    if (!scales) scales = c.empty({scale_rows, scale_cols}, at::kFloat);
    c.tensor(*codes, 2, t, "codes");
    c.tensor(*scales, 2, at::kFloat, "scales");
    if (codes->size(0) != rows || codes->size(1) != cols) refuse("codes must have the shape of values");
    if (scales->size(0) != scale_rows || scales->size(1) != scale_cols)
        refuse("scales must be [" + std::to_string(scale_rows) + "][" + std::to_string(scale_cols) + "]");
}

py::tuple quantize_fp8(int64_t context, int device, const Tensor &values, int blocks, int type, Maybe codes, Maybe scales, Maybe codes_down, Maybe scales_down)
{
    const Call c = call_of(context, device);
    c.tensor(values, 2, "values");
    const int dtype = value_type(values.scalar_type());
    if (!dtype) refuse("values must be float32, bfloat16 or float16");
    if (blocks < 1 || blocks > 4) refuse("block must be (1, 128), (128, 1) or (128, 128)");
    if (type != 5 && type != 6) refuse("dtype must be float8_e4m3fn or float8_e5m2");
    const int64_t n = values.size(0), cols = values.size(1);
    const Maybe given[] = {codes, scales, codes_down, scales_down};
    if (blocks != 2) blocks_into(c, codes, scales, n, cols, blocks == 4 ? blocks_of(n) : n, blocks_of(cols), type);
    if (blocks == 2 || blocks == 3) blocks_into(c, codes_down, scales_down, n, cols, blocks_of(n), cols, type);
    auto stride = [](const Maybe &t) { return t ? row_stride(*t) : 0; };
    check(lb_quantize_fp8(c.context, address<void>(values), dtype, n, cols, row_stride(values), blocks, type, address<uint8_t>(codes), stride(codes),
                          address<float>(scales), stride(scales), address<uint8_t>(codes_down), stride(codes_down), address<float>(scales_down),
                          stride(scales_down), c.stream()));
    for (const Maybe &t : given) written(t);
    if (blocks == 3) return py::make_tuple(*codes, *scales, *codes_down, *scales_down);
    return blocks == 2 ? py::make_tuple(*codes_down, *scales_down) : py::make_tuple(*codes, *scales);
}

Tensor dequantize_fp8(int64_t context, int device, const Tensor &codes, const Tensor &scales, int dtype, const Maybe &out)
{
    const Call c = call_of(context, device);
    c.tensor(codes, 2, "codes");
    const int type = code_type(codes, "codes");
    c.tensor(scales, 2, at::kFloat, "scales");
    const int64_t n = codes.size(0), cols = codes.size(1), r = scales.size(0), q = scales.size(1);
    // where two kinds of blocks have scales of the same shape they are the same blocks
    const int blocks = r == n && q == blocks_of(cols) ? 1 : r == blocks_of(n) && q == cols ? 2 : r == blocks_of(n) && q == blocks_of(cols) ? 4 : 0;
    if (!blocks) refuse("scales must have one entry for each block of 128 columns, 128 rows or 128 x 128");
    const Tensor to = result(c, out, n, cols, dtype);
    check(lb_dequantize_fp8(c.context, address<uint8_t>(codes), type, row_stride(codes), address<float>(scales), row_stride(scales), blocks, n, cols,
                            address<void>(to), value_type(to.scalar_type()), row_stride(to), c.stream()));
    written(out);
    return to;
}

// [rows][k] with its scales; dense along either axis
lb_fp8_operand operand(const Call &c, const Tensor &t, const Tensor &scales, const char *what)
{
    if (!t.is_cuda() || t.get_device() != c.device) refuse(std::string(what) + " must be a tensor on cuda:" + std::to_string(c.device));
    if (t.dim() != 2) refuse(std::string(what) + " must have 2 dimension(s)");
    lb_fp8_operand o = {};
    o.code_type = code_type(t, what);
    const int64_t rows = t.size(0), k = t.size(1);
    const bool along = k <= 1 || t.stride(1) == 1, across = rows <= 1 || t.stride(0) == 1;
    if (!along && !across) refuse(std::string(what) + " must be dense along one of its axes");
    // a single column that is dense as a row: the row
    o.across = !along || (across && k == 1 && rows > 1);
    o.codes = address<uint8_t>(t);
    o.stride = o.across ? (k > 1 ? t.stride(1) : rows) : (rows > 1 ? t.stride(0) : k);
    if (!scales.is_cuda() || scales.get_device() != c.device || scales.scalar_type() != at::kFloat || scales.dim() != 2)
        refuse(std::string("the scales of ") + what + " must be a float32 tensor of 2 dimensions on cuda:" + std::to_string(c.device));
    if (scales.size(1) != blocks_of(k) || (scales.size(0) != rows && scales.size(0) != blocks_of(rows)))
        refuse(std::string("the scales of ") + what + " must be [" + std::to_string(rows) + "][" + std::to_string(blocks_of(k)) + "] or [" +
               std::to_string(blocks_of(rows)) + "][" + std::to_string(blocks_of(k)) + "]");
    o.scales = address<float>(scales);
    o.scale_row = scales.stride(0);
    o.scale_block = scales.stride(1);
    o.scale_rows = scales.size(0) == rows ? 1 : 128;
    return o;
}

Tensor fp8_matmul(int64_t context, int device, const Tensor &a, const Tensor &a_scale, const Tensor &b, const Tensor &b_scale, int dtype, const Maybe &out)
{
    const Call c = call_of(context, device);
    const lb_fp8_operand x = operand(c, a, a_scale, "a"), y = operand(c, b, b_scale, "b");
    const int64_t m = a.size(0), n = b.size(0), k = a.size(1);
    if (b.size(1) != k) refuse("a and b must have rows of the same length");
    const Tensor to = result(c, out, m, n, dtype);
    const size_t need = lb_fp8_matmul_workspace_bytes(m, n, k, &x, &y);
    const Tensor ws = c.workspace(need);
    check(lb_fp8_matmul(c.context, m, n, k, &x, &y, address<void>(to), value_type(to.scalar_type()), row_stride(to), address<void>(ws), need, c.stream()));
    written(out);
    return to;
}

// ---- a layer's training step: y = x w^T and the gradients of x and w, a call each ---------------------------------------------------
// t [..., k] as a matrix whose rows are dense and apart: not so are transposed ones, and the gradient of a sum, one value for all
Tensor matrix(const Tensor &t)
{
    const int64_t k = t.size(-1), rows = k ? t.numel() / k : t.sizes().size() < 2 ? 1 : c10::multiply_integers(t.sizes().slice(0, t.dim() - 1));
    const Tensor m = t.dim() == 2 ? t : t.reshape({rows, k});
    return m.stride(1) == 1 && (rows < 2 || m.stride(0) >= k) ? m : m.contiguous();
}
struct Coded {
    Tensor codes, scales, down, down_scales;
};
Coded coded(const Call &c, const Tensor &m, int blocks, int type)
{
    Maybe codes, scales, down, down_scales;
    const int64_t n = m.size(0), cols = m.size(1);
    c.tensor(m, 2, "an operand");
    const int dtype = value_type(m.scalar_type());
    if (!dtype) refuse("an operand must be float32, bfloat16 or float16");
    if (blocks != 2) blocks_into(c, codes, scales, n, cols, blocks == 4 ? blocks_of(n) : n, blocks_of(cols), type);
    if (blocks == 2 || blocks == 3) blocks_into(c, down, down_scales, n, cols, blocks_of(n), cols, type);
    auto stride = [](const Maybe &t) { return t ? row_stride(*t) : 0; };
    check(lb_quantize_fp8(c.context, address<void>(m), dtype, n, cols, row_stride(m), blocks, type, address<uint8_t>(codes), stride(codes),
                          address<float>(scales), stride(scales), address<uint8_t>(down), stride(down), address<float>(down_scales),
                          stride(down_scales), c.stream()));
    return {codes.value_or(Tensor()), scales.value_or(Tensor()), down.value_or(Tensor()), down_scales.value_or(Tensor())};
}
// codes and their scales as they lie, or both with their axes exchanged
lb_fp8_operand stored_operand(const Tensor &codes, const Tensor &scales, bool across, int scale_rows, int type)
{
    lb_fp8_operand o = {};
    o.codes = address<uint8_t>(codes);
    o.stride = row_stride(codes);
    o.across = across;
    o.code_type = type;
    o.scales = address<float>(scales);
    o.scale_row = across ? 1 : row_stride(scales);
    o.scale_block = across ? row_stride(scales) : 1;
    o.scale_rows = scale_rows;
    return o;
}
Tensor product(const Call &c, int64_t m, int64_t n, int64_t k, const lb_fp8_operand &x, const lb_fp8_operand &y, at::IntArrayRef shape, at::ScalarType type)
{
    const Tensor to = c.empty(shape, type);
    const size_t need = lb_fp8_matmul_workspace_bytes(m, n, k, &x, &y);
    const Tensor ws = c.workspace(need);
    check(lb_fp8_matmul(c.context, m, n, k, &x, &y, address<void>(to), value_type(type), n, address<void>(ws), need, c.stream()));
    return to;
}

// The context's owner, a Python object: asked for the handle again in the backward pass, so that a context closed in between is refused
struct Owner : torch::CustomClassHolder {
    PyObject *object;
    explicit Owner(const py::handle &o) : object(o.inc_ref().ptr()) {}
    ~Owner() override
    {
        if (!Py_IsInitialized()) return;
        py::gil_scoped_acquire gil;
        Py_DECREF(object);
    }
    int64_t handle() const
    {
        py::gil_scoped_acquire gil;
        return py::handle(object).attr("_handle")().cast<int64_t>();
    }
};

struct Fp8Linear : torch::autograd::Function<Fp8Linear> {
    static Tensor forward(torch::autograd::AutogradContext *ctx, const Tensor &x, const Tensor &w, const Call &c, const c10::intrusive_ptr<Owner> &owner, int type,
                          bool need_x, bool need_w)
    {
        const Tensor xm = matrix(x), wm = matrix(w);
        const Coded xc = coded(c, xm, need_w ? 3 : 1, 5), wc = coded(c, wm, 4, 5);
        const int64_t m = xm.size(0), n = wm.size(0), k = xm.size(1);
        at::DimVector shape(x.sizes().begin(), x.sizes().end());
        shape.back() = n;
        // x in blocks along its rows' axis is for the gradient of w, w's codes are for that of x
        ctx->save_for_backward({need_w ? xc.down : Tensor(), need_w ? xc.down_scales : Tensor(), need_x ? wc.codes : Tensor(), need_x ? wc.scales : Tensor()});
        ctx->saved_data["owner"] = c10::IValue::make_capsule(owner);
        ctx->saved_data["device"] = (int64_t)c.device;
        ctx->saved_data["type"] = (int64_t)type;
        ctx->saved_data["x"] = x.scalar_type();
        ctx->saved_data["w"] = w.scalar_type();
        return product(c, m, n, k, stored_operand(xc.codes, xc.scales, false, 1, 5), stored_operand(wc.codes, wc.scales, false, 128, 5), shape, x.scalar_type());
    }

    static torch::autograd::variable_list backward(torch::autograd::AutogradContext *ctx, const torch::autograd::variable_list &grads)
    {
        torch::autograd::variable_list out(7);
        const Tensor &g = grads[0];
        const auto kept = ctx->get_saved_variables();
        const Tensor &xd = kept[0], &xds = kept[1], &w8 = kept[2], &ws = kept[3];
        if (!g.defined() || (!xd.defined() && !w8.defined())) return out;
        const bool again = at::GradMode::is_enabled();
        try {
            at::NoGradGuard none;
            const Call c = call_of(c10::static_intrusive_pointer_cast<Owner>(ctx->saved_data["owner"].toCapsule())->handle(), (int)ctx->saved_data["device"].toInt());
            const int type = (int)ctx->saved_data["type"].toInt();
            const Tensor gm = matrix(g);
            const Coded gc = coded(c, gm, w8.defined() ? (xd.defined() ? 3 : 1) : 2, type);
            const int64_t m = gm.size(0), n = gm.size(1);
            if (w8.defined()) {
                at::DimVector shape(g.sizes().begin(), g.sizes().end());
                shape.back() = w8.size(1);
                out[0] = product(c, m, w8.size(1), n, stored_operand(gc.codes, gc.scales, false, 1, type), stored_operand(w8, ws, true, 128, 5), shape,
                                 ctx->saved_data["x"].toScalarType());
            }
            if (xd.defined())
                out[1] = product(c, n, xd.size(1), m, stored_operand(gc.down, gc.down_scales, true, 1, type), stored_operand(xd, xds, true, 1, 5), {n, xd.size(1)},
                                 ctx->saved_data["w"].toScalarType());
        } catch (const Refused &e) { // this may be a thread of the autograd engine, which carries torch's exceptions to the caller
            TORCH_CHECK_VALUE(e.code != LB_ERR_INVALID_ARG, e.message);
            TORCH_CHECK(false, e.message);
        }
        if (again) { // gradients of the gradients are not there: whoever asks for them is told
            torch::autograd::variable_list found;
            for (Tensor &t : out)
                if (t.defined()) found.push_back(t.detach().set_requires_grad(true));
            const auto error = std::make_shared<torch::autograd::DelayedError>("the gradients of fp8_linear are not differentiable", (int64_t)found.size());
            found = (*error)(std::move(found));
            size_t i = 0;
            for (Tensor &t : out)
                if (t.defined()) t = found[i++];
        }
        return out;
    }
};

Tensor fp8_linear(const py::object &lb, int device, const Tensor &x, const Tensor &w, int type)
{
    const Call c = call_of(lb.attr("_handle")().cast<int64_t>(), device);
    if (x.dim() < 1 || w.dim() != 2 || x.size(-1) != w.size(1)) refuse("x must be [..., k] and w [n][k]");
    if (type != 5 && type != 6) refuse("grad_dtype must be float8_e4m3fn or float8_e5m2");
    const bool grad = at::GradMode::is_enabled();
    return Fp8Linear::apply(x, w, c, c10::make_intrusive<Owner>(lb), type, grad && x.requires_grad(), grad && w.requires_grad());
}

// ---- clipping -------------------------------------------------------------------------------------------------------------------
Tensor clip_updates(int64_t context, int device, const py::object &updates, std::optional<double> max_norm, const Maybe &out)
{
    const Call c = call_of(context, device);
    std::vector<int> clients, dtypes, out_dtypes;
    std::vector<const void *> tensors;
    std::vector<void *> outs;
    std::vector<int64_t> sizes;
    std::vector<Tensor> held;
    const bool in_place = max_norm && !out;
    int n = 0;
    auto add = [&](const Tensor &t, int64_t size, int64_t offset) {
        clients.push_back(n);
        dtypes.push_back(value_type(t.scalar_type()));
        tensors.push_back(size ? static_cast<char *>(t.data_ptr()) + offset * t.element_size() : nullptr);
        sizes.push_back(size);
    };
    if (THPVariable_Check(updates.ptr())) { // [clients][values]
        const Tensor t = THPVariable_Unpack(updates.ptr());
        c.tensor(t, 2, "updates");
        if (!value_type(t.scalar_type())) refuse("updates must be float32, bfloat16 or float16");
        if (t.size(0) > 1 && t.stride(0) < t.size(1)) refuse("the rows of updates overlap");
        for (; n < t.size(0); ++n) add(t, t.size(1), n * t.stride(0));
        held.push_back(t);
    } else {
        if (!py::isinstance<py::sequence>(updates)) refuse("updates must be a matrix, or for each client a list of tensors");
        auto add_tensor = [&](const Tensor &t) {
            if (!t.is_cuda() || t.get_device() != c.device || t.layout() != at::kStrided) refuse("an update's tensors must be on cuda:" + std::to_string(device));
            if (!value_type(t.scalar_type())) refuse("an update's tensors must be float32, bfloat16 or float16");
            // the order of the values is the result's where they are copied
            if (out ? !t.is_contiguous() : !t.is_non_overlapping_and_dense()) refuse(out ? "an update's tensors must be contiguous" : "an update's tensors must be dense");
            add(t, t.numel(), 0);
        };
        auto each = [&](const py::handle &client, auto &&use) {
            if (THPVariable_Check(client.ptr()) || !py::isinstance<py::sequence>(client)) refuse("updates must be a matrix, or for each client a list of tensors");
            const py::object items = py::reinterpret_steal<py::object>(PySequence_Fast(client.ptr(), "updates"));
            if (!items) throw py::error_already_set();
            for (Py_ssize_t i = 0; i < PySequence_Fast_GET_SIZE(items.ptr()); ++i) {
                const py::handle item = PySequence_Fast_GET_ITEM(items.ptr(), i);
                if (!THPVariable_Check(item.ptr())) refuse("updates must be a matrix, or for each client a list of tensors");
                use(THPVariable_Unpack(item.ptr()));
            }
        };
        // Lists and tuples keep their tensors, and nothing runs in this thread's place, or in another's, that could take them away before the launch.  Any other
        // sequence may make its items when they are asked for, and change lists meanwhile: then all tensors are held, before the first address is taken
        auto keeps = [](PyObject *of) { return PyList_CheckExact(of) || PyTuple_CheckExact(of); };
        bool lasting = keeps(updates.ptr());
        for (Py_ssize_t k = 0; lasting && k < PySequence_Fast_GET_SIZE(updates.ptr()); ++k) lasting = keeps(PySequence_Fast_GET_ITEM(updates.ptr(), k));
        if (lasting) {
            for (; n < PySequence_Fast_GET_SIZE(updates.ptr()); ++n)
                each(PySequence_Fast_GET_ITEM(updates.ptr(), n), [&](const Tensor &t) {
                    add_tensor(t);
                    if (in_place) held.push_back(t);
                });
        } else {
            std::vector<size_t> ends; // of each client's tensors
            for (const py::object client : py::reinterpret_borrow<py::sequence>(updates)) {
                each(client, [&](const Tensor &t) { held.push_back(t); });
                ends.push_back(held.size());
            }
            size_t i = 0;
            for (const size_t end : ends) {
                for (; i < end; ++i) add_tensor(held[i]);
                ++n;
            }
        }
    }
    if (max_norm && !(*max_norm >= 0.0)) refuse("max_norm is a number that is not negative");
    if (out) {
        c.tensor(*out, 2, "out");
        const int type = value_type(out->scalar_type());
        if (!type) refuse("out must be float32, bfloat16 or float16");
        if (out->size(0) != n) refuse("out must have a row for each of the " + std::to_string(n) + " client(s)");
        if (n > 1 && out->stride(0) < out->size(1)) refuse("the rows of out overlap");
        int64_t at = 0;
        for (size_t i = 0; i <= sizes.size(); ++i) {
            const bool next = i == sizes.size() || (i > 0 && clients[i] != clients[i - 1]);
            if (next && i > 0 && at != out->size(1)) refuse("an update does not have the " + std::to_string(out->size(1)) + " values of a row of out");
            if (i == sizes.size()) break;
            if (next || i == 0) at = 0;
            outs.push_back(sizes[i] ? static_cast<char *>(out->data_ptr()) + (clients[i] * (n > 1 ? out->stride(0) : 0) + at) * out->element_size() : nullptr);
            at += sizes[i];
        }
        std::vector<bool> some(n);
        for (const int k : clients) some[k] = true;
        for (int k = 0; k < n; ++k)
            if (!some[k] && out->size(1)) refuse("an update does not have the " + std::to_string(out->size(1)) + " values of a row of out");
        out_dtypes.assign(sizes.size(), type);
    } else if (in_place) {
        for (const void *p : tensors) outs.push_back(const_cast<void *>(p));
        out_dtypes = dtypes;
    }
    const Tensor norms = c.empty({n}, at::kDouble);
    const int count = (int)sizes.size();
    const int *writes = out || in_place ? out_dtypes.data() : nullptr;
    const size_t need = n ? lb_clip_updates_workspace_bytes(n, count, sizes.data()) : 0;
    const Tensor ws = c.workspace(need);
    check(lb_clip_updates(c.context, n, count, clients.data(), tensors.data(), dtypes.data(), sizes.data(), max_norm ? *max_norm : HUGE_VAL,
                          out || in_place ? outs.data() : nullptr, writes, address<double>(norms), address<void>(ws), need, c.stream()));
    written(out);
    if (in_place)
        for (const Tensor &t : held) written(t);
    return norms;
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
    m.def("quantize_fp8", &quantize_fp8);
    m.def("dequantize_fp8", &dequantize_fp8);
    m.def("fp8_matmul", &fp8_matmul);
    m.def("clip_updates", &clip_updates);
    m.def("fp8_linear", &fp8_linear);
}
