// The host side of trips_amd/adamw.py, lookup.py, table_loss.py and dropout.py: what the C ABI takes of each tensor, collected from the objects
// that torch keeps. In Python a tensor's score of attributes and checks took 1.3 to 2 us, more than its share of the kernels'
// time in a step over a net (18 tensors 32 us a step and 17 so, 40 with copies 68 and 29), and a lookup 10 us.
#include <c10/hip/HIPStream.h>
#include <torch/csrc/DynamicTypes.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/extension.h>

#include <string>
#include <vector>

#include "../../../include/trips_lookup.h"
#include "../../../include/trips_loss.h"
#include "../../../include/trips_optim.h"

namespace py = pybind11;

namespace
{
// TRIPS_DTYPE_* of a tensor, or -1
int dtype_of(const at::Tensor& t)
{
    switch (t.scalar_type())
    {
        case at::kFloat: return TRIPS_DTYPE_F32;
        case at::kBFloat16: return TRIPS_DTYPE_BF16;
        case at::kHalf: return TRIPS_DTYPE_F16;
        default: return -1;
    }
}

const at::Tensor& tensor_of(PyObject* o, const char* what)
{
    if (!o || !THPVariable_Check(o)) throw py::type_error(std::string(what) + ": a tensor expected");
    return THPVariable_Unpack(o);
}

// One device for all tensors of a call, a GPU.
void check_device(const at::Tensor& t, int& device)
{
    const int own = t.is_cuda() ? (int)t.get_device() : -1;
    if (device >= 0 && own != device) throw std::runtime_error("all tensors of a call must be on one device");
    if (own < 0) throw std::runtime_error("the kernels need tensors on a GPU: there is no CPU implementation");
    device = own;
}

// A gradient as the kernels read it; a copy is kept in `temporaries`.
at::Tensor readable(const at::Tensor& g, std::vector<at::Tensor>& temporaries)
{
    if (g.layout() != at::kStrided) throw std::runtime_error("sparse gradients are not supported");
    if (dtype_of(g) < 0) throw std::runtime_error("gradients are float32, bfloat16 or float16, not " + std::string(torch::getTHPDtype(g.scalar_type())->name));
    if (g.is_contiguous()) return g;
    temporaries.push_back(g.detach().contiguous());
    return temporaries.back();
}

PyObject* item(PyObject* dict, PyObject* key)  // borrowed, or NULL
{
    PyObject* v = PyDict_GetItemWithError(dict, key);
    if (!v && PyErr_Occurred()) throw py::error_already_set();
    return v;
}

// A tensor of the optimiser's state, as the kernels expect it.
void* state_ptr(PyObject* st, const char* name, at::ScalarType type, int64_t n, int device)
{
    const at::Tensor& t = tensor_of(PyDict_GetItemString(st, name), name);
    if (t.scalar_type() != type || t.numel() != n || !t.is_contiguous() || !t.is_cuda() || t.get_device() != device)
        throw std::runtime_error(std::string("state of a parameter: ") + name + " is not a contiguous tensor of its type and size on the parameter's device");
    return t.data_ptr();
}

class StepTable
{
   public:
    // Everything that the step takes of the parameters with a gradient; (how many, their device or -1).
    std::pair<int, int> collect(const py::list& groups, const py::dict& state, const py::dict& copies, const py::object& grads, const py::function& make_state)
    {
        clear();
        int device        = -1;
        const bool own    = grads.is_none();
        const bool plain  = !own && PyDict_Check(grads.ptr());
        const bool copied = !copies.empty();
        for (const py::handle& g_ : groups)
        {
            const py::dict group = py::reinterpret_borrow<py::dict>(g_);
            const py::tuple betas(group["betas"]);
            const double lr = group["lr"].cast<double>(), b1 = betas[0].cast<double>(), b2 = betas[1].cast<double>(), eps = group["eps"].cast<double>(),
                         decay = group["weight_decay"].cast<double>();
            const py::list listed(group["params"]);
            tensors.reserve(tensors.size() + listed.size()), written.reserve(written.size() + 2 * listed.size() + 1);
            for (const py::handle& o : listed)
            {
                const at::Tensor& p = tensor_of(o.ptr(), "a parameter");
                at::Tensor g;
                if (own)
                    g = p.grad();
                else
                {
                    py::object v = plain ? py::reinterpret_borrow<py::object>(item(grads.ptr(), o.ptr()) ? item(grads.ptr(), o.ptr()) : Py_None) : grads.attr("get")(o);
                    if (!v.is_none()) g = tensor_of(v.ptr(), "a gradient");
                }
                if (!g.defined()) continue;
                g = readable(g, temporaries);
                TripsAdamWTensor t;
                t.weight_dtype = dtype_of(p), t.grad_dtype = dtype_of(g), t.n = p.numel();
                if (t.weight_dtype < 0 || !p.is_contiguous()) throw std::runtime_error("AdamW needs contiguous float32, bfloat16 or float16 parameters");
                if (g.numel() != t.n) throw std::runtime_error("a gradient of " + std::to_string(g.numel()) + " elements for a parameter of " + std::to_string(t.n));
                check_device(p, device);
                check_device(g, device);
                py::object st = py::reinterpret_borrow<py::object>(item(state.ptr(), o.ptr()));
                if (!st || !PyDict_Check(st.ptr()) || PyDict_Size(st.ptr()) == 0) st = make_state(o, group);
                const bool eight = PyDict_GetItemString(st.ptr(), "first_scale") != nullptr;
                t.state_bits     = eight ? 8 : 32;
                t.first_moment   = state_ptr(st.ptr(), "first_moment", eight ? at::kFloat8_e4m3fn : at::kFloat, t.n, device);
                t.second_moment  = state_ptr(st.ptr(), "second_moment", eight ? at::kFloat8_e5m2 : at::kFloat, t.n, device);
                const int64_t blocks = (t.n + TRIPS_MOMENT_BLOCK - 1) / TRIPS_MOMENT_BLOCK;
                t.first_scale    = eight ? (float*)state_ptr(st.ptr(), "first_scale", at::kFloat, blocks, device) : nullptr;
                t.second_scale   = eight ? (float*)state_ptr(st.ptr(), "second_scale", at::kFloat, blocks, device) : nullptr;
                t.step           = (int32_t*)state_ptr(st.ptr(), "step", at::kInt, 1, device);
                t.weights = p.data_ptr(), t.grads = g.data_ptr(), t.copy = nullptr, t.copy_dtype = 0;
                if (PyObject* c = copied ? item(copies.ptr(), o.ptr()) : nullptr)
                {
                    const at::Tensor& copy = tensor_of(c, "a copy");
                    t.copy = copy.data_ptr(), t.copy_dtype = dtype_of(copy);
                    // (what set_copy() checked may have changed since)
                    if (copy.numel() != t.n || t.copy_dtype < 0 || !copy.is_contiguous() || !copy.is_cuda() || copy.get_device() != device)
                        throw std::runtime_error("a copy is no longer a contiguous float32, bfloat16 or float16 tensor of its parameter's size, on its device");
                    written.push_back(copy);
                }
                t.lr = lr, t.beta1 = b1, t.beta2 = b2, t.eps = eps, t.weight_decay = decay;
                tensors.push_back(t);
                written.push_back(p);
            }
        }
        return {(int)tensors.size(), device};
    }

    // trips_adamw_step for what was collected; its return value.
    int step(uintptr_t ctx, uint32_t seed, const std::optional<at::Tensor>& grad_norm, bool compute_norm, float max_norm, float loss_scale, const at::Tensor& workspace,
             uintptr_t stream)
    {
        TripsAdamWOptions o;
        o.abi_version = TRIPS_ABI_VERSION, o.seed = seed, o.grad_norm = grad_norm ? (float*)grad_norm->data_ptr() : nullptr;
        o.compute_norm = compute_norm, o.max_norm = max_norm, o.loss_scale = loss_scale;
        const int rc = trips_adamw_step(reinterpret_cast<TripsCtx*>(ctx), tensors.data(), (int)tensors.size(), &o, workspace.data_ptr(), workspace.nbytes(),
                                        reinterpret_cast<void*>(stream));
        if (compute_norm && grad_norm) written.push_back(*grad_norm);
        if (rc == TRIPS_OK)  // (a backward pass that needs the old values raises)
            for (const at::Tensor& t : written)
                if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
        clear();
        return rc;
    }

    void clear() { tensors.clear(), written.clear(), temporaries.clear(); }

   private:
    std::vector<TripsAdamWTensor> tensors;
    std::vector<at::Tensor> written, temporaries;  // parameters, their copies and the norm
};

class NormTable
{
   public:
    std::pair<int, int> collect(const py::iterable& grads)
    {
        clear();
        int device = -1;
        for (const py::handle& o : grads)
        {
            const at::Tensor g = readable(tensor_of(o.ptr(), "a gradient"), temporaries);
            check_device(g, device);
            tensors.push_back(TripsGradTensor{g.data_ptr(), g.numel(), dtype_of(g)});
        }
        return {(int)tensors.size(), device};
    }
    int norm(uintptr_t ctx, float max_norm, float loss_scale, const at::Tensor& out, const at::Tensor& workspace, uintptr_t stream)
    {
        const int rc = trips_grad_norm(reinterpret_cast<TripsCtx*>(ctx), tensors.data(), (int)tensors.size(), max_norm, loss_scale, (float*)out.data_ptr(),
                                       workspace.data_ptr(), workspace.nbytes(), reinterpret_cast<void*>(stream));
        clear();
        return rc;
    }
    void clear() { tensors.clear(), temporaries.clear(); }

   private:
    std::vector<TripsGradTensor> tensors;
    std::vector<at::Tensor> temporaries;
};

// ---- table lookups ----

void check(int rc)
{
    if (rc == TRIPS_OK) return;
    py::gil_scoped_acquire gil;  // (a backward pass runs without it)
    py::module_::import("trips_amd._lib").attr("check")(rc);
}

int index_dtype_of(const at::Tensor& index, const char* name = "index", const char* what = "lookups need")
{
    if (index.scalar_type() != at::kInt && index.scalar_type() != at::kLong)
        throw py::value_error(std::string(name) + ": int32 or int64 expected, got " + std::string(torch::getTHPDtype(index.scalar_type())->name));
    if (!index.is_cuda()) throw std::runtime_error(std::string(what) + " tensors on a GPU: there is no CPU implementation");
    return index.scalar_type() == at::kInt ? TRIPS_INDEX_I32 : TRIPS_INDEX_I64;
}

// A matrix on the index's device with adjacent elements in a row (a copy of it, if need be), and the distance of its rows.
at::Tensor rows_of(const char* name, const at::Tensor& t, const at::Tensor& index, int64_t& stride, const char* where = "index's")
{
    if (t.dim() != 2 || dtype_of(t) < 0 || t.layout() != at::kStrided || t.device() != index.device())
        throw py::value_error(std::string(name) + ": a float32, bfloat16 or float16 matrix on the " + where + " device expected");
    const at::Tensor m = t.stride(1) != 1 && t.size(1) > 1 ? t.detach().contiguous() : t;
    stride             = m.size(0) > 1 ? m.stride(0) : m.size(1);
    return m;
}

at::Tensor bytes(size_t n, const at::Tensor& like)
{
    return n ? torch::empty({(int64_t)n}, like.options().dtype(at::kByte).requires_grad(false)) : at::Tensor();
}
void* data(const at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

void check_layout(int layout)
{
    if (layout != TRIPS_TABLE_COLUMNS && layout != TRIPS_TABLE_ROWS) throw py::value_error("layout: COLUMNS or ROWS expected, got " + std::to_string(layout));
}

TripsLookupDesc lookup_desc(int layout, int dtype, int index_dtype, int64_t texels, int64_t points, int64_t channels, float scale)
{
    TripsLookupDesc d{};
    d.abi_version = TRIPS_ABI_VERSION, d.layout = layout, d.dtype = dtype, d.index_dtype = index_dtype;
    d.num_texels = texels, d.num_points = points, d.num_channels = (int32_t)std::min<int64_t>(channels, INT32_MAX), d.scale = scale;
    return d;
}

at::Tensor lookup(uintptr_t ctx, uintptr_t stream, const at::Tensor& table, const at::Tensor& index, float scale, int layout)
{
    int64_t stride;
    check_layout(layout);
    const int index_dtype = index_dtype_of(index);
    const at::Tensor t    = rows_of("table", table, index, stride);
    const bool columns    = layout == TRIPS_TABLE_COLUMNS;
    const int64_t n = index.numel(), c = t.size(columns ? 0 : 1);
    TripsLookupDesc d = lookup_desc(layout, dtype_of(t), index_dtype, t.size(columns ? 1 : 0), n, c, scale);
    at::Tensor values = torch::empty({columns ? c : n, columns ? n : c}, t.options().requires_grad(false));
    if (c == 0 || n == 0) return values;
    d.table_stride = stride, d.values_stride = values.size(1);
    size_t need = 0;
    check(trips_lookup_workspace_size(&d, &need));
    const at::Tensor workspace = bytes(need, t), i = index.contiguous();
    check(trips_lookup_forward(reinterpret_cast<TripsCtx*>(ctx), &d, t.data_ptr(), i.data_ptr(), values.data_ptr(), data(workspace), need, reinterpret_cast<void*>(stream)));
    return values;
}

size_t plan_bytes(const at::Tensor& index, int64_t texels)
{
    if (texels < 0) throw py::value_error("num_texels = " + std::to_string(texels));
    size_t need = 0;
    check(trips_lookup_plan_workspace_size(texels, index.numel(), &need));
    return need;
}

std::pair<at::Tensor, at::Tensor> lookup_plan(uintptr_t ctx, uintptr_t stream, const at::Tensor& index, int64_t texels)
{
    const int index_dtype = index_dtype_of(index);
    const size_t need     = plan_bytes(index, texels);
    const auto options    = index.options().dtype(at::kInt);
    at::Tensor order = torch::empty({index.numel()}, options), starts = torch::empty({texels + 1}, options);
    const at::Tensor workspace = bytes(need, index), i = index.contiguous();
    check(trips_lookup_plan(reinterpret_cast<TripsCtx*>(ctx), texels, index.numel(), i.data_ptr(), index_dtype, (int32_t*)order.data_ptr(), (int32_t*)starts.data_ptr(),
                            data(workspace), need, reinterpret_cast<void*>(stream)));
    return {order, starts};
}

// A plan's tensor, as the kernels read it.
void check_plan(const char* name, const at::Tensor& t, int64_t n, const at::Tensor& index)
{
    if (t.scalar_type() != at::kInt || t.numel() != n || t.device() != index.device() || !t.is_contiguous())
        throw py::value_error(std::string("plan: ") + name + " of " + std::to_string(n) + " adjacent int32 numbers on the index's device expected");
}

// order, starts: of the plan, or neither: it is made here.
at::Tensor lookup_backward(uintptr_t ctx, uintptr_t stream, const at::Tensor& grad, const at::Tensor& index, const std::optional<at::Tensor>& order,
                           const std::optional<at::Tensor>& starts, int64_t texels, float scale, int layout, const std::optional<at::Tensor>& out)
{
    int64_t stride;
    check_layout(layout);
    const int index_dtype = index_dtype_of(index);
    const at::Tensor g    = rows_of("grad", grad, index, stride);
    const bool columns    = layout == TRIPS_TABLE_COLUMNS;
    const int64_t n = g.size(columns ? 1 : 0), c = g.size(columns ? 0 : 1);
    if (n != index.numel()) throw py::value_error("grad: " + std::to_string(n) + " points, index has " + std::to_string(index.numel()));
    if (order) check_plan("order", *order, n, index), check_plan("starts", *starts, texels + 1, index);
    const size_t plan = order ? 0 : plan_bytes(index, texels);
    TripsLookupDesc d  = lookup_desc(layout, dtype_of(g), index_dtype, texels, n, c, scale);
    const int64_t rows = columns ? c : texels, row = columns ? texels : c;
    at::Tensor d_table;
    if (out)
    {
        d_table = *out;
        if (d_table.dim() != 2 || d_table.size(0) != rows || d_table.size(1) != row || d_table.scalar_type() != g.scalar_type() || d_table.device() != g.device() ||
            (d_table.stride(1) != 1 && row > 1) || (rows > 1 && d_table.stride(0) < row))
            throw py::value_error("out: a tensor of the gradient's type of " + std::to_string(rows) + " x " + std::to_string(row) + " with adjacent elements in a row expected");
    }
    else
        d_table = torch::empty({rows, row}, g.options().requires_grad(false));
    if (rows == 0 || row == 0) return d_table;
    d.accumulate = out.has_value(), d.table_stride = rows > 1 ? d_table.stride(0) : row, d.values_stride = stride;
    size_t need = 0;
    check(trips_lookup_backward_workspace_size(&d, &need));
    // one piece of memory for it, and for the plan that is made here
    auto up = [](size_t b) { return (b + 255) & ~(size_t)255; };
    const size_t at_starts = up(need), at_order = at_starts + (order ? 0 : up((texels + 1) * 4)), at_plan = at_order + (order ? 0 : up(n * 4));
    const at::Tensor workspace = bytes(at_plan + plan, g);
    char* w                    = (char*)data(workspace);
    const int32_t *order_at, *starts_at;
    if (order)
        order_at = (const int32_t*)order->data_ptr(), starts_at = (const int32_t*)starts->data_ptr();
    else
    {
        const at::Tensor i = index.contiguous();
        order_at = (int32_t*)(w + at_order), starts_at = (int32_t*)(w + at_starts);
        check(trips_lookup_plan(reinterpret_cast<TripsCtx*>(ctx), texels, n, i.data_ptr(), index_dtype, (int32_t*)(w + at_order), (int32_t*)(w + at_starts), w + at_plan, plan,
                                reinterpret_cast<void*>(stream)));
    }
    check(trips_lookup_backward(reinterpret_cast<TripsCtx*>(ctx), &d, g.data_ptr(), order_at, starts_at, d_table.data_ptr(), w, need, reinterpret_cast<void*>(stream)));
    if (out && !d_table.is_inference()) d_table.unsafeGetTensorImpl()->bump_version();
    return d_table;
}

// ---- a table's cross entropy ----

int64_t stream_of(const at::Tensor& t) { return (int64_t)(uintptr_t)c10::hip::getCurrentHIPStream(t.get_device()).stream(); }

TripsTableLossDesc loss_desc(const at::Tensor& table, int64_t rows, double scale, int64_t reduction)
{
    TripsTableLossDesc d{};
    d.abi_version = TRIPS_ABI_VERSION, d.dtype = dtype_of(table), d.reduction = (int32_t)reduction, d.scale = (float)scale;
    d.num_rows = rows, d.num_entries = table.size(0), d.num_channels = (int32_t)std::min<int64_t>(table.size(1), INT32_MAX);
    return d;
}

// {loss, what the gradients need}
std::pair<at::Tensor, at::Tensor> table_loss(int64_t ctx, int64_t stream, const at::Tensor& rows, const at::Tensor& table, const at::Tensor& target, double scale, int64_t reduction)
{
    const int index_dtype = index_dtype_of(target, "target", "the cross entropy needs");
    int64_t rows_stride, table_stride;
    const at::Tensor x = rows_of("rows", rows, target, rows_stride, "target's"), w = rows_of("table", table, target, table_stride, "target's");
    if (w.scalar_type() != x.scalar_type() || w.size(1) != x.size(1))
        throw py::value_error("rows and table: matrices of one type and as many channels expected, got " + std::to_string(x.size(1)) + " and " + std::to_string(w.size(1)) + " channels");
    if (target.numel() != x.size(0)) throw py::value_error("target: " + std::to_string(target.numel()) + " entries for " + std::to_string(x.size(0)) + " rows");
    TripsTableLossDesc d = loss_desc(w, x.size(0), scale, reduction);
    d.index_dtype = index_dtype, d.rows_stride = rows_stride, d.table_stride = table_stride;
    size_t need = 0, keep = 0;
    check(trips_table_loss_workspace_size(&d, 0, &need));
    check(trips_table_loss_kept_size(&d, &keep));
    const auto options = x.options().dtype(at::kFloat).requires_grad(false);
    at::Tensor loss = reduction == TRIPS_REDUCE_NONE ? torch::empty({d.num_rows}, options) : torch::empty({}, options), kept = bytes(keep, x);
    const at::Tensor workspace = bytes(need, x), t = target.contiguous();
    check(trips_table_loss_forward(reinterpret_cast<TripsCtx*>(ctx), &d, x.data_ptr(), w.data_ptr(), t.data_ptr(), (float*)loss.data_ptr(), kept.data_ptr(), keep, data(workspace), need,
                                   reinterpret_cast<void*>(stream)));
    return {loss, kept};
}

// {d_rows, d_table}, undefined where they are not asked for
std::pair<at::Tensor, at::Tensor> table_loss_gradients(int64_t ctx, int64_t stream, const at::Tensor& d_loss, const at::Tensor& table, const at::Tensor& kept, int64_t rows, double scale,
                                                       int64_t reduction, bool want_rows, bool want_table)
{
    int64_t table_stride;
    const at::Tensor w   = rows_of("table", table, kept, table_stride, "rows'");
    TripsTableLossDesc d = loss_desc(w, rows, scale, reduction);
    const int64_t losses = reduction == TRIPS_REDUCE_NONE ? d.num_rows : 1;
    if (d_loss.scalar_type() != at::kFloat || d_loss.numel() != losses || d_loss.device() != w.device())
        throw py::value_error("the loss's gradient: " + std::to_string(losses) + " float32 numbers on the rows' device expected");
    if (kept.scalar_type() != at::kByte || !kept.is_contiguous()) throw py::value_error("kept is not what the loss left");
    d.table_stride = table_stride, d.d_rows_stride = d.d_table_stride = d.num_channels;
    const auto options = w.options().requires_grad(false);
    at::Tensor d_rows, d_table;
    if (want_rows) d_rows = torch::empty({d.num_rows, d.num_channels}, options);
    if (want_table) d_table = torch::empty({d.num_entries, d.num_channels}, options);
    size_t need = 0;
    check(trips_table_loss_workspace_size(&d, 1, &need));
    const at::Tensor workspace = bytes(need, w), g = d_loss.contiguous();
    check(trips_table_loss_backward(reinterpret_cast<TripsCtx*>(ctx), &d, w.data_ptr(), kept.data_ptr(), kept.nbytes(), (const float*)g.data_ptr(), data(d_rows), data(d_table),
                                    data(workspace), need, reinterpret_cast<void*>(stream)));
    return {d_rows, d_table};
}
std::pair<std::optional<at::Tensor>, std::optional<at::Tensor>> table_loss_backward(int64_t ctx, int64_t stream, const at::Tensor& d_loss, const at::Tensor& table, const at::Tensor& kept,
                                                                                    int64_t rows, double scale, int64_t reduction, bool want_rows, bool want_table)
{
    auto [d_rows, d_table] = table_loss_gradients(ctx, stream, d_loss, table, kept, rows, scale, reduction, want_rows, want_table);
    return {d_rows.defined() ? std::optional<at::Tensor>(d_rows) : std::nullopt, d_table.defined() ? std::optional<at::Tensor>(d_table) : std::nullopt};
}

// Gradients that cannot be differentiated again: where that could be asked for, it raises.
void only_once(torch::autograd::variable_list& grads, const at::Tensor& upstream)
{
    if (!at::GradMode::is_enabled() || !upstream.requires_grad()) return;
    torch::autograd::variable_list in;
    for (at::Tensor& g : grads)
        if (g.defined()) g = g.detach().set_requires_grad(true), in.push_back(g);
    if (in.empty()) return;
    auto error = std::make_shared<torch::autograd::DelayedError>("trying to differentiate twice a function that has its gradients once", (int64_t)in.size());
    auto out   = (*error)(std::move(in));
    size_t at  = 0;
    for (at::Tensor& g : grads)
        if (g.defined()) g = out[at++];
}

// The function that a graph records (in Python, its two ways through the interpreter would take as long as the kernels of a small problem: 25 rows
// of 5000 entries 104 us a pass, so 70).
struct TableLoss : torch::autograd::Function<TableLoss>
{
    static at::Tensor forward(torch::autograd::AutogradContext* own, const at::Tensor& rows, const at::Tensor& table, const at::Tensor& target, int64_t ctx, int64_t stream, double scale,
                              int64_t reduction)
    {
        auto [loss, kept] = table_loss(ctx, stream, rows.detach(), table.detach(), target, scale, reduction);
        own->save_for_backward({table, kept});
        own->saved_data["ctx"] = ctx, own->saved_data["scale"] = scale, own->saved_data["reduction"] = reduction, own->saved_data["rows"] = rows.size(0);
        return loss;
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* own, torch::autograd::variable_list upstream)
    {
        const auto saved = own->get_saved_variables();
        const at::Tensor d_loss = upstream[0], &table = saved[0], &kept = saved[1];
        torch::autograd::variable_list grads(7);
        if (!d_loss.defined()) return grads;
        auto [d_rows, d_table] = table_loss_gradients(own->saved_data["ctx"].toInt(), stream_of(kept), d_loss.detach(), table.detach(), kept, own->saved_data["rows"].toInt(),
                                                      own->saved_data["scale"].toDouble(), own->saved_data["reduction"].toInt(), own->needs_input_grad(0), own->needs_input_grad(1));
        grads[0] = d_rows, grads[1] = d_table;
        only_once(grads, d_loss);
        return grads;
    }
};
at::Tensor table_loss_graph(int64_t ctx, int64_t stream, const at::Tensor& rows, const at::Tensor& table, const at::Tensor& target, double scale, int64_t reduction)
{
    return TableLoss::apply(rows, table, target, ctx, stream, scale, reduction);
}

// ---- dropout ----

// {out, the step that was used (undefined where it was not read from the device, or is not asked for)}
std::pair<at::Tensor, at::Tensor> dropped(int64_t ctx, int64_t stream, const at::Tensor& x, double p, int64_t seed, int64_t call, int64_t step, const std::optional<at::Tensor>& step_at,
                                          const std::optional<at::Tensor>& residual, bool want_step)
{
    if (!(p >= 0.0 && p <= 1.0)) throw py::value_error("p: 0 to 1 expected, got " + std::to_string(p));
    if (dtype_of(x) < 0 || x.layout() != at::kStrided) throw py::value_error("x: a float32, bfloat16 or float16 tensor expected");
    if (!x.is_cuda()) throw std::runtime_error("dropout needs tensors on a GPU: there is no CPU implementation");
    if (residual && (residual->scalar_type() != x.scalar_type() || residual->sizes() != x.sizes() || residual->device() != x.device() || residual->layout() != at::kStrided))
        throw py::value_error("residual: a tensor of x's type and shape on its device expected");
    if (step_at && ((step_at->scalar_type() != at::kInt && step_at->scalar_type() != at::kLong) || step_at->numel() != 1 || step_at->device() != x.device()))
        throw py::value_error("step: a number, or one int32 or int64 on x's device, expected");
    TripsDropoutDesc d{};
    d.abi_version = TRIPS_ABI_VERSION, d.dtype = dtype_of(x), d.n = x.numel(), d.p = p, d.seed = (uint64_t)seed, d.call = (uint32_t)call, d.step = (uint32_t)step;
    const at::Tensor from = x.detach().contiguous(), added = residual ? residual->detach().contiguous() : at::Tensor();
    at::Tensor out = torch::empty(x.sizes(), x.options().requires_grad(false)), used;
    if (step_at && want_step) used = torch::empty({}, x.options().dtype(at::kInt).requires_grad(false));
    // (the low word of an int64)
    check(trips_dropout(reinterpret_cast<TripsCtx*>(ctx), &d, from.data_ptr(), data(added), step_at ? (const uint32_t*)step_at->data_ptr() : nullptr, (uint32_t*)data(used), out.data_ptr(),
                        reinterpret_cast<void*>(stream)));
    return {out, used};
}
std::pair<at::Tensor, std::optional<at::Tensor>> dropout(int64_t ctx, int64_t stream, const at::Tensor& x, double p, int64_t seed, int64_t call, int64_t step,
                                                         const std::optional<at::Tensor>& step_at, const std::optional<at::Tensor>& residual, bool want_step)
{
    auto [out, used] = dropped(ctx, stream, x, p, seed, call, step, step_at, residual, want_step);
    return {out, used.defined() ? std::optional<at::Tensor>(used) : std::nullopt};
}

struct Dropout : torch::autograd::Function<Dropout>
{
    static at::Tensor forward(torch::autograd::AutogradContext* own, const at::Tensor& x, const std::optional<at::Tensor>& residual, int64_t ctx, int64_t stream, double p, int64_t seed,
                              int64_t call, int64_t step, const std::optional<at::Tensor>& step_at)
    {
        // (the step may have gone on when the gradient is made: what was used is kept)
        auto [out, used] = dropped(ctx, stream, x, p, seed, call, step, step_at, residual, true);
        if (used.defined()) own->save_for_backward({used});
        own->saved_data["ctx"] = ctx, own->saved_data["p"] = p, own->saved_data["seed"] = seed, own->saved_data["call"] = call, own->saved_data["step"] = step;
        own->saved_data["used"] = used.defined(), own->saved_data["residual"] = residual.has_value();
        return out;
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* own, torch::autograd::variable_list upstream)
    {
        torch::autograd::variable_list grads(9);
        const at::Tensor g = upstream[0];
        if (!g.defined()) return grads;
        if (own->needs_input_grad(0))
        {
            const std::optional<at::Tensor> used = own->saved_data["used"].toBool() ? std::optional<at::Tensor>(own->get_saved_variables()[0]) : std::nullopt;
            grads[0] = dropped(own->saved_data["ctx"].toInt(), stream_of(g), g, own->saved_data["p"].toDouble(), own->saved_data["seed"].toInt(), own->saved_data["call"].toInt(),
                               own->saved_data["step"].toInt(), used, std::nullopt, false)
                           .first;
            only_once(grads, g);
        }
        if (own->saved_data["residual"].toBool() && own->needs_input_grad(1)) grads[1] = g;  // (an edge of its own where there is one)
        return grads;
    }
};
at::Tensor dropout_graph(int64_t ctx, int64_t stream, const at::Tensor& x, const std::optional<at::Tensor>& residual, double p, int64_t seed, int64_t call, int64_t step,
                         const std::optional<at::Tensor>& step_at)
{
    return Dropout::apply(x, residual, ctx, stream, p, seed, call, step, step_at);
}
}  // namespace

PYBIND11_MODULE(_trips_host, m)
{
    py::class_<StepTable>(m, "StepTable").def(py::init<>()).def("collect", &StepTable::collect).def("step", &StepTable::step).def("clear", &StepTable::clear);
    py::class_<NormTable>(m, "NormTable").def(py::init<>()).def("collect", &NormTable::collect).def("norm", &NormTable::norm).def("clear", &NormTable::clear);
    m.def("lookup", &lookup);
    m.def("lookup_plan", &lookup_plan);
    m.def("lookup_backward", &lookup_backward);
    m.def("table_loss", &table_loss);
    m.def("table_loss_backward", &table_loss_backward);
    m.def("table_loss_graph", &table_loss_graph);
    m.def("dropout", &dropout);
    m.def("dropout_graph", &dropout_graph);
}
