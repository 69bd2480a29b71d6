// The binding's part for dense rows of scores and sparse ones of the teacher's or the router's: routing, the gradient for a matrix's
// stored values, distillation.  Included by binding.cpp, inside its namespace, after what both parts share.
//
// ops.py calls the py_* functions.  Where a gradient is wanted they go through the dispatcher, whose Autograd
// kernels are here; otherwise straight to the library.  Each backward is an operator too, so that it traces.
#pragma once

struct ScoreLibrary {
    int (*route)(const csrspmm_b200_route_args*, int32_t*, int32_t*, float*, csrspmm_b200_stream_t);
    int (*route_backward)(const csrspmm_b200_route_args*, const int32_t*, const float*, const float*, int64_t, void*, int64_t, csrspmm_b200_stream_t);
    int (*sddmm)(int32_t, int32_t, int32_t, int64_t, const int32_t*, const int32_t*, const float*, int64_t, const float*, int64_t, float, float*,
                 csrspmm_b200_stream_t);
    int (*transposed_pays)(int32_t, int32_t, int64_t);
    int (*transposed)(int32_t, int32_t, int32_t, int64_t, const int32_t*, const int32_t*, const float*, const float*, int64_t, float, float*, int64_t,
                      csrspmm_b200_stream_t);
    int (*distill)(const csrspmm_b200_distill_args*, float*, float*, csrspmm_b200_stream_t);
    int (*distill_backward)(const csrspmm_b200_distill_args*, const float*, const float*, int64_t, void*, int64_t, csrspmm_b200_stream_t);
    int (*distill_grad)(const csrspmm_b200_distill_args*, const float*, int64_t, float*, void*, int64_t, csrspmm_b200_stream_t);
};
ScoreLibrary g_scores = {};

// A matrix with unit stride along its rows and rows that do not overlap; any other one is copied.
at::Tensor row_major(const at::Tensor& t) { return (t.stride(1) == 1 || t.size(1) <= 1) && rows_apart(t) ? t : t.contiguous(); }
int64_t leading(const at::Tensor& t) { return t.size(0) > 1 ? std::max(t.stride(0), t.size(1)) : t.size(1); }

int score_type(const at::Tensor& t, const char* name)
{
    if (t.is_cuda() && t.dim() == 2) {
        if (t.scalar_type() == at::kFloat) return CSRSPMM_B200_F32;
        if (t.scalar_type() == at::kHalf) return CSRSPMM_B200_F16;
        if (t.scalar_type() == at::kBFloat16) return CSRSPMM_B200_BF16;
    }
    throw std::runtime_error(std::string(name) + " must be a 2-D CUDA tensor of float32, float16 or bfloat16");
}

void want_vector(const at::Tensor& t, at::ScalarType type, at::Device device, const char* message)
{
    want(t.is_cuda() && t.device() == device && t.scalar_type() == type && t.dim() == 1 && t.is_contiguous(), message);
}

// The backward passes are kernels and have no derivative themselves: a second one is refused, not taken as zero.
void first_derivative_only(const char* what)
{
    if (at::GradMode::is_enabled()) throw std::runtime_error(std::string(what) + " has no second derivative (create_graph)");
}

void refuse_tangents(std::initializer_list<at::Tensor> tensors, const char* what)
{
    for (const at::Tensor& t : tensors) TORCH_CHECK_NOT_IMPLEMENTED(!torch::autograd::isFwGradDefined(t), what, " has no forward-mode derivative");
}

bool wants_gradient(const at::Tensor& t, const char* what)
{
    refuse_tangents({t}, what);
    return at::GradMode::is_enabled() && t.requires_grad();
}

int32_t as_int32(int64_t v, const char* message)
{
    want(v >= 0 && v <= INT32_MAX, message);
    return static_cast<int32_t>(v);
}

template <class F>
auto dispatched(const char* name)
{
    return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<F>();
}

// ---- routing ----------------------------------------------------------------------------------------------

using Triple = std::tuple<at::Tensor, at::Tensor, at::Tensor>;

int score_id(c10::string_view name)
{
    if (name == "softmax") return CSRSPMM_B200_SOFTMAX;
    if (name == "sigmoid") return CSRSPMM_B200_SIGMOID;
    throw std::runtime_error("unknown score '" + std::string(name) + "' (softmax or sigmoid)");
}

csrspmm_b200_route_args route_args(const at::Tensor& x, int64_t k, c10::string_view score, int64_t groups, int64_t top_groups, int64_t group_top,
                                   bool renormalize, double scale)
{
    csrspmm_b200_route_args a = {};
    a.struct_size = sizeof(a);
    a.score_type = score_type(x, "logits");
    a.T = as_int32(x.size(0), "logits has too many rows");
    a.E = as_int32(x.size(1), "logits has too many columns");
    a.k = as_int32(k, "k out of range");
    a.score = score_id(score);
    a.groups = as_int32(groups, "groups out of range");
    a.top_groups = as_int32(top_groups, "top_groups out of range");
    a.group_top = as_int32(group_top, "group_top out of range");
    a.renormalize = renormalize;
    a.scale = static_cast<float>(scale);
    return a;
}

Triple op_route(const at::Tensor& logits, int64_t k, const std::optional<at::Tensor>& bias, c10::string_view score, int64_t groups, int64_t top_groups,
                int64_t group_top, bool renormalize, double scale)
{
    return as_operator([&]() -> Triple {
        csrspmm_b200_route_args a = route_args(logits, k, score, groups, top_groups, group_top, renormalize, scale);
        const auto device = logits.device();
        if (bias) {
            want_vector(*bias, at::kFloat, device, "bias must be a contiguous 1-D float32 tensor on the logits' device");
            want(bias->size(0) == a.E, "bias must have one entry per expert");
            a.bias = address<float>(*bias);
        }
        const c10::cuda::CUDAGuard guard(device);
        const at::Tensor x = row_major(logits);
        a.scores = x.data_ptr();
        a.ld = leading(x);
        const int64_t n = static_cast<int64_t>(a.T) * a.k;
        want(n <= INT32_MAX, "more than 2^31 - 1 entries");
        at::Tensor rp = new_array(static_cast<int64_t>(a.T) + 1, at::kInt, device), ci = new_array(n, at::kInt, device), va = new_array(n, at::kFloat, device);
        int status;
        {
            const WithoutGil nogil;
            status = g_scores.route(&a, address<int32_t>(rp), address<int32_t>(ci), address<float>(va), current_stream(device));
        }
        check(status, "csrspmm_b200_route");
        return {rp, ci, va};
    });
}

at::Tensor op_route_backward(const at::Tensor& grad, const at::Tensor& logits, const at::Tensor& ci, const at::Tensor& va, int64_t k, c10::string_view score,
                             bool renormalize, double scale)
{
    return as_operator([&] {
        csrspmm_b200_route_args a = route_args(logits, k, score, 1, 1, 1, renormalize, scale);
        const auto device = logits.device();
        const int64_t n = static_cast<int64_t>(a.T) * a.k;
        want_vector(ci, at::kInt, device, "col_idx must be a contiguous 1-D int32 tensor on the logits' device");
        want_vector(va, at::kFloat, device, "values must be a contiguous 1-D float32 tensor on the logits' device");
        want(grad.is_cuda() && grad.device() == device && grad.scalar_type() == at::kFloat && grad.dim() == 1,
             "the gradient must be a 1-D float32 tensor on the logits' device");
        want(ci.size(0) == n && va.size(0) == n && grad.size(0) == n, "col_idx, values and gradient must have k entries per row");
        const c10::cuda::CUDAGuard guard(device);
        const at::Tensor x = row_major(logits);
        a.scores = x.data_ptr();
        a.ld = leading(x);
        at::Tensor dx = at::detail::empty_cuda({a.T, a.E}, logits.scalar_type(), device, std::nullopt);
        int status;
        {
            const WithoutGil nogil;
            status = g_scores.route_backward(&a, address<int32_t>(ci), address<float>(va), address<float>(grad), n > 1 ? grad.stride(0) : 1,
                                             dx.data_ptr(), a.E, current_stream(device));
        }
        check(status, "csrspmm_b200_route_backward");
        return dx;
    });
}

Triple call_route(const at::Tensor& logits, int64_t k, const std::optional<at::Tensor>& bias, c10::string_view score, int64_t groups, int64_t top_groups,
                  int64_t group_top, bool renormalize, double scale)
{
    static const auto op = dispatched<decltype(op_route)>("csrspmm_b200::route");
    return op.call(logits, k, bias, score, groups, top_groups, group_top, renormalize, scale);
}

at::Tensor call_route_backward(const at::Tensor& grad, const at::Tensor& logits, const at::Tensor& ci, const at::Tensor& va, int64_t k,
                               c10::string_view score, bool renormalize, double scale)
{
    static const auto op = dispatched<decltype(op_route_backward)>("csrspmm_b200::route_backward");
    return op.call(grad, logits, ci, va, k, score, renormalize, scale);
}

struct RouteWithGradient : torch::autograd::Function<RouteWithGradient> {
    static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const at::Tensor& logits, int64_t k,
                                                  const std::optional<at::Tensor>& bias, std::string score, int64_t groups, int64_t top_groups,
                                                  int64_t group_top, bool renormalize, double scale)
    {
        ctx->set_materialize_grads(false);
        Triple out;
        {
            at::AutoDispatchBelowADInplaceOrView below;
            out = call_route(logits, k, bias, score, groups, top_groups, group_top, renormalize, scale);
        }
        const auto& [rp, ci, va] = out;
        ctx->mark_non_differentiable({rp, ci});
        ctx->save_for_backward({logits, ci, va});
        ctx->saved_data["k"] = k;
        ctx->saved_data["score"] = score;
        ctx->saved_data["renormalize"] = renormalize;
        ctx->saved_data["scale"] = scale;
        return {rp, ci, va};
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads)
    {
        torch::autograd::variable_list out(9);
        if (ctx->needs_input_grad(0) && grads[2].defined()) {
            first_derivative_only("csrspmm_b200::route");
            const auto saved = ctx->get_saved_variables();
            out[0] = call_route_backward(grads[2], saved[0], saved[1], saved[2], ctx->saved_data["k"].toInt(), ctx->saved_data["score"].toStringRef(),
                                         ctx->saved_data["renormalize"].toBool(), ctx->saved_data["scale"].toDouble());
        }
        return out;
    }
};

Triple autograd_route(const at::Tensor& logits, int64_t k, const std::optional<at::Tensor>& bias, c10::string_view score, int64_t groups,
                      int64_t top_groups, int64_t group_top, bool renormalize, double scale)
{
    refuse_tangents({logits}, "route");
    const auto out = RouteWithGradient::apply(logits, k, bias, std::string(score), groups, top_groups, group_top, renormalize, scale);
    return {out[0], out[1], out[2]};
}

// route(logits, k, bias|None, score, groups, top_groups, group_top, renormalize, scale) -> (row_ptr, col_idx, values)
PyObject* py_route(PyObject*, PyObject* const* args, Py_ssize_t nargs)
{
    BEGIN_BINDING
    expect_args(nargs, 9);
    const at::Tensor logits = tensor_of(args[0], "logits");
    std::optional<at::Tensor> bias;
    if (args[2] != Py_None) bias = tensor_of(args[2], "bias");
    const char* score = PyUnicode_AsUTF8(args[3]);
    if (score == nullptr) throw python_error();
    const bool renormalize = PyObject_IsTrue(args[7]) == 1;
    const auto run = wants_gradient(logits, "route") ? call_route : op_route;
    const Triple out = run(logits, as_int_of(args[1]), bias, score, as_int_of(args[4]), as_int_of(args[5]), as_int_of(args[6]), renormalize,
                           as_double(args[8]));
    return Py_BuildValue("(NNN)", THPVariable_Wrap(std::get<0>(out)), THPVariable_Wrap(std::get<1>(out)), THPVariable_Wrap(std::get<2>(out)));
    END_BINDING
}

// ---- the gradient for the stored values -----------------------------------------------------------------------

at::Tensor op_sddmm(const at::Tensor& rp, const at::Tensor& ci, const at::Tensor& G, const at::Tensor& B, double alpha)
{
    return as_operator([&] {
        want(rp.is_cuda() && ci.is_cuda() && G.is_cuda() && B.is_cuda(), "row_ptr, col_idx, G and B must be CUDA tensors");
        const auto device = B.device();
        want(rp.device() == device && ci.device() == device && G.device() == device, "all tensors must be on the same device");
        want_vector(rp, at::kInt, device, "row_ptr must be contiguous 1-D int32");
        want_vector(ci, at::kInt, device, "col_idx must be contiguous 1-D int32");
        want(G.scalar_type() == at::kFloat && B.scalar_type() == at::kFloat && G.dim() == 2 && B.dim() == 2, "G and B must be 2-D float32");
        want(rp.size(0) >= 1 && G.size(0) == rp.size(0) - 1, "G must have a row for each row of the matrix");
        want(G.size(1) == B.size(1), "G and B must have the same number of columns");
        const int32_t M = as_int32(G.size(0), "too many rows"), Kd = as_int32(B.size(0), "B has too many rows"),
                      Nd = as_int32(B.size(1), "B has too many columns");
        want(ci.size(0) == 0 || (M > 0 && Kd > 0), "entries, but no rows or columns");
        const c10::cuda::CUDAGuard guard(device);
        const at::Tensor g = row_major(G), b = row_major(B);
        at::Tensor out = new_array(ci.size(0), at::kFloat, device);
        int status;
        {
            const WithoutGil nogil;
            status = g_scores.sddmm(M, Kd, Nd, ci.size(0), address<int32_t>(rp), address<int32_t>(ci), address<float>(g), leading(g), address<float>(b),
                                    leading(b), static_cast<float>(alpha), address<float>(out), current_stream(device));
        }
        check(status, "csrspmm_b200_sddmm");
        return out;
    });
}

at::Tensor call_sddmm(const at::Tensor& rp, const at::Tensor& ci, const at::Tensor& G, const at::Tensor& B, double alpha)
{
    static const auto op = dispatched<decltype(op_sddmm)>("csrspmm_b200::sddmm");
    return op.call(rp, ci, G, B, alpha);
}

// No derivative: none is recorded, and a tangent is refused, not dropped.
at::Tensor autograd_sddmm(const at::Tensor& rp, const at::Tensor& ci, const at::Tensor& G, const at::Tensor& B, double alpha)
{
    refuse_tangents({G, B}, "sddmm");
    at::AutoDispatchBelowADInplaceOrView below;
    return call_sddmm(rp, ci, G, B, alpha);
}

// alpha * A^T * G: in one launch where the matrix is small, else by its transpose
at::Tensor op_spmm_transposed(const at::Tensor& rp, const at::Tensor& ci, const at::Tensor& va, const at::Tensor& G, c10::SymInt rows, double alpha)
{
    return as_operator([&] {
        const int64_t Kd = rows.expect_int();
        check_csr(rp, ci, va, G, false);
        want(va.size(0) == ci.size(0), "values and col_idx differ in length");
        want(G.size(0) == rp.size(0) - 1, "G must have a row for each row of the matrix");
        const int32_t Nd = as_int32(G.size(1), "G has too many columns"), M = as_int32(G.size(0), "too many rows");
        // an odd number of columns is counted in single floats, as those of an unaligned G are read
        const bool whole = Nd % 4 == 0 ? reinterpret_cast<uintptr_t>(G.data_ptr()) % 16 == 0 && leading(G) % 4 == 0
                                       : reinterpret_cast<uintptr_t>(G.data_ptr()) % 8 == 0 && leading(G) % 2 == 0;
        if (!g_scores.transposed_pays(as_int32(Kd, "too many columns"), whole ? Nd : Nd | 1, ci.size(0))) {
            Product q;
            std::tie(q.rp, q.ci, q.va) = transpose(rp, ci, va, Kd);
            q.B = G;
            q.alpha = alpha;
            return run_product(q);
        }
        want(ci.size(0) == 0 || (M > 0 && Kd > 0), "entries, but no rows or columns");
        const c10::cuda::CUDAGuard guard(G.device());
        at::Tensor C = at::detail::empty_cuda({Kd, G.size(1)}, at::kFloat, G.device(), std::nullopt);
        int status;
        {
            const WithoutGil nogil;
            status = g_scores.transposed(M, static_cast<int32_t>(Kd), Nd, ci.size(0), address<int32_t>(rp), address<int32_t>(ci), address<float>(va),
                                         address<float>(G), leading(G), static_cast<float>(alpha), address<float>(C), G.size(1),
                                         current_stream(G.device()));
        }
        check(status, "csrspmm_b200_spmm_transposed");
        return C;
    });
}

at::Tensor call_spmm_transposed(const at::Tensor& rp, const at::Tensor& ci, const at::Tensor& va, const at::Tensor& G, c10::SymInt rows, double alpha)
{
    static const auto op = dispatched<decltype(op_spmm_transposed)>("csrspmm_b200::spmm_transposed");
    return op.call(rp, ci, va, G, rows, alpha);
}

at::Tensor op_weighted_spmm(const at::Tensor& rp, const at::Tensor& ci, const at::Tensor& va, const at::Tensor& B, double alpha)
{
    return op_spmm(rp, ci, va, B, alpha, "auto");
}

at::Tensor call_weighted_spmm(const at::Tensor& rp, const at::Tensor& ci, const at::Tensor& va, const at::Tensor& B, double alpha)
{
    static const auto op = dispatched<decltype(op_weighted_spmm)>("csrspmm_b200::weighted_spmm");
    return op.call(rp, ci, va, B, alpha);
}

// dvalues = sddmm(dC, B), dB = alpha * A^T dC
struct WeightedSpmm : torch::autograd::Function<WeightedSpmm> {
    static at::Tensor forward(torch::autograd::AutogradContext* ctx, const at::Tensor& rp, const at::Tensor& ci, const at::Tensor& va,
                              const at::Tensor& B, double alpha)
    {
        ctx->save_for_backward({rp, ci, B.requires_grad() ? va : at::Tensor(), va.requires_grad() ? B : at::Tensor()});
        ctx->saved_data["Kd"] = B.sym_size(0);
        ctx->saved_data["alpha"] = alpha;
        at::AutoDispatchBelowADInplaceOrView below;
        return call_weighted_spmm(rp, ci, va, B, alpha);
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads)
    {
        torch::autograd::variable_list out(5);
        if (!grads[0].defined()) return out;
        first_derivative_only("csrspmm_b200::weighted_spmm");
        const auto saved = ctx->get_saved_variables();
        const double alpha = ctx->saved_data["alpha"].toDouble();
        const at::Tensor G = grads[0].contiguous();
        if (ctx->needs_input_grad(2)) out[2] = call_sddmm(saved[0], saved[1], G, saved[3], alpha);
        if (ctx->needs_input_grad(3)) out[3] = call_spmm_transposed(saved[0], saved[1], saved[2], G, ctx->saved_data["Kd"].toSymInt(), alpha);
        return out;
    }
};

at::Tensor autograd_weighted_spmm(const at::Tensor& rp, const at::Tensor& ci, const at::Tensor& va, const at::Tensor& B, double alpha)
{
    refuse_tangents({va, B}, "weighted_spmm");
    return WeightedSpmm::apply(rp, ci, va, B, alpha);
}

// sddmm(row_ptr, col_idx, G, B, alpha) -> values
PyObject* py_sddmm(PyObject*, PyObject* const* args, Py_ssize_t nargs)
{
    BEGIN_BINDING
    expect_args(nargs, 5);
    const at::Tensor G = tensor_of(args[2], "G"), B = tensor_of(args[3], "B");
    refuse_tangents({G, B}, "sddmm");
    return THPVariable_Wrap(op_sddmm(tensor_of(args[0], "row_ptr"), tensor_of(args[1], "col_idx"), G, B, as_double(args[4])));
    END_BINDING
}

// weighted_spmm(row_ptr, col_idx, values, B, alpha) -> C
PyObject* py_weighted_spmm(PyObject*, PyObject* const* args, Py_ssize_t nargs)
{
    BEGIN_BINDING
    expect_args(nargs, 5);
    const at::Tensor values = tensor_of(args[2], "A_values"), B = tensor_of(args[3], "B");
    const bool for_values = wants_gradient(values, "weighted_spmm"), for_B = wants_gradient(B, "weighted_spmm");
    const auto run = for_values || for_B ? call_weighted_spmm : op_weighted_spmm;
    return THPVariable_Wrap(run(tensor_of(args[0], "A_row_ptr"), tensor_of(args[1], "A_col_idx"), values, B, as_double(args[4])));
    END_BINDING
}

// ---- distillation -----------------------------------------------------------------------------------------------

// Keeps the tensors that the arguments point to.
struct Distillation {
    csrspmm_b200_distill_args a = {};
    at::Tensor x;

    Distillation(const at::Tensor& logits, const at::Tensor& rp, const at::Tensor& ci, const at::Tensor& va, double temperature, bool log_probs)
    {
        a.struct_size = sizeof(a);
        a.logit_type = score_type(logits, "logits");
        const auto device = logits.device();
        want_vector(rp, at::kInt, device, "row_ptr must be a contiguous 1-D int32 tensor on the logits' device");
        want_vector(ci, at::kInt, device, "col_idx must be a contiguous 1-D int32 tensor on the logits' device");
        want_vector(va, at::kFloat, device, "values must be a contiguous 1-D float32 tensor on the logits' device");
        want(rp.size(0) == logits.size(0) + 1, "row_ptr must have one entry more than logits has rows");
        want(ci.size(0) == va.size(0), "values and col_idx differ in length");
        a.T = as_int32(logits.size(0), "logits has too many rows");
        a.V = as_int32(logits.size(1), "logits has too many columns");
        x = row_major(logits);
        a.logits = x.data_ptr();
        a.ld = leading(x);
        a.nnz = ci.size(0);
        a.row_ptr = address<int32_t>(rp);
        a.col_idx = address<int32_t>(ci);
        a.values = address<float>(va);
        a.temperature = static_cast<float>(temperature);
        a.log_probs = log_probs;
    }
    at::Tensor new_gradient() const { return at::detail::empty_cuda({a.T, a.V}, x.scalar_type(), x.device(), std::nullopt); }
};

// A weight for each row of `logits`, or one for all
void want_weights(const at::Tensor& w, const at::Tensor& logits)
{
    want(w.is_cuda() && w.device() == logits.device() && w.scalar_type() == at::kFloat, "weights must be float32 on the logits' device");
    want(w.dim() == 0 || (w.dim() == 1 && w.size(0) == logits.size(0)), "weights must be one number or one per row");
}
int64_t weight_stride(const at::Tensor& w) { return w.dim() == 0 ? 0 : w.stride(0); }

// (loss, stats)
std::tuple<at::Tensor, at::Tensor> distill_forward(const at::Tensor& logits, const at::Tensor& rp, const at::Tensor& ci, const at::Tensor& va,
                                                   double temperature, bool log_probs, bool with_stats)
{
    score_type(logits, "logits");
    const c10::cuda::CUDAGuard guard(logits.device());
    const Distillation d(logits, rp, ci, va, temperature, log_probs);
    const auto device = logits.device();
    at::Tensor loss = new_array(d.a.T, at::kFloat, device), stats;
    if (with_stats) stats = new_array(4 * static_cast<int64_t>(d.a.T), at::kFloat, device);
    int status;
    {
        const WithoutGil nogil;
        status = g_scores.distill(&d.a, address<float>(loss), with_stats ? address<float>(stats) : nullptr, current_stream(device));
    }
    check(status, "csrspmm_b200_distill");
    return {loss, stats};
}

at::Tensor op_distill_loss(const at::Tensor& logits, const at::Tensor& rp, const at::Tensor& ci, const at::Tensor& va, double temperature, bool log_probs)
{
    return as_operator([&] { return std::get<0>(distill_forward(logits, rp, ci, va, temperature, log_probs, false)); });
}

std::tuple<at::Tensor, at::Tensor> op_distill_with_stats(const at::Tensor& logits, const at::Tensor& rp, const at::Tensor& ci, const at::Tensor& va,
                                                         double temperature, bool log_probs)
{
    return as_operator([&] { return distill_forward(logits, rp, ci, va, temperature, log_probs, true); });
}

at::Tensor op_distill_backward(const at::Tensor& grad, const at::Tensor& logits, const at::Tensor& rp, const at::Tensor& ci, const at::Tensor& va,
                               const at::Tensor& stats, double temperature, bool log_probs)
{
    return as_operator([&] {
        score_type(logits, "logits");
        const c10::cuda::CUDAGuard guard(logits.device());
        const Distillation d(logits, rp, ci, va, temperature, log_probs);
        want_weights(grad, logits);
        want_vector(stats, at::kFloat, logits.device(), "stats must be a contiguous 1-D float32 tensor on the logits' device");
        want(stats.size(0) == 4 * logits.size(0), "stats must have four entries per row");
        at::Tensor dx = d.new_gradient();
        int status;
        {
            const WithoutGil nogil;
            status = g_scores.distill_backward(&d.a, address<float>(stats), address<float>(grad), weight_stride(grad), dx.data_ptr(), d.a.V,
                                               current_stream(logits.device()));
        }
        check(status, "csrspmm_b200_distill_backward");
        return dx;
    });
}

std::tuple<at::Tensor, at::Tensor> op_distill_loss_grad(const at::Tensor& logits, const at::Tensor& rp, const at::Tensor& ci, const at::Tensor& va,
                                                        const at::Tensor& weight, double temperature, bool log_probs)
{
    return as_operator([&]() -> std::tuple<at::Tensor, at::Tensor> {
        score_type(logits, "logits");
        const c10::cuda::CUDAGuard guard(logits.device());
        const Distillation d(logits, rp, ci, va, temperature, log_probs);
        want_weights(weight, logits);
        at::Tensor loss = new_array(d.a.T, at::kFloat, logits.device()), dx = d.new_gradient();
        int status;
        {
            const WithoutGil nogil;
            status = g_scores.distill_grad(&d.a, address<float>(weight), weight_stride(weight), address<float>(loss), dx.data_ptr(), d.a.V,
                                           current_stream(logits.device()));
        }
        check(status, "csrspmm_b200_distill_grad");
        return {loss, dx};
    });
}

at::Tensor call_distill_loss(const at::Tensor& logits, const at::Tensor& rp, const at::Tensor& ci, const at::Tensor& va, double temperature, bool log_probs)
{
    static const auto op = dispatched<decltype(op_distill_loss)>("csrspmm_b200::distill_loss");
    return op.call(logits, rp, ci, va, temperature, log_probs);
}

// The teacher's values have no gradient here: the teacher is not trained.
struct DistillWithGradient : torch::autograd::Function<DistillWithGradient> {
    static at::Tensor forward(torch::autograd::AutogradContext* ctx, const at::Tensor& logits, const at::Tensor& rp, const at::Tensor& ci,
                              const at::Tensor& va, double temperature, bool log_probs)
    {
        static const auto op = dispatched<decltype(op_distill_with_stats)>("csrspmm_b200::distill_with_stats");
        TORCH_CHECK(!va.requires_grad(), "distill_loss has no gradient for the teacher's values");
        at::Tensor loss, stats;
        {
            at::AutoDispatchBelowADInplaceOrView below;
            std::tie(loss, stats) = op.call(logits, rp, ci, va, temperature, log_probs);
        }
        ctx->save_for_backward({logits, rp, ci, va, stats});
        ctx->saved_data["temperature"] = temperature;
        ctx->saved_data["log_probs"] = log_probs;
        return loss;
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads)
    {
        static const auto op = dispatched<decltype(op_distill_backward)>("csrspmm_b200::distill_backward");
        torch::autograd::variable_list out(6);
        if (ctx->needs_input_grad(0) && grads[0].defined()) {
            first_derivative_only("csrspmm_b200::distill_loss");
            const auto s = ctx->get_saved_variables();
            out[0] = op.call(grads[0], s[0], s[1], s[2], s[3], s[4], ctx->saved_data["temperature"].toDouble(), ctx->saved_data["log_probs"].toBool());
        }
        return out;
    }
};

at::Tensor autograd_distill_loss(const at::Tensor& logits, const at::Tensor& rp, const at::Tensor& ci, const at::Tensor& va, double temperature,
                                 bool log_probs)
{
    refuse_tangents({logits, va}, "distill_loss");
    return DistillWithGradient::apply(logits, rp, ci, va, temperature, log_probs);
}

// The gradient is handed out; none is recorded.
std::tuple<at::Tensor, at::Tensor> autograd_distill_loss_grad(const at::Tensor& logits, const at::Tensor& rp, const at::Tensor& ci, const at::Tensor& va,
                                                              const at::Tensor& weight, double temperature, bool log_probs)
{
    static const auto op = dispatched<decltype(op_distill_loss_grad)>("csrspmm_b200::distill_loss_grad");
    refuse_tangents({logits, va, weight}, "distill_loss_grad");
    at::AutoDispatchBelowADInplaceOrView below;
    return op.call(logits, rp, ci, va, weight, temperature, log_probs);
}

// distill_loss(logits, row_ptr, col_idx, values, temperature, log_probs) -> loss
PyObject* py_distill_loss(PyObject*, PyObject* const* args, Py_ssize_t nargs)
{
    BEGIN_BINDING
    expect_args(nargs, 6);
    const at::Tensor logits = tensor_of(args[0], "logits"), values = tensor_of(args[3], "values");
    want(!wants_gradient(values, "distill_loss"), "distill_loss has no gradient for the teacher's values");
    const auto run = wants_gradient(logits, "distill_loss") ? call_distill_loss : op_distill_loss;
    return THPVariable_Wrap(run(logits, tensor_of(args[1], "row_ptr"), tensor_of(args[2], "col_idx"), values, as_double(args[4]),
                                PyObject_IsTrue(args[5]) == 1));
    END_BINDING
}

// distill_loss_grad(logits, row_ptr, col_idx, values, weight, temperature, log_probs) -> (loss, dlogits)
PyObject* py_distill_loss_grad(PyObject*, PyObject* const* args, Py_ssize_t nargs)
{
    BEGIN_BINDING
    expect_args(nargs, 7);
    const at::Tensor logits = tensor_of(args[0], "logits"), values = tensor_of(args[3], "values"), weight = tensor_of(args[4], "weight");
    refuse_tangents({logits, values, weight}, "distill_loss_grad");
    const auto out = op_distill_loss_grad(logits, tensor_of(args[1], "row_ptr"), tensor_of(args[2], "col_idx"), values, weight, as_double(args[5]),
                                          PyObject_IsTrue(args[6]) == 1);
    return Py_BuildValue("(NN)", THPVariable_Wrap(std::get<0>(out)), THPVariable_Wrap(std::get<1>(out)));
    END_BINDING
}

TORCH_LIBRARY_IMPL(csrspmm_b200, CUDA, scores)
{
    scores.impl("route", op_route);
    scores.impl("route_backward", op_route_backward);
    scores.impl("sddmm", op_sddmm);
    scores.impl("spmm_transposed", op_spmm_transposed);
    scores.impl("weighted_spmm", op_weighted_spmm);
    scores.impl("distill_loss", op_distill_loss);
    scores.impl("distill_with_stats", op_distill_with_stats);
    scores.impl("distill_backward", op_distill_backward);
    scores.impl("distill_loss_grad", op_distill_loss_grad);
}

TORCH_LIBRARY_IMPL(csrspmm_b200, Autograd, scores)
{
    scores.impl("route", autograd_route);
    scores.impl("sddmm", autograd_sddmm);
    scores.impl("distill_loss_grad", autograd_distill_loss_grad);
    scores.impl("weighted_spmm", autograd_weighted_spmm);
    scores.impl("distill_loss", autograd_distill_loss);
}
