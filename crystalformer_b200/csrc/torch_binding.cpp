// The operators of an encoder layer beside the attention as torch functions: checks of arguments, outputs and workspaces from torch's
// allocator, the current stream of the tensors' device, and one autograd node each.  Around the C ABI and in C++ because the calls
// are short: of a training step's 250 us on the host through ctypes and a Python autograd function, 150 were spent outside the library
// (a backward runs on a thread of autograd's own, where Python code is slow).
#include <c10/core/AutogradState.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/extension.h>

#include "crystalformer_b200.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptTensor = std::optional<Tensor>;

// What Python gets as TypeError, ValueError and NotImplementedError; other std::runtime_errors become RuntimeError.
struct TypeProblem : std::runtime_error { using std::runtime_error::runtime_error; };
struct ValueProblem : std::runtime_error { using std::runtime_error::runtime_error; };
struct NotThere : std::runtime_error { using std::runtime_error::runtime_error; };

// A C-ABI call that returned a negative status: CrystalformerB200Error in Python.
struct LibraryError : std::runtime_error {
    std::string name, message;
    int code;
    LibraryError(const char *n, int c, const char *m) : std::runtime_error(std::string(n) + ": " + m), name(n), message(m), code(c) {}
};
#define CF_CALL(name, ...)                                                        \
    do {                                                                          \
        const int code_ = name(__VA_ARGS__);                                      \
        if (code_ != CF_OK) throw LibraryError(#name, code_, cf_last_error());    \
    } while (0)

template <class... Parts>
std::string text(const Parts &...parts)
{
    std::ostringstream s;
    (s << ... << parts);
    return s.str();
}

int type_code(at::ScalarType t)
{
    return t == at::kFloat ? CF_FLOAT32 : t == at::kBFloat16 ? CF_BFLOAT16 : t == at::kHalf ? CF_FLOAT16 : -1;
}

// The tensor that gives a call its type and device.
void check_first(const Tensor &t, const char *name, int64_t dims)
{
    if (!t.is_cuda()) throw std::runtime_error(text(name, " must be a CUDA tensor: crystalformer_b200 has no CPU path"));
    if (type_code(t.scalar_type()) < 0) throw TypeProblem(text(name, " must be float32, bfloat16 or float16, got ", t.scalar_type()));
    if (t.dim() != dims) throw ValueProblem(text(name, " must have ", dims, " dimensions, got the shape ", t.sizes()));
}

// ... and one that has to lie where it does, with its type and a shape.
void check_like(const Tensor &t, const Tensor &first, const char *name, at::IntArrayRef shape)
{
    if (!t.defined()) return;
    if (t.device() != first.device()) throw std::runtime_error(text(name, " is on ", t.device(), ", expected ", first.device()));
    if (t.scalar_type() != first.scalar_type()) throw TypeProblem(text(name, " must be ", first.scalar_type(), ", got ", t.scalar_type()));
    if (t.sizes() != shape) throw ValueProblem(text(name, " must have the shape ", shape, ", got ", t.sizes()));
}

void *address(const Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; }
Tensor or_none(const OptTensor &t) { return t.has_value() ? *t : Tensor(); }
// What is read by address, negated first where that is still to be done (the imaginary part of a conjugated view).
Tensor values_of(const Tensor &t) { return t.is_neg() ? t.resolve_neg() : t; }
// the rows of t with their entries as neighbours
Tensor with_rows(const Tensor &t) { return values_of(t.size(-1) <= 1 || t.stride(-1) != 1 ? t.contiguous() : t); }
Tensor whole(const Tensor &t) { return t.defined() ? values_of(t.contiguous()) : t; }

struct Place {  // a call's device and stream
    c10::cuda::CUDAGuard guard;
    void *stream;
    explicit Place(const Tensor &t) : guard(t.device()), stream(c10::cuda::getCurrentCUDAStream(t.device().index()).stream()) {}
};
Tensor bytes_like(const Tensor &t, int64_t n) { return at::empty({n}, t.options().dtype(at::kByte)); }

// The gradients of an operator with a backward pass but no second one: where one could be asked for, an error waits behind them.
variable_list once(variable_list grads)
{
    if (!at::GradMode::is_enabled()) return grads;
    variable_list some;
    for (Tensor &g : grads)
        if (g.defined()) some.push_back(g.detach().requires_grad_(true));
    auto wait = std::make_shared<torch::autograd::DelayedError>("the operator can be differentiated once only", (int64_t)some.size());
    some = (*wait)(std::move(some));
    size_t i = 0;
    for (Tensor &g : grads)
        if (g.defined()) g = some[i++];
    return grads;
}

// A tangent of forward-mode differentiation would end here without a word: outputs are written by address.
void refuse_tangents(std::initializer_list<const Tensor *> tensors)
{
    if (!c10::AutogradState::get_tls_state().get_fw_grad_mode()) return;
    for (const Tensor *t : tensors)
        if (t->defined() && t->_fw_grad(0).defined()) throw NotThere("the operator has no forward-mode derivative");
}

bool wants_gradients(std::initializer_list<const Tensor *> tensors)
{
    if (!at::GradMode::is_enabled()) return false;
    for (const Tensor *t : tensors)
        if (t->defined() && t->requires_grad()) return true;
    return false;
}

// ---- embedding -----------------------------------------------------------------------------------------------------------------
Tensor whole_ids(const Tensor &ids, const Tensor &first)
{
    if (ids.device() != first.device()) throw std::runtime_error(text("ids are on ", ids.device(), ", expected ", first.device()));
    if (!at::isIntegralType(ids.scalar_type(), false)) throw TypeProblem(text("ids must be whole numbers, got ", ids.scalar_type()));
    return whole(ids.to(at::kLong));
}

Tensor embed_fwd(const Tensor &ids_in, const Tensor &table_in, double scale)
{
    refuse_tangents({&table_in});
    check_first(table_in, "table", 2);
    const Tensor table = values_of(table_in);
    const Tensor ids = whole_ids(ids_in, table);
    const int64_t V = table.size(0), D = table.size(1);
    const Place place(table);
    auto shape = ids.sizes().vec();
    shape.push_back(D);
    Tensor out = at::empty(shape, table.options());
    CF_CALL(cf_embed_fwd, table.data_ptr(), table.stride(0), table.stride(1), type_code(table.scalar_type()), ids.data_ptr<int64_t>(), ids.numel(), V, D, scale,
            out.data_ptr(), place.stream);
    return out;
}

Tensor embed_bwd(const Tensor &ids_in, const Tensor &gout, int64_t V, double scale, bool transposed)
{
    refuse_tangents({&gout});
    if (gout.dim() < 1) throw ValueProblem("gout must have rows");
    const int64_t D = gout.size(-1), N = ids_in.numel();
    if (gout.sizes().slice(0, gout.dim() - 1) != ids_in.sizes()) throw ValueProblem(text("gout ", gout.sizes(), " does not belong to ids ", ids_in.sizes()));
    const Tensor rows = with_rows(gout.reshape({N, D}));
    check_first(rows, "gout", 2);
    const Tensor ids = whole_ids(ids_in, gout);
    const Place place(gout);
    Tensor gtable = at::empty(transposed ? at::IntArrayRef{D, V} : at::IntArrayRef{V, D}, gout.options());
    Tensor work = bytes_like(gout, cf_embed_bwd_workspace_bytes(N, D));
    CF_CALL(cf_embed_bwd, rows.data_ptr(), N > 1 ? rows.stride(0) : D, type_code(gout.scalar_type()), ids.data_ptr<int64_t>(), N, V, D, scale, gtable.data_ptr(),
            transposed, work.data_ptr(), place.stream);
    return transposed ? gtable.t() : gtable;
}

struct Embed : torch::autograd::Function<Embed> {
    static Tensor forward(AutogradContext *ctx, const Tensor &table, const Tensor &ids, double scale)
    {
        ctx->save_for_backward({ids});
        ctx->saved_data["rows"] = table.size(0);
        ctx->saved_data["scale"] = scale;
        ctx->saved_data["transposed"] = table.stride(0) < table.stride(1);
        return embed_fwd(ids, table, scale);
    }
    static variable_list backward(AutogradContext *ctx, variable_list g)
    {
        const auto saved = ctx->get_saved_variables();
        return once({embed_bwd(saved[0], g[0], ctx->saved_data["rows"].toInt(), ctx->saved_data["scale"].toDouble(), ctx->saved_data["transposed"].toBool()), Tensor(),
                     Tensor()});
    }
};

Tensor embed(const Tensor &ids, const Tensor &table, double scale)
{
    refuse_tangents({&table});
    return wants_gradients({&table}) ? Embed::apply(table, ids, scale) : embed_fwd(ids, table, scale);
}

// ---- norms and rotation of queries and keys ----------------------------------------------------------------------------------------
struct HeadCall {
    Tensor q, k, wq, wk, pos, waves;
    cf_qk_norm args{};

    HeadCall(const Tensor &q_in, const Tensor &k_in, const Tensor &wq_in, const Tensor &wk_in, const Tensor &pos_in, const Tensor &waves_in, double eps,
             bool interleaved)
    {
        refuse_tangents({&q_in, &k_in, &wq_in, &wk_in, &pos_in, &waves_in});
        check_first(q_in, "q", 3);
        check_first(k_in, "k", 3);
        const int64_t N = q_in.size(0), Hq = q_in.size(1), D = q_in.size(2), Hk = k_in.size(1);
        check_like(k_in, q_in, "k", {N, Hk, D});
        auto weight = [&](const Tensor &w, const char *name, int64_t H) {
            if (w.defined() && w.dim() == 2) check_like(w, q_in, name, {H, D});
            else check_like(w, q_in, name, {D});
            return whole(w);
        };
        wq = weight(wq_in, "wq", Hq);
        wk = weight(wk_in, "wk", Hk);
        q = with_rows(q_in);
        k = with_rows(k_in);
        args.wave_heads = 1;
        if (waves_in.defined()) {
            if (waves_in.dim() != 3 || !pos_in.defined() || pos_in.dim() != 2 || pos_in.size(0) != N || pos_in.size(1) != waves_in.size(2))
                throw ValueProblem(text("waves (heads, pairs, axes) and pos (rows, axes) go together: got ", waves_in.sizes(), " and ",
                                                 pos_in.defined() ? text(pos_in.sizes()) : "none", " for ", N, " rows"));
            for (const Tensor &t : {pos_in, waves_in}) {
                if (t.device() != q.device()) throw std::runtime_error(text("positions and waves are on ", t.device(), ", expected ", q.device()));
                if (t.scalar_type() != at::kFloat) throw TypeProblem(text("positions and waves must be float32, got ", t.scalar_type()));
            }
            pos = whole(pos_in);
            waves = whole(waves_in);
            args.wave_heads = waves.size(0); args.P = waves.size(1); args.C = waves.size(2);
        } else if (pos_in.defined()) {
            throw ValueProblem("positions without waves");
        }
        args.type = type_code(q.scalar_type());
        args.interleaved = interleaved;
        args.N = N; args.Hq = Hq; args.Hk = Hk; args.D = D;
        args.q = address(q); args.q_row = q.stride(0); args.q_head = q.stride(1);
        args.k = address(k); args.k_row = k.stride(0); args.k_head = k.stride(1);
        args.wq = address(wq); args.wq_head = wq.defined() && wq.dim() == 2 ? D : 0;
        args.wk = address(wk); args.wk_head = wk.defined() && wk.dim() == 2 ? D : 0;
        args.pos = static_cast<const float *>(address(pos));
        args.waves = static_cast<const float *>(address(waves));
        args.eps = eps;
    }
};

variable_list qk_norm_fwd(const HeadCall &c)
{
    const Place place(c.q);
    Tensor q = at::empty(c.q.sizes(), c.q.options()), k = at::empty(c.k.sizes(), c.k.options());
    CF_CALL(cf_qk_norm_fwd, &c.args, q.data_ptr(), k.data_ptr(), place.stream);
    return {q, k};
}

variable_list qk_norm_bwd(const HeadCall &c, const Tensor &gq_out, const Tensor &gk_out, bool want_wq, bool want_wk)
{
    refuse_tangents({&gq_out, &gk_out});
    check_like(gq_out, c.q, "gq_out", c.q.sizes());
    check_like(gk_out, c.q, "gk_out", c.k.sizes());
    const Place place(c.q);
    const Tensor a = whole(gq_out), b = whole(gk_out);
    Tensor gq = at::empty(c.q.sizes(), c.q.options()), gk = at::empty(c.k.sizes(), c.k.options()), gwq, gwk, work;
    if (want_wq && c.wq.defined()) gwq = at::empty(c.wq.sizes(), c.wq.options());
    if (want_wk && c.wk.defined()) gwk = at::empty(c.wk.sizes(), c.wk.options());
    if (gwq.defined() || gwk.defined()) work = bytes_like(c.q, cf_qk_norm_bwd_workspace_bytes(&c.args));
    CF_CALL(cf_qk_norm_bwd, &c.args, a.data_ptr(), b.data_ptr(), gq.data_ptr(), gk.data_ptr(), address(gwq), address(gwk), address(work), place.stream);
    return {gq, gk, gwq, gwk};
}

struct NormalizeRotate : torch::autograd::Function<NormalizeRotate> {
    static variable_list forward(AutogradContext *ctx, const Tensor &q, const Tensor &k, const OptTensor &wq_in, const OptTensor &wk_in, const OptTensor &pos_in,
                                 const OptTensor &waves_in, double eps, bool interleaved)
    {
        const Tensor wq = or_none(wq_in), wk = or_none(wk_in), pos = or_none(pos_in), waves = or_none(waves_in);
        ctx->save_for_backward({q, k, wq, wk, pos, waves});
        ctx->saved_data["eps"] = eps;
        ctx->saved_data["interleaved"] = interleaved;
        return qk_norm_fwd(HeadCall(q, k, wq, wk, pos, waves, eps, interleaved));
    }
    static variable_list backward(AutogradContext *ctx, variable_list g)
    {
        const auto s = ctx->get_saved_variables();
        const HeadCall call(s[0], s[1], s[2], s[3], s[4], s[5], ctx->saved_data["eps"].toDouble(), ctx->saved_data["interleaved"].toBool());
        const bool with_wq = s[2].defined(), with_wk = s[3].defined();  // (an argument that is not there has no edge)
        variable_list grads = qk_norm_bwd(call, g[0], g[1], with_wq && ctx->needs_input_grad(2), with_wk && ctx->needs_input_grad(with_wq ? 3 : 2));
        grads.resize(8);
        return once(std::move(grads));
    }
};

std::tuple<Tensor, Tensor> normalize_rotate(const Tensor &q, const Tensor &k, const OptTensor &wq_in, const OptTensor &wk_in, const OptTensor &pos,
                                            const OptTensor &waves, double eps, bool interleaved)
{
    const Tensor wq = or_none(wq_in), wk = or_none(wk_in);
    const Tensor place = or_none(pos), cycles = or_none(waves);
    refuse_tangents({&q, &k, &wq, &wk, &place, &cycles});
    if (wants_gradients({&place, &cycles})) throw ValueProblem("positions and waves have no gradients here: detach them");
    const variable_list y = wants_gradients({&q, &k, &wq, &wk})
                                ? NormalizeRotate::apply(q, k, wq_in, wk_in, pos, waves, eps, interleaved)
                                : qk_norm_fwd(HeadCall(q, k, wq, wk, place, cycles, eps, interleaved));
    return {y[0], y[1]};
}

std::tuple<Tensor, Tensor, OptTensor, OptTensor> normalize_rotate_backward(const Tensor &q, const Tensor &k, const OptTensor &wq, const OptTensor &wk,
                                                                           const OptTensor &pos, const OptTensor &waves, double eps, bool interleaved,
                                                                           const Tensor &gq_out, const Tensor &gk_out, bool want_wq, bool want_wk)
{
    const HeadCall call(q, k, or_none(wq), or_none(wk), or_none(pos), or_none(waves), eps, interleaved);
    const variable_list g = qk_norm_bwd(call, gq_out, gk_out, want_wq, want_wk);
    auto opt = [](const Tensor &t) { return t.defined() ? OptTensor(t) : OptTensor(); };
    return {g[0], g[1], opt(g[2]), opt(g[3])};
}

// ---- gated feed-forward ------------------------------------------------------------------------------------------------------------
struct GatedCall {
    Tensor t[7];  // x, w_gate, w_up, w_down, b_gate, b_up, b_down
    cf_gated_ffn args{};

    GatedCall(const Tensor &x, const Tensor &wg, const Tensor &wu, const Tensor &wd, const Tensor &bg, const Tensor &bu, const Tensor &bd, int64_t activation)
    {
        refuse_tangents({&x, &wg, &wu, &wd, &bg, &bu, &bd});
        check_first(x, "x", 2);
        if (!wg.defined() || !wu.defined() || !wd.defined()) throw TypeProblem("the weights must be tensors");
        if (wg.dim() != 2) throw ValueProblem(text("w_gate must have 2 dimensions, got the shape ", wg.sizes()));
        const int64_t N = x.size(0), D = x.size(1), F = wg.size(0);
        check_like(wg, x, "w_gate", {F, D});
        check_like(wu, x, "w_up", {F, D});
        check_like(wd, x, "w_down", {D, F});
        check_like(bg, x, "b_gate", {F});
        check_like(bu, x, "b_up", {F});
        check_like(bd, x, "b_down", {D});
        t[0] = with_rows(x);
        t[1] = whole(wg); t[2] = whole(wu); t[3] = whole(wd);
        t[4] = whole(bg); t[5] = whole(bu); t[6] = whole(bd);
        args.type = type_code(x.scalar_type());
        args.activation = (int32_t)activation;
        args.N = N; args.D = D; args.F = F;
        args.x = address(t[0]);
        args.ldx = N > 1 ? t[0].stride(0) : D;
        args.w_gate = address(t[1]); args.w_up = address(t[2]); args.w_down = address(t[3]);
        args.b_gate = address(t[4]); args.b_up = address(t[5]); args.b_down = address(t[6]);
    }
};

Tensor gated_fwd(const GatedCall &c)
{
    const Place place(c.t[0]);
    Tensor y = at::empty(c.t[0].sizes(), c.t[0].options());
    Tensor work = bytes_like(y, cf_gated_ffn_workspace_bytes(&c.args, nullptr, 0));
    CF_CALL(cf_gated_ffn_fwd, &c.args, y.data_ptr(), work.data_ptr(), place.stream);
    return y;
}

variable_list gated_bwd(const GatedCall &c, const Tensor &gy_in, const std::array<bool, 7> &wanted)
{
    refuse_tangents({&gy_in});
    check_like(gy_in, c.t[0], "gy", c.t[0].sizes());
    const Place place(c.t[0]);
    const Tensor gy = whole(gy_in);
    variable_list grads(7);
    for (int i = 0; i < 7; ++i)
        if (wanted[i] && c.t[i].defined()) grads[i] = at::empty(c.t[i].sizes(), c.t[i].options());
    Tensor work = bytes_like(gy, cf_gated_ffn_workspace_bytes(&c.args, gy.data_ptr(), 1));
    const cf_gated_ffn_grads to{gy.data_ptr(), address(grads[0]), address(grads[1]), address(grads[2]), address(grads[3]), address(grads[4]), address(grads[5]),
                                address(grads[6])};
    CF_CALL(cf_gated_ffn_bwd, &c.args, &to, work.data_ptr(), place.stream);
    return grads;
}

struct Gated : torch::autograd::Function<Gated> {
    static Tensor forward(AutogradContext *ctx, const Tensor &x, const Tensor &wg, const Tensor &wu, const Tensor &wd, const OptTensor &bg_in,
                          const OptTensor &bu_in, const OptTensor &bd_in, int64_t activation)
    {
        const Tensor bg = or_none(bg_in), bu = or_none(bu_in), bd = or_none(bd_in);
        ctx->save_for_backward({x, wg, wu, wd, bg, bu, bd});
        ctx->saved_data["activation"] = activation;
        return gated_fwd(GatedCall(x, wg, wu, wd, bg, bu, bd, activation));
    }
    static variable_list backward(AutogradContext *ctx, variable_list g)
    {
        const auto s = ctx->get_saved_variables();
        std::array<bool, 7> wanted;
        for (size_t i = 0, edge = 0; i < 7; ++i) wanted[i] = s[i].defined() && ctx->needs_input_grad(edge++);  // (no edge where there is no argument)
        variable_list grads = gated_bwd(GatedCall(s[0], s[1], s[2], s[3], s[4], s[5], s[6], ctx->saved_data["activation"].toInt()), g[0], wanted);
        grads.resize(8);
        return once(std::move(grads));
    }
};

Tensor gated(const Tensor &x_in, const Tensor &wg, const Tensor &wu, const Tensor &wd, const OptTensor &bg_in, const OptTensor &bu_in, const OptTensor &bd_in,
             int64_t activation)
{
    const Tensor bg = or_none(bg_in), bu = or_none(bu_in), bd = or_none(bd_in);
    refuse_tangents({&x_in, &wg, &wu, &wd, &bg, &bu, &bd});
    const bool rows = x_in.dim() == 2 || x_in.dim() == 0;
    const Tensor x = rows ? x_in : x_in.reshape({-1, x_in.size(-1)});
    const Tensor y = wants_gradients({&x, &wg, &wu, &wd, &bg, &bu, &bd}) ? Gated::apply(x, wg, wu, wd, bg_in, bu_in, bd_in, activation)
                                                                      : gated_fwd(GatedCall(x, wg, wu, wd, bg, bu, bd, activation));
    return rows ? y : y.view(x_in.sizes());
}

std::vector<OptTensor> gated_backward(const Tensor &x, const Tensor &wg, const Tensor &wu, const Tensor &wd, const OptTensor &bg, const OptTensor &bu,
                                      const OptTensor &bd, int64_t activation, const Tensor &gy, const std::array<bool, 7> &wanted)
{
    const variable_list g = gated_bwd(GatedCall(x, wg, wu, wd, or_none(bg), or_none(bu), or_none(bd), activation), gy, wanted);
    std::vector<OptTensor> out;
    for (const Tensor &t : g) out.push_back(t.defined() ? OptTensor(t) : OptTensor());
    return out;
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m)
{
    pybind11::register_exception_translator([](std::exception_ptr p) {
        try {
            if (p) std::rethrow_exception(p);
        } catch (const LibraryError &e) {
            pybind11::object kind = pybind11::module_::import("crystalformer_b200._lib").attr("CrystalformerB200Error");
            PyErr_SetObject(kind.ptr(), kind(e.name, e.code, e.message).ptr());
        } catch (const TypeProblem &e) {
            PyErr_SetString(PyExc_TypeError, e.what());
        } catch (const ValueProblem &e) {
            PyErr_SetString(PyExc_ValueError, e.what());
        } catch (const NotThere &e) {
            PyErr_SetString(PyExc_NotImplementedError, e.what());
        }
    });
    using Free = pybind11::call_guard<pybind11::gil_scoped_release>;
    m.def("embed", &embed, Free());
    m.def("embed_fwd", [](const Tensor &ids, const Tensor &table, double scale) { at::NoGradGuard no; return embed_fwd(ids, table, scale); }, Free());
    m.def("embed_bwd", [](const Tensor &ids, const Tensor &gout, int64_t V, double scale, bool transposed) {
        at::NoGradGuard no;
        return embed_bwd(ids, gout, V, scale, transposed);
    }, Free());
    m.def("normalize_rotate", &normalize_rotate, Free());
    m.def("normalize_rotate_backward", [](const Tensor &q, const Tensor &k, const OptTensor &wq, const OptTensor &wk, const OptTensor &pos, const OptTensor &waves,
                                          double eps, bool interleaved, const Tensor &gq_out, const Tensor &gk_out, bool want_wq, bool want_wk) {
        at::NoGradGuard no;
        return normalize_rotate_backward(q, k, wq, wk, pos, waves, eps, interleaved, gq_out, gk_out, want_wq, want_wk);
    }, Free());
    m.def("gated", &gated, Free());
    m.def("gated_backward", [](const Tensor &x, const Tensor &wg, const Tensor &wu, const Tensor &wd, const OptTensor &bg, const OptTensor &bu, const OptTensor &bd,
                               int64_t activation, const Tensor &gy, const std::array<bool, 7> &wanted) {
        at::NoGradGuard no;
        return gated_backward(x, wg, wu, wd, bg, bu, bd, activation, gy, wanted);
    }, Free());
}
