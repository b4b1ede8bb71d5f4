// The operators of a pre-norm gated block: C++ autograd functions over tgt_add_rms_norm_*, tgt_gated_linear_* and tgt_linear_epilogue_*.
//
//   torchgt::add_rms_norm(x, residual?, weight, eps) -> (sum, y)
//   torchgt::add_rms_norm_8bit(x, residual?, weight, eps) -> (sum, codes, scales)                       no gradients
//   torchgt::quantize_rows(w) -> (codes, scales)                                                          no gradients
//   torchgt::gated_linear(x, gate_weight, up_weight, gate_bias?, up_bias?, act) -> h
//   torchgt::gated_linear_8bit(x, x_scales, gate_weight, gate_scales, up_weight, up_scales, gate_bias?, up_bias?, act, dtype) -> h     no gradients
//   torchgt::linear_act(x, weight, bias?, residual?, act) -> y
//   torchgt::linear_act_8bit(x, x_scales, weight, weight_scales, bias?, residual?, act, dtype) -> y       no gradients
//
// Calls that nobody differentiates go past the autograd node: a call for one row is bound by the host.
#include "torch_common.h"

namespace {

using namespace tgt_torch;
using Optional = c10::optional<Tensor>;

bool given(const Optional& t) { return t.has_value() && t->defined(); }
Optional compact(const Optional& t) { return given(t) ? Optional(t->contiguous()) : Optional(); }

// The rows and the features of x, checked
struct RowsOf {
    int64_t N = 0, C = 0;
    RowsOf(const Tensor& x, const char* op) {
        on_gpu(x, op);
        TORCH_CHECK(x.dim() >= 1 && x.size(-1) >= 1, op, ": x must have at least one feature, in its last dimension");
        C = x.size(-1);
        TORCH_CHECK(C <= (1 << 24), op, ": at most 2^24 features, got ", C);
        N = x.numel() / C;
        TORCH_CHECK(N <= 0x7fffffff, op, ": at most 2^31 - 1 rows, got ", N);
    }
};
void same_kind(const Tensor& t, const Tensor& x, const char* op, const char* name) {
    same_gpu(t, x, op, name);
    TORCH_CHECK(t.scalar_type() == x.scalar_type(), op, ": ", name, " must be ", x.scalar_type(), " like x, got ", t.scalar_type());
}
void no_gradients(std::initializer_list<const Tensor*> ts, const char* op) {
    Wanted w;
    for (const Tensor* t : ts) w.look(*t);
    TORCH_CHECK(!w.node(), op, " has no gradient: call it under torch.no_grad() or on detached tensors");
}
// a backward that is itself recorded would give gradients that depend on nothing
void once(const char* op) { TORCH_CHECK(!at::GradMode::is_enabled(), op, ": no second derivatives (backward with create_graph=True)"); }
std::vector<int64_t> with_last(const Tensor& x, int64_t last) {
    std::vector<int64_t> s(x.sizes().vec());
    s.back() = last;
    return s;
}

// ---- norm --------------------------------------------------------------------------------------------------------------------------
void check_norm(const Tensor& x, const Optional& r, const Tensor& weight, const RowsOf& rows, const char* op) {
    (void)dtype_code(x);
    same_kind(weight, x, op, "weight");
    TORCH_CHECK(weight.dim() == 1 && weight.size(0) == rows.C, op, ": weight must be [", rows.C, "]");
    if (given(r)) {
        same_kind(*r, x, op, "residual");
        TORCH_CHECK(r->sizes() == x.sizes(), op, ": residual must have x's shape");
    }
}
struct Normed { Tensor s, y, rstd; };
Normed norm_forward(const Tensor& x, const Optional& r, const Tensor& w, const RowsOf& rows, double eps, bool keep) {
    Tensor x2 = x.contiguous(), r2 = given(r) ? r->contiguous() : Tensor();
    Normed o;
    o.s = given(r) ? at::empty_like(x2, at::MemoryFormat::Contiguous) : x2;
    o.y = at::empty_like(x2, at::MemoryFormat::Contiguous);
    if (keep) o.rstd = at::empty({rows.N}, x.options().dtype(at::kFloat));
    check(tgt_add_rms_norm_fwd(x2.data_ptr(), given(r) ? r2.data_ptr() : nullptr, w.data_ptr(), rows.N, (int)rows.C, (float)eps, dtype_code(x),
                               given(r) ? o.s.data_ptr() : nullptr, o.y.data_ptr(), keep ? o.rstd.data_ptr<float>() : nullptr, stream_of(x)),
          "tgt_add_rms_norm_fwd");
    return o;
}
struct AddRmsNorm : public torch::autograd::Function<AddRmsNorm> {
    static variable_list forward(AutogradContext* ctx, Tensor x, Optional r, Tensor weight, double eps) {
        const RowsOf rows(x, "add_rms_norm");
        c10::DeviceGuard guard(x.device());
        Tensor w = weight.contiguous();
        Normed o = norm_forward(x, r, w, rows, eps, true);
        ctx->save_for_backward({o.s, w, o.rstd});
        ctx->saved_data["has_r"] = given(r);
        ctx->saved_data["N"] = rows.N;
        ctx->set_materialize_grads(false);
        return {o.s.view(x.sizes()), o.y};
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        once("add_rms_norm");
        auto saved = ctx->get_saved_variables();
        const Tensor &s = saved[0], &w = saved[1], &rstd = saved[2];
        const bool has_r = ctx->saved_data["has_r"].toBool();
        const int64_t N = ctx->saved_data["N"].toInt(), C = w.size(0);
        c10::DeviceGuard guard(s.device());
        Tensor extra = grads[0].defined() ? grads[0].contiguous() : Tensor();
        if (!grads[1].defined()) return {extra, has_r ? extra : Tensor(), Tensor(), Tensor()};
        Tensor dy = grads[1].contiguous();
        Tensor ds = at::empty_like(s), dw = at::empty_like(w);
        const int64_t nbytes = tgt_rms_norm_bwd_workspace_bytes(N, (int)C);
        Tensor ws = at::empty({nbytes}, s.options().dtype(at::kByte));
        check(tgt_rms_norm_bwd(s.data_ptr(), w.data_ptr(), rstd.data_ptr<float>(), dy.data_ptr(), extra.defined() ? extra.data_ptr() : nullptr, N, (int)C,
                               dtype_code(s), ds.data_ptr(), dw.data_ptr(), ws.data_ptr(), nbytes, stream_of(s)),
              "tgt_rms_norm_bwd");
        return {ds, has_r ? ds : Tensor(), dw, Tensor()};
    }
};
std::tuple<Tensor, Tensor> add_rms_norm(const Tensor& x, const Optional& r, const Tensor& weight, double eps) {
    const RowsOf rows(x, "add_rms_norm");
    check_norm(x, r, weight, rows, "add_rms_norm");
    Wanted want;
    want.look(x);
    want.look(weight);
    if (given(r)) want.look(*r);
    if (!want.node()) {
        c10::DeviceGuard guard(x.device());
        Normed o = norm_forward(x, r, weight.contiguous(), rows, eps, false);
        return {given(r) ? o.s : x, o.y};
    }
    auto o = AddRmsNorm::apply(x, r, weight, eps);
    return {o[0], o[1]};
}
std::tuple<Tensor, Tensor, Tensor> add_rms_norm_8bit(const Tensor& x, const Optional& r, const Tensor& weight, double eps) {
    const char* op = "add_rms_norm_8bit";
    const RowsOf rows(x, op);
    check_norm(x, r, weight, rows, op);
    no_gradients({&x, &weight}, op);
    if (given(r)) no_gradients({&*r}, op);
    c10::DeviceGuard guard(x.device());
    Tensor x2 = x.contiguous(), w = weight.contiguous(), r2 = given(r) ? r->contiguous() : Tensor();
    Tensor s = given(r) ? at::empty_like(x2, at::MemoryFormat::Contiguous) : x;
    Tensor codes = at::empty(x.sizes(), x.options().dtype(at::kFloat8_e4m3fn)), scales = at::empty(x.sizes().slice(0, x.dim() - 1), x.options().dtype(at::kFloat));
    check(tgt_add_rms_norm_8bit(x2.data_ptr(), given(r) ? r2.data_ptr() : nullptr, w.data_ptr(), rows.N, (int)rows.C, (float)eps, dtype_code(x),
                                given(r) ? s.data_ptr() : nullptr, codes.data_ptr(), scales.data_ptr<float>(), stream_of(x)),
          "tgt_add_rms_norm_8bit");
    return {s, codes, scales};
}
std::tuple<Tensor, Tensor> quantize_rows(const Tensor& w) {
    const char* op = "quantize_rows";
    const RowsOf rows(w, op);
    const int code = dtype_code(w);
    no_gradients({&w}, op);
    c10::DeviceGuard guard(w.device());
    Tensor w2 = w.contiguous();
    Tensor codes = at::empty(w.sizes(), w.options().dtype(at::kFloat8_e4m3fn)), scales = at::empty(w.sizes().slice(0, w.dim() - 1), w.options().dtype(at::kFloat));
    check(tgt_quantize_rows(w2.data_ptr(), rows.N, (int)rows.C, code, codes.data_ptr(), scales.data_ptr<float>(), stream_of(w)), "tgt_quantize_rows");
    return {codes, scales};
}

// ---- projections -----------------------------------------------------------------------------------------------------------------------
// A weight [F, C] and its bias [F] beside x [..., C]
void check_weight(const Tensor& w, const Tensor& x, int64_t F, int64_t C, const char* op, const char* name) {
    same_kind(w, x, op, name);
    TORCH_CHECK(w.dim() == 2 && w.size(0) == F && w.size(1) == C && F >= 1 && F <= (1 << 24), op, ": ", name, " must be [", F, ", ", C, "], at most 2^24 rows");
}
void check_bias(const Optional& b, const Tensor& x, at::ScalarType type, int64_t F, const char* op, const char* name) {
    if (!given(b)) return;
    same_gpu(*b, x, op, name);
    TORCH_CHECK(b->scalar_type() == type && b->dim() == 1 && b->size(0) == F, op, ": ", name, " must be ", type, " [", F, "]");
}
void check_residual(const Optional& r, const Tensor& x, at::ScalarType type, int64_t F, const char* op) {
    if (!given(r)) return;
    same_gpu(*r, x, op, "residual");
    TORCH_CHECK(r->scalar_type() == type && r->sizes() == at::IntArrayRef(with_last(x, F)), op, ": residual must be ", type, " of the result's shape");
}

Tensor room(int64_t bytes, const Tensor& x) { return bytes > 0 ? at::empty({bytes}, x.options().dtype(at::kByte)) : Tensor(); }
void* at_of(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

// kept: null, or where to put what the forward keeps for a backward
Tensor gated_forward(const Tensor& x, const Tensor& wg, const Tensor& wu, const Optional& bg, const Optional& bu, const RowsOf& rows, int64_t act, Tensor* kept) {
    const int64_t F = wg.size(0);
    Tensor h = at::empty(with_last(x, F), x.options());
    if (kept) *kept = room(tgt_gated_linear_kept_bytes(rows.N, (int)rows.C, (int)F, dtype_code(x), (int)act), x);
    const int64_t nbytes = tgt_gated_linear_fwd_workspace_bytes(rows.N, (int)rows.C, (int)F, dtype_code(x));
    const Tensor work = room(nbytes, x);
    check(tgt_gated_linear_fwd(x.data_ptr(), wg.data_ptr(), wu.data_ptr(), ptr(bg), ptr(bu), rows.N, (int)rows.C, (int)F, dtype_code(x), (int)act, h.data_ptr(),
                               kept ? at_of(*kept) : nullptr, at_of(work), nbytes, stream_of(x)),
          "tgt_gated_linear_fwd");
    return h;
}
struct GatedLinear : public torch::autograd::Function<GatedLinear> {
    static Tensor forward(AutogradContext* ctx, Tensor x, Tensor wg, Tensor wu, Optional bg, Optional bu, int64_t act) {
        const RowsOf rows(x, "gated_linear");
        c10::DeviceGuard guard(x.device());
        Tensor x2 = x.contiguous(), g2 = wg.contiguous(), u2 = wu.contiguous();
        Optional b1 = compact(bg), b2 = compact(bu);
        Tensor kept, h = gated_forward(x2, g2, u2, b1, b2, rows, act, &kept);
        ctx->save_for_backward({x2, g2, u2, given(b1) ? *b1 : Tensor(), given(b2) ? *b2 : Tensor(), kept});
        ctx->saved_data["act"] = act;
        ctx->saved_data["dx"] = x.requires_grad();
        ctx->saved_data["dw"] = wg.requires_grad() || wu.requires_grad();
        ctx->saved_data["db"] = (int64_t)((given(bg) && bg->requires_grad() ? 1 : 0) | (given(bu) && bu->requires_grad() ? 2 : 0));
        return h;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        once("gated_linear");
        auto saved = ctx->get_saved_variables();
        const Tensor &x = saved[0], &wg = saved[1], &wu = saved[2], &bg = saved[3], &bu = saved[4], &kept = saved[5];
        const int64_t F = wg.size(0), C = wg.size(1), N = x.numel() / C, act = ctx->saved_data["act"].toInt(), biases = ctx->saved_data["db"].toInt();
        c10::DeviceGuard guard(x.device());
        Tensor dh = grads[0].contiguous(), dx, dwg, dwu, dbg, dbu;
        if (ctx->saved_data["dx"].toBool()) dx = at::empty_like(x, at::MemoryFormat::Contiguous);
        if (ctx->saved_data["dw"].toBool()) { dwg = at::empty_like(wg); dwu = at::empty_like(wu); }
        if (biases & 1) dbg = at::empty({F}, x.options());
        if (biases & 2) dbu = at::empty({F}, x.options());
        void *dW[2] = {at_of(dwg), at_of(dwu)}, *db[2] = {at_of(dbg), at_of(dbu)};
        const int64_t nbytes = tgt_gated_linear_bwd_workspace_bytes(N, (int)C, (int)F, dtype_code(x));
        Tensor ws = at::empty({nbytes}, x.options().dtype(at::kByte));
        check(tgt_gated_linear_bwd(x.data_ptr(), wg.data_ptr(), wu.data_ptr(), at_of(bg), at_of(bu), dh.data_ptr(), N, (int)C, (int)F, dtype_code(x), (int)act,
                                   at_of(kept), at_of(dx), dW, db, ws.data_ptr(), nbytes, stream_of(x)),
              "tgt_gated_linear_bwd");
        return {dx, dwg, dwu, dbg, dbu, Tensor()};
    }
};
Tensor gated_linear(const Tensor& x, const Tensor& wg, const Tensor& wu, const Optional& bg, const Optional& bu, int64_t act) {
    const char* op = "gated_linear";
    const RowsOf rows(x, op);
    (void)dtype_code(x);
    TORCH_CHECK(wg.dim() == 2, op, ": gate_weight must be [out, in]");
    const int64_t F = wg.size(0);
    check_weight(wg, x, F, rows.C, op, "gate_weight");
    check_weight(wu, x, F, rows.C, op, "up_weight");
    check_bias(bg, x, x.scalar_type(), F, op, "gate_bias");
    check_bias(bu, x, x.scalar_type(), F, op, "up_bias");
    Wanted want;
    want.look(x); want.look(wg); want.look(wu);
    if (given(bg)) want.look(*bg);
    if (given(bu)) want.look(*bu);
    if (want.node()) return GatedLinear::apply(x, wg, wu, bg, bu, act);
    c10::DeviceGuard guard(x.device());
    return gated_forward(x.contiguous(), wg.contiguous(), wu.contiguous(), compact(bg), compact(bu), rows, act, nullptr);
}

Tensor linear_act_forward(const Tensor& x, const Tensor& w, const Optional& b, const Optional& r, const RowsOf& rows, int64_t act, Tensor* kept) {
    const int64_t F = w.size(0);
    Tensor y = at::empty(with_last(x, F), x.options());
    if (kept) *kept = room(tgt_linear_epilogue_kept_bytes(rows.N, (int)rows.C, (int)F, dtype_code(x), (int)act), x);
    const int64_t nbytes = tgt_linear_epilogue_fwd_workspace_bytes(rows.N, (int)rows.C, (int)F, dtype_code(x));
    const Tensor work = room(nbytes, x);
    check(tgt_linear_epilogue_fwd(x.data_ptr(), w.data_ptr(), ptr(b), ptr(r), rows.N, (int)rows.C, (int)F, dtype_code(x), (int)act, y.data_ptr(),
                                  kept ? at_of(*kept) : nullptr, at_of(work), nbytes, stream_of(x)),
          "tgt_linear_epilogue_fwd");
    return y;
}
struct LinearAct : public torch::autograd::Function<LinearAct> {
    static Tensor forward(AutogradContext* ctx, Tensor x, Tensor w, Optional b, Optional r, int64_t act) {
        const RowsOf rows(x, "linear_act");
        c10::DeviceGuard guard(x.device());
        Tensor x2 = x.contiguous(), w2 = w.contiguous();
        Optional b2 = compact(b);
        Tensor kept, y = linear_act_forward(x2, w2, b2, compact(r), rows, act, &kept);
        ctx->save_for_backward({x2, w2, given(b2) ? *b2 : Tensor(), kept});
        ctx->saved_data["act"] = act;
        ctx->saved_data["dx"] = x.requires_grad();
        ctx->saved_data["dw"] = w.requires_grad();
        ctx->saved_data["db"] = given(b) && b->requires_grad();
        ctx->saved_data["dr"] = given(r) && r->requires_grad();
        return y;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        once("linear_act");
        auto saved = ctx->get_saved_variables();
        const Tensor &x = saved[0], &w = saved[1], &b = saved[2], &kept = saved[3];
        const int64_t F = w.size(0), C = w.size(1), N = x.numel() / C, act = ctx->saved_data["act"].toInt();
        c10::DeviceGuard guard(x.device());
        Tensor dx, dw, db;
        const bool want_x = ctx->saved_data["dx"].toBool(), want_w = ctx->saved_data["dw"].toBool(), want_b = ctx->saved_data["db"].toBool();
        if (want_x || want_w || want_b) {
            Tensor dy = grads[0].contiguous();
            if (want_x) dx = at::empty_like(x, at::MemoryFormat::Contiguous);
            if (want_w) dw = at::empty_like(w);
            if (want_b) db = at::empty({F}, x.options());
            const int64_t nbytes = tgt_linear_epilogue_bwd_workspace_bytes(N, (int)C, (int)F, dtype_code(x), (int)act);
            Tensor ws = at::empty({nbytes}, x.options().dtype(at::kByte));
            check(tgt_linear_epilogue_bwd(x.data_ptr(), w.data_ptr(), at_of(b), dy.data_ptr(), N, (int)C, (int)F, dtype_code(x), (int)act, at_of(kept), at_of(dx), at_of(dw),
                                          at_of(db), ws.data_ptr(), nbytes, stream_of(x)),
                  "tgt_linear_epilogue_bwd");
        }
        return {dx, dw, db, ctx->saved_data["dr"].toBool() ? grads[0] : Tensor(), Tensor()};
    }
};
Tensor linear_act(const Tensor& x, const Tensor& w, const Optional& b, const Optional& r, int64_t act) {
    const char* op = "linear_act";
    const RowsOf rows(x, op);
    (void)dtype_code(x);
    TORCH_CHECK(w.dim() == 2, op, ": weight must be [out, in]");
    const int64_t F = w.size(0);
    check_weight(w, x, F, rows.C, op, "weight");
    check_bias(b, x, x.scalar_type(), F, op, "bias");
    check_residual(r, x, x.scalar_type(), F, op);
    Wanted want;
    want.look(x); want.look(w);
    if (given(b)) want.look(*b);
    if (given(r)) want.look(*r);
    if (want.node()) return LinearAct::apply(x, w, b, r, act);
    c10::DeviceGuard guard(x.device());
    return linear_act_forward(x.contiguous(), w.contiguous(), compact(b), compact(r), rows, act, nullptr);
}

// ---- operands in 8 bits --------------------------------------------------------------------------------------------------------------------
void check_codes(const Tensor& codes, const Tensor& scales, const Tensor& x, const char* op, const char* name) {
    same_gpu(codes, x, op, name);
    same_gpu(scales, x, op, "scales");
    TORCH_CHECK(codes.scalar_type() == at::kFloat8_e4m3fn, op, ": ", name, " must be float8_e4m3fn, got ", codes.scalar_type());
    TORCH_CHECK(scales.scalar_type() == at::kFloat && scales.sizes() == codes.sizes().slice(0, codes.dim() - 1), op, ": the scales of ", name,
                " must be float32, one per row");
}
int result_code(at::ScalarType t, const char* op) {
    TORCH_CHECK(t == at::kFloat || t == at::kBFloat16, op, ": results are float32 or bfloat16, got ", t);
    return t == at::kFloat ? TGT_DTYPE_F32 : TGT_DTYPE_BF16;
}
Tensor gated_linear_8bit(const Tensor& x, const Tensor& xs, const Tensor& wg, const Tensor& gs, const Tensor& wu, const Tensor& us, const Optional& bg,
                         const Optional& bu, int64_t act, at::ScalarType type) {
    const char* op = "gated_linear_8bit";
    const RowsOf rows(x, op);
    const int code = result_code(type, op);
    TORCH_CHECK(wg.dim() == 2, op, ": gate_weight must be [out, in]");
    const int64_t F = wg.size(0);
    check_codes(x, xs, x, op, "x");
    check_codes(wg, gs, x, op, "gate_weight");
    check_codes(wu, us, x, op, "up_weight");
    check_weight(wg, x, F, rows.C, op, "gate_weight");
    check_weight(wu, x, F, rows.C, op, "up_weight");
    check_bias(bg, x, type, F, op, "gate_bias");
    check_bias(bu, x, type, F, op, "up_bias");
    no_gradients({&x, &xs, &wg, &gs, &wu, &us}, op);
    if (given(bg)) no_gradients({&*bg}, op);
    if (given(bu)) no_gradients({&*bu}, op);
    c10::DeviceGuard guard(x.device());
    Tensor x2 = x.contiguous(), xs2 = xs.contiguous(), g2 = wg.contiguous(), gs2 = gs.contiguous(), u2 = wu.contiguous(), us2 = us.contiguous();
    Optional b1 = compact(bg), b2 = compact(bu);
    Tensor h = at::empty(with_last(x, F), x.options().dtype(type));
    const int64_t nbytes = tgt_gated_linear_8bit_workspace_bytes(rows.N, (int)rows.C, (int)F);
    const Tensor work = room(nbytes, x);
    check(tgt_gated_linear_8bit_fwd(x2.data_ptr(), xs2.data_ptr<float>(), g2.data_ptr(), gs2.data_ptr<float>(), u2.data_ptr(), us2.data_ptr<float>(), ptr(b1), ptr(b2),
                                    rows.N, (int)rows.C, (int)F, code, (int)act, h.data_ptr(), at_of(work), nbytes, stream_of(x)),
          "tgt_gated_linear_8bit_fwd");
    return h;
}
Tensor linear_act_8bit(const Tensor& x, const Tensor& xs, const Tensor& w, const Tensor& ws, const Optional& b, const Optional& r, int64_t act, at::ScalarType type) {
    const char* op = "linear_act_8bit";
    const RowsOf rows(x, op);
    const int code = result_code(type, op);
    TORCH_CHECK(w.dim() == 2, op, ": weight must be [out, in]");
    const int64_t F = w.size(0);
    check_codes(x, xs, x, op, "x");
    check_codes(w, ws, x, op, "weight");
    check_weight(w, x, F, rows.C, op, "weight");
    check_bias(b, x, type, F, op, "bias");
    check_residual(r, x, type, F, op);
    no_gradients({&x, &xs, &w, &ws}, op);
    if (given(b)) no_gradients({&*b}, op);
    if (given(r)) no_gradients({&*r}, op);
    c10::DeviceGuard guard(x.device());
    Tensor x2 = x.contiguous(), xs2 = xs.contiguous(), w2 = w.contiguous(), ws2 = ws.contiguous();
    Optional b2 = compact(b), r2 = compact(r);
    Tensor y = at::empty(with_last(x, F), x.options().dtype(type));
    const int64_t nbytes = tgt_linear_epilogue_8bit_workspace_bytes(rows.N, (int)rows.C, (int)F);
    const Tensor work = room(nbytes, x);
    check(tgt_linear_epilogue_8bit_fwd(x2.data_ptr(), xs2.data_ptr<float>(), w2.data_ptr(), ws2.data_ptr<float>(), ptr(b2), ptr(r2), rows.N, (int)rows.C, (int)F, code,
                                       (int)act, y.data_ptr(), at_of(work), nbytes, stream_of(x)),
          "tgt_linear_epilogue_8bit_fwd");
    return y;
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(torchgt, m) {
    m.def("add_rms_norm(Tensor x, Tensor? residual, Tensor weight, float eps) -> (Tensor, Tensor)");
    m.def("add_rms_norm_8bit(Tensor x, Tensor? residual, Tensor weight, float eps) -> (Tensor, Tensor, Tensor)");
    m.def("quantize_rows(Tensor w) -> (Tensor, Tensor)");
    m.def("gated_linear(Tensor x, Tensor gate_weight, Tensor up_weight, Tensor? gate_bias, Tensor? up_bias, int act) -> Tensor");
    m.def("gated_linear_8bit(Tensor x, Tensor x_scales, Tensor gate_weight, Tensor gate_scales, Tensor up_weight, Tensor up_scales, Tensor? gate_bias, "
          "Tensor? up_bias, int act, ScalarType dtype) -> Tensor");
    m.def("linear_act(Tensor x, Tensor weight, Tensor? bias, Tensor? residual, int act) -> Tensor");
    m.def("linear_act_8bit(Tensor x, Tensor x_scales, Tensor weight, Tensor weight_scales, Tensor? bias, Tensor? residual, int act, ScalarType dtype) -> Tensor");
}
TORCH_LIBRARY_IMPL(torchgt, CompositeImplicitAutograd, m) {
    m.impl("add_rms_norm", add_rms_norm);
    m.impl("add_rms_norm_8bit", add_rms_norm_8bit);
    m.impl("quantize_rows", quantize_rows);
    m.impl("gated_linear", gated_linear);
    m.impl("gated_linear_8bit", gated_linear_8bit);
    m.impl("linear_act", linear_act);
    m.impl("linear_act_8bit", linear_act_8bit);
}
