// Host side of the operators around wide layers (dwo_gated.hip, dwo_head.hip, dwo_check8.hip): argument checks, allocation, and their
// nodes of autograd.  Included by dwo_host.cpp, inside its namespace.
//
// Parameters of another type than the activations are converted on the way in and get gradients of their own type, from the fp32 sums.
// Gradients of gradients are refused: what the passes hold (8 bits, fp32 halves of the hidden tensor) has no history.
#pragma once

using Context = torch::autograd::AutogradContext;
using List = torch::autograd::variable_list;

// x [.., C] as rows
struct Rows {
    int64_t rows, C;
    explicit Rows(const Tensor &x, const char *name) {
        check_glue(x, name);
        if (x.dim() < 1 || x.size(-1) < 1) fail(std::string(name) + " must have a last dimension of at least one channel");
        C = x.size(-1), rows = x.numel() / C;
    }
};
std::vector<int64_t> with_last(const Tensor &x, int64_t n) {
    std::vector<int64_t> s = x.sizes().vec();
    s.back() = n;
    return s;
}
void check_weight(const Tensor &x, const Tensor &w, int64_t rows, int64_t cols, const char *name) {
    check_glue(w, name);
    check_pair(x, w);
    if (w.dim() != 2 || w.size(1) != cols || (rows >= 0 && w.size(0) != rows) || w.size(0) < 1)
        fail(std::string(name) + " must be [" + (rows >= 0 ? std::to_string(rows) : "N") + ", " + std::to_string(cols) + "]");
}
void check_bias(const Tensor &x, const OptTensor &b, int64_t n, const char *name) {
    if (!b.has_value()) return;
    check_glue(*b, name);
    check_pair(x, *b);
    if (b->dim() != 1 || b->size(0) != n) fail(std::string(name) + " must be [" + std::to_string(n) + "]");
}
// a parameter as the kernels take it
Tensor like(const Tensor &x, const Tensor &p) { return dense(p.scalar_type() == x.scalar_type() ? p : p.detach().to(x.scalar_type())); }
Tensor like(const Tensor &x, const OptTensor &p) { return p.has_value() ? like(x, *p) : Tensor(); }
const void *dptr(const Tensor &t) { return t.defined() ? t.const_data_ptr() : nullptr; }
void *mptr(const Tensor &t) { return t.defined() ? t.mutable_data_ptr() : nullptr; }
bool trains(const Tensor &t) { return t.requires_grad(); }
bool trains(const OptTensor &t) { return t.has_value() && t->requires_grad(); }
// What a backward pass refuses before it launches anything.  Under stream capture: a leaf of an eager graph that still lives has its node
// on that graph's stream; the engine would wait for it there, drawing a stream that is not captured into the capture, whose end
// then ends the process.
void backward_allowed(const Place &at) {
    if (at::GradMode::is_enabled()) fail("gradients of this operator's gradients are not available (create_graph=True)");
    hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
    if (hipStreamIsCapturing((hipStream_t)at.stream, &status) != hipSuccess || status == hipStreamCaptureStatusNone) return;
    const auto current = c10::hip::getCurrentHIPStream();
    std::vector<torch::autograd::Node *> todo{torch::autograd::get_current_node().get()};
    std::unordered_set<torch::autograd::Node *> seen;
    while (!todo.empty()) {
        torch::autograd::Node *node = todo.back();
        todo.pop_back();
        if (node == nullptr || !seen.insert(node).second) continue;
        for (const auto &edge : node->next_edges()) todo.push_back(edge.function.get());
        const auto stream = node->next_edges().empty() ? node->stream() : std::nullopt;
        if (stream.has_value() && stream->device_index() == current.device_index() && stream->id() != current.id())
            fail("this backward pass cannot be captured: an eager graph of the same leaves lives, on another stream (delete its results "
                 "before the capture)");
    }
}
Tensor as_type(const Tensor &t, at::ScalarType type) { return !t.defined() || t.scalar_type() == type ? t : t.to(type); }

// ------------------------------------------------------------------------------------------------- 8-bit checkpoints
// (codes and exponents or nothing, act(x) or nothing)
std::tuple<Tensor, Tensor, Tensor> pack8(const Tensor &x_, int64_t act, bool with_codes, bool with_value) {
    const Rows r(x_, "x");
    const Place at(x_);
    const Tensor x = dense(x_);
    Tensor codes, exps;
    if (with_codes) {
        codes = at::empty(x.sizes(), x.options().dtype(at::kChar));
        exps = at::empty(with_last(x, up(r.C, 32)), x.options().dtype(at::kByte));
    }
    Tensor y = with_value ? at::empty(x.sizes(), x.options()) : Tensor();
    if (r.rows > 0)
        check(lib.pack8(ptr(x), mptr(y), mptr(codes), mptr(exps), (size_t)r.rows, as_int(r.C), (int)act, dtype_code(x), at.stream),
              "dwo_pack8");
    return {codes, exps, y};
}
// the values held in `type`, or dy times the activation's slope there
Tensor unpack8(const Tensor &codes_, const Tensor &exps_, const OptTensor &dy_, int64_t act, at::ScalarType type) {
    if (!codes_.is_cuda() || codes_.scalar_type() != at::kChar || codes_.dim() < 1 || codes_.size(-1) < 1)
        fail("codes must be a CUDA tensor of type int8 with a last dimension of at least one channel");
    const int64_t C = codes_.size(-1), rows = codes_.numel() / C;
    check_pair(codes_, exps_);
    if (exps_.scalar_type() != at::kByte || exps_.sizes() != at::IntArrayRef(with_last(codes_, up(C, 32))))
        fail("exponents must be uint8, one for every 32 values of a row");
    if (dtype_code(type) < 0) fail("values are held for float32, bfloat16 or float16");
    if (dy_.has_value() && (dy_->scalar_type() != type || dy_->sizes() != codes_.sizes() || dy_->device() != codes_.device()))
        fail("dy must match what is held");
    const Place at(codes_);
    const Tensor codes = dense(codes_), exps = dense(exps_);
    const Tensor dy = dy_.has_value() ? dense(*dy_) : Tensor();
    Tensor out = at::empty(codes.sizes(), codes.options().dtype(type));
    if (rows > 0)
        check(lib.unpack8(ptr(codes), ptr(exps), dptr(dy), out.data_ptr(), (size_t)rows, as_int(C), (int)act, dtype_code(type), at.stream),
              "dwo_unpack8");
    return out;
}

struct Act8 : torch::autograd::Function<Act8> {
    static Tensor forward(Context *ctx, const Tensor &x, int64_t act) {
        ctx->set_materialize_grads(false);
        auto [codes, exps, y] = pack8(x, act, true, true);
        ctx->save_for_backward({codes, exps});
        ctx->saved_data["act"] = act, ctx->saved_data["type"] = (int64_t)x.scalar_type();
        return y;
    }
    static List backward(Context *ctx, const List &grads) {
        if (!grads[0].defined()) return {Tensor(), Tensor()};
        const List s = ctx->get_saved_variables();
        backward_allowed(Place(s[0]));
        const auto type = (at::ScalarType)ctx->saved_data["type"].toInt();
        return {unpack8(s[0], s[1], as_type(grads[0], type), ctx->saved_data["act"].toInt(), type), Tensor()};
    }
};
Tensor act8(const Tensor &x, int64_t act) {
    py::gil_scoped_release nogil;
    if (at::GradMode::is_enabled() && trains(x)) return Act8::apply(x, act);
    return std::get<2>(pack8(x, act, false, true));
}
std::tuple<Tensor, Tensor> pack8_entry(const Tensor &x) {
    py::gil_scoped_release nogil;
    auto [codes, exps, none] = pack8(x.detach(), 0, true, false);
    return {codes, exps};
}
Tensor unpack8_entry(const Tensor &codes, const Tensor &exps, at::ScalarType type) {
    py::gil_scoped_release nogil;
    return unpack8(codes, exps, std::nullopt, 0, type);
}

// y = x w^T + b (codes, exps: x's checkpoint, or undefined)
Tensor layer8(const Tensor &x, const Tensor &w, const Tensor &b, const Tensor &codes, const Tensor &exps) {
    const Place at(x);
    const int64_t C = x.size(-1), rows = x.numel() / C, D = w.size(0);
    Tensor y = at::empty(with_last(x, D), x.options());
    if (rows == 0) return y;
    const int dt = dtype_code(x);
    const size_t need = lib.layer8_workspace_bytes((size_t)rows, as_int(C), as_int(D), 0, dt);
    const Tensor ws = bytes(x, need);
    check(lib.layer8(ptr(x), ptr(w), dptr(b), y.data_ptr(), mptr(codes), mptr(exps), ws.data_ptr(), need, (size_t)rows, as_int(C), as_int(D),
                     dt, at.stream),
          "dwo_layer8");
    return y;
}
struct Linear8 : torch::autograd::Function<Linear8> {
    static Tensor forward(Context *ctx, const Tensor &x_, const Tensor &w_, const OptTensor &b_) {
        ctx->set_materialize_grads(false);
        const Place at(x_);
        const Tensor x = dense(x_), w = like(x, w_), b = like(x, b_);
        Tensor codes, exps;
        if (trains(w_) || trains(b_)) {
            codes = at::empty(x.sizes(), x.options().dtype(at::kChar));
            exps = at::empty(with_last(x, up(x.size(-1), 32)), x.options().dtype(at::kByte));
        }
        ctx->save_for_backward({codes, exps, w});
        ctx->saved_data["p"] = std::vector<int64_t>{(int64_t)x.scalar_type(), (int64_t)w_.scalar_type(),
                                                    b_.has_value() ? (int64_t)b_->scalar_type() : -1};
        return layer8(x, w, b, codes, exps);
    }
    static List backward(Context *ctx, const List &grads) {
        List out(3);
        if (!grads[0].defined()) return out;
        const List s = ctx->get_saved_variables();
        const Tensor &codes = s[0], &exps = s[1], &w = s[2];
        const std::vector<int64_t> p = ctx->saved_data["p"].toIntVector();
        const auto type = (at::ScalarType)p[0], w_type = (at::ScalarType)p[1];
        const bool need_db = p[2] >= 0 && ctx->needs_input_grad(2), need_dw = ctx->needs_input_grad(1) || need_db;
        const Place at(w);
        backward_allowed(at);
        const Tensor dy = dense(as_type(grads[0], type));
        const int64_t D = w.size(0), C = w.size(1), rows = dy.numel() / D;
        const auto grad = w.options().dtype(w_type);
        Tensor dx, dw, db;
        if (ctx->needs_input_grad(0)) dx = at::empty(with_last(dy, C), dy.options());
        if (need_dw) dw = rows > 0 ? at::empty({D, C}, grad) : at::zeros({D, C}, grad);
        if (need_db) db = rows > 0 ? at::empty({D}, grad) : at::zeros({D}, grad);
        if (rows > 0 && (dx.defined() || need_dw)) {
            const int dt = dtype_code(dy);
            const size_t need = lib.layer8_workspace_bytes((size_t)rows, as_int(C), as_int(D), 1, dt);
            const Tensor ws = bytes(dy, need);
            // (without the weights' gradients nothing is read of the checkpoint)
            check(lib.layer8_backward(ptr(dy), codes.defined() ? ptr(codes) : ws.data_ptr(), exps.defined() ? ptr(exps) : ws.data_ptr(),
                                      ptr(w), mptr(dx), mptr(dw), mptr(db), ws.data_ptr(), need, (size_t)rows, as_int(C), as_int(D), dt,
                                      dtype_code(w_type), at.stream),
                  "dwo_layer8_backward");
        }
        out[0] = dx;
        if (ctx->needs_input_grad(1)) out[1] = dw;
        if (need_db) out[2] = as_type(db, (at::ScalarType)p[2]);
        return out;
    }
};
Tensor linear8(const Tensor &x, const Tensor &w, const OptTensor &b) {
    const Rows r(x, "x");
    check_weight(x, w, -1, r.C, "weight");
    check_bias(x, b, w.size(0), "bias");
    py::gil_scoped_release nogil;
    if (!at::GradMode::is_enabled()) {
        const Place at(x);
        const Tensor d = dense(x);
        return layer8(d, like(d, w), like(d, b), Tensor(), Tensor());
    }
    return Linear8::apply(x, w, b);
}

// ------------------------------------------------------------------------------------------------- gated feed-forward block
int64_t up8(int64_t n) { return up(n, 8) * 8; }
Tensor gated_forward(const Tensor &x, const Tensor &w_in, const Tensor &b_in, const Tensor &w_out, const Tensor &b_out, const Tensor &keep,
                     int64_t act) {
    const int64_t C = x.size(-1), rows = x.numel() / C, D = w_out.size(0), H = w_out.size(1);
    Tensor y = at::empty(with_last(x, D), x.options());
    if (rows == 0) return y;
    const Place at(x);
    const int dt = dtype_code(x);
    const size_t need = lib.gated_workspace_bytes((size_t)rows, as_int(C), as_int(H), as_int(D), 0, 0, dt);
    const Tensor ws = bytes(x, need);
    check(lib.gated_forward(ptr(x), ptr(w_in), dptr(b_in), ptr(w_out), dptr(b_out), y.data_ptr(), (float *)mptr(keep), ws.data_ptr(), need,
                            (size_t)rows, as_int(C), as_int(H), as_int(D), (int)act, dt, at.stream),
          "dwo_gated_forward");
    return y;
}
struct Gated : torch::autograd::Function<Gated> {
    static Tensor forward(Context *ctx, const Tensor &x_, const Tensor &w_in_, const OptTensor &b_in_, const Tensor &w_out_,
                          const OptTensor &b_out_, int64_t act, bool held8) {
        ctx->set_materialize_grads(false);
        const Place at(x_);
        const Tensor x = dense(x_), w_in = like(x, w_in_), b_in = like(x, b_in_), w_out = like(x, w_out_), b_out = like(x, b_out_);
        const int64_t rows = x.numel() / x.size(-1), H = w_out.size(1);
        Tensor held = x, exps, keep;
        if (held8) {
            auto [codes, e, none] = pack8(x, 0, true, false);
            held = codes, exps = e;
        } else {
            keep = at::empty({2, rows, up8(H)}, x.options().dtype(at::kFloat));
            if (!trains(w_in_) && !trains(b_in_)) held = Tensor();
        }
        ctx->save_for_backward({held, exps, keep, w_in, held8 ? b_in : Tensor(), w_out});
        auto type = [](const OptTensor &t) { return t.has_value() ? (int64_t)t->scalar_type() : -1; };
        ctx->saved_data["p"] = std::vector<int64_t>{act, (int64_t)x.scalar_type(), (int64_t)w_in_.scalar_type(), type(b_in_),
                                                    (int64_t)w_out_.scalar_type(), type(b_out_)};
        return gated_forward(x, w_in, b_in, w_out, b_out, keep, act);
    }
    static List backward(Context *ctx, const List &grads) {
        List out(7);
        if (!grads[0].defined()) return out;
        const List s = ctx->get_saved_variables();
        const Tensor &held = s[0], &exps = s[1], &keep = s[2], &w_in = s[3], &b_in = s[4], &w_out = s[5];
        const std::vector<int64_t> p = ctx->saved_data["p"].toIntVector();
        const auto type = (at::ScalarType)p[1], in_type = (at::ScalarType)p[2], out_type = (at::ScalarType)p[4];
        // (places of the inputs that are there)
        size_t k = 0;
        const bool need_x = ctx->needs_input_grad(k++), need_wi = ctx->needs_input_grad(k++),
                   need_bi = p[3] >= 0 && ctx->needs_input_grad(k++), need_wo = ctx->needs_input_grad(k++),
                   need_bo = p[5] >= 0 && ctx->needs_input_grad(k++);
        const bool held8 = exps.defined();
        const Place at(w_in);
        backward_allowed(at);
        const Tensor dy = dense(as_type(grads[0], type));
        const int64_t D = w_out.size(0), H = w_out.size(1), C = w_in.size(1), rows = dy.numel() / D;
        // (both weights' gradients are written as one type)
        const at::ScalarType grad_type = in_type == out_type ? in_type : at::kFloat;
        const auto grad = w_in.options().dtype(grad_type);
        auto room = [&](bool need, at::IntArrayRef shape) {
            return !need ? Tensor() : rows > 0 ? at::empty(shape, grad) : at::zeros(shape, grad);
        };
        Tensor dx = need_x ? at::empty(with_last(dy, C), dy.options()) : Tensor();
        const Tensor dwi = room(need_wi || need_bi, {2 * H, C}), dbi = room(need_bi, {2 * H}), dwo = room(need_wo || need_bo, {D, H}),
                     dbo = room(need_bo, {D});
        if (rows > 0) {
            const int dt = dtype_code(dy);
            const size_t need = lib.gated_workspace_bytes((size_t)rows, as_int(C), as_int(H), as_int(D), 1, held8, dt);
            const Tensor ws = bytes(dy, need);
            // (x is read for w_in's gradient alone)
            const void *x = held.defined() ? ptr(held) : ws.data_ptr();
            check(lib.gated_backward(ptr(dy), held8 ? nullptr : x, held8 ? x : nullptr, held8 ? ptr(exps) : nullptr,
                                     held8 ? nullptr : (const float *)ptr(keep), ptr(w_in), dptr(b_in), ptr(w_out), mptr(dx), mptr(dwi),
                                     mptr(dbi), mptr(dwo), mptr(dbo), ws.data_ptr(), need, (size_t)rows, as_int(C), as_int(H), as_int(D),
                                     (int)p[0], dt, dtype_code(grad_type), at.stream),
                  "dwo_gated_backward");
        }
        out[0] = dx;
        if (need_wi) out[1] = as_type(dwi, in_type);
        if (need_bi) out[2] = as_type(dbi, (at::ScalarType)p[3]);
        if (need_wo) out[3] = as_type(dwo, out_type);
        if (need_bo) out[4] = as_type(dbo, (at::ScalarType)p[5]);
        return out;
    }
};
Tensor gated(const Tensor &x, const Tensor &w_in, const OptTensor &b_in, const Tensor &w_out, const OptTensor &b_out, int64_t act,
             bool held8) {
    const Rows r(x, "x");
    check_glue(w_out, "w_out");
    if (w_out.dim() != 2 || w_out.size(1) < 1) fail("w_out must be [D, H]");
    check_weight(x, w_in, 2 * w_out.size(1), r.C, "w_in");
    check_weight(x, w_out, -1, w_out.size(1), "w_out");
    check_bias(x, b_in, w_in.size(0), "b_in");
    check_bias(x, b_out, w_out.size(0), "b_out");
    py::gil_scoped_release nogil;
    if (at::GradMode::is_enabled() && (trains(x) || trains(w_in) || trains(b_in) || trains(w_out) || trains(b_out)))
        return Gated::apply(x, w_in, b_in, w_out, b_out, act, held8);
    const Place at(x);
    const Tensor d = dense(x);
    return gated_forward(d, like(d, w_in), like(d, b_in), like(d, w_out), like(d, b_out), Tensor(), act);
}

// ------------------------------------------------------------------------------------------------- cross entropy of many classes
// (loss, lse, number of rows that count or undefined)
std::tuple<Tensor, Tensor, Tensor> head_forward(const Tensor &x, const Tensor &w, const Tensor &b, const Tensor &target, bool mean,
                                                int64_t ignore, double smoothing) {
    const Place at(x);
    const int64_t C = x.size(-1), rows = x.numel() / C, V = w.size(0);
    const auto f32 = x.options().dtype(at::kFloat);
    Tensor loss = mean ? at::empty({}, f32) : at::empty(target.sizes(), f32);
    Tensor lse = at::empty({rows}, f32), count = mean ? at::empty({}, f32) : Tensor();
    if (rows == 0) {
        if (mean) loss.fill_(NAN), count.zero_();
        return {loss, lse, count};
    }
    const int dt = dtype_code(x);
    const size_t need = lib.head_workspace_bytes((size_t)rows, as_int(C), as_int(V), 0, dt);
    const Tensor ws = bytes(x, need);
    check(lib.head_forward(ptr(x), ptr(w), dptr(b), ptr(target), ignore, (float)smoothing, (float *)lse.data_ptr(), (float *)loss.data_ptr(),
                           (float *)mptr(count), ws.data_ptr(), need, (size_t)rows, as_int(C), as_int(V), dt, at.stream),
          "dwo_head_forward");
    return {loss, lse, count};
}
struct Head : torch::autograd::Function<Head> {
    static Tensor forward(Context *ctx, const Tensor &x_, const Tensor &w_, const OptTensor &b_, const Tensor &target_, bool mean,
                          int64_t ignore, double smoothing) {
        ctx->set_materialize_grads(false);
        const Place at(x_);
        const Tensor x = dense(x_), w = like(x, w_), b = like(x, b_), target = target_.contiguous();
        auto [loss, lse, count] = head_forward(x, w, b, target, mean, ignore, smoothing);
        ctx->save_for_backward({x, w, b, target, lse, count});
        ctx->saved_data["p"] = std::vector<int64_t>{ignore, (int64_t)w_.scalar_type(), b_.has_value() ? (int64_t)b_->scalar_type() : -1};
        ctx->saved_data["s"] = smoothing;
        return loss;
    }
    static List backward(Context *ctx, const List &grads) {
        List out(7);
        if (!grads[0].defined()) return out;
        const List s = ctx->get_saved_variables();
        const Tensor &x = s[0], &w = s[1], &b = s[2], &target = s[3], &lse = s[4], &count = s[5];
        const std::vector<int64_t> p = ctx->saved_data["p"].toIntVector();
        const auto w_type = (at::ScalarType)p[1];
        const bool need_db = p[2] >= 0 && ctx->needs_input_grad(2), need_dw = ctx->needs_input_grad(1) || need_db;
        const Place at(x);
        backward_allowed(at);
        const Tensor up = dense(as_type(grads[0], at::kFloat));
        const int64_t V = w.size(0), C = w.size(1), rows = x.numel() / C;
        const auto grad = w.options().dtype(w_type);
        Tensor dx, dw, db;
        if (ctx->needs_input_grad(0)) dx = at::empty(x.sizes(), x.options());
        if (need_dw) dw = rows > 0 ? at::empty({V, C}, grad) : at::zeros({V, C}, grad);
        if (need_db) db = rows > 0 ? at::empty({V}, grad) : at::zeros({V}, grad);
        if (rows > 0) {
            const int dt = dtype_code(x);
            const size_t need = lib.head_workspace_bytes((size_t)rows, as_int(C), as_int(V), 1, dt);
            const Tensor ws = bytes(x, need);
            check(lib.head_backward((const float *)ptr(up), ptr(x), ptr(w), dptr(b), ptr(target), p[0],
                                    (float)ctx->saved_data["s"].toDouble(), (const float *)ptr(lse), (const float *)dptr(count), mptr(dx),
                                    mptr(dw), mptr(db), ws.data_ptr(), need, (size_t)rows, as_int(C), as_int(V), dt, dtype_code(w_type),
                                    at.stream),
                  "dwo_head_backward");
        }
        out[0] = dx;
        if (ctx->needs_input_grad(1)) out[1] = dw;
        if (need_db) out[2] = as_type(db, (at::ScalarType)p[2]);
        return out;
    }
};
Tensor head(const Tensor &x, const Tensor &w, const OptTensor &b, const Tensor &target, bool mean, int64_t ignore, double smoothing) {
    const Rows r(x, "x");
    check_weight(x, w, -1, r.C, "weight");
    check_bias(x, b, w.size(0), "bias");
    check_pair(x, target);
    if (target.scalar_type() != at::kLong || target.sizes() != x.sizes().slice(0, x.dim() - 1))
        fail("target must be int64, one class for every row of x");
    if (!(smoothing >= 0.0 && smoothing <= 1.0)) fail("label_smoothing must be between 0 and 1");
    py::gil_scoped_release nogil;
    if (at::GradMode::is_enabled() && (trains(x) || trains(w) || trains(b)))
        return Head::apply(x, w, b, target, mean, ignore, smoothing);
    const Place at(x);
    const Tensor d = dense(x);
    return std::get<0>(head_forward(d, like(d, w), like(d, b), target.contiguous(), mean, ignore, smoothing));
}
