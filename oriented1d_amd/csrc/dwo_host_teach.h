// Host side of the operators between a teacher and its student (dwo_int8.hip, dwo_top.hip, dwo_distill.hip): argument checks, allocation, and the
// loss's node of autograd.  Included by dwo_host.cpp, inside its namespace, behind dwo_host_wide.h.
#pragma once

std::vector<int64_t> without_last(const Tensor &x) { return x.sizes().slice(0, x.dim() - 1).vec(); }
int64_t up16(int64_t n) { return up(n, 16) * 16; }

// ------------------------------------------------------------------------------------------------- 8-bit integers
std::tuple<Tensor, Tensor> int8_rows(const Tensor &x_) {
    const Rows r(x_, "x");
    py::gil_scoped_release nogil;
    const Place at(x_);
    const Tensor x = dense(x_.detach());
    Tensor codes = at::empty(with_last(x, up16(r.C)), x.options().dtype(at::kChar)), steps = at::empty(without_last(x), x.options().dtype(at::kFloat));
    if (r.rows > 0)
        check(lib.int8_rows(ptr(x), codes.data_ptr(), (float *)steps.data_ptr(), (size_t)r.rows, as_int(r.C), dtype_code(x), at.stream),
              "dwo_int8_rows");
    return {codes, steps};
}
// act: -1 none
Tensor int8_linear(const Tensor &x_, const Tensor &codes_, const Tensor &steps_, const OptTensor &b_, int64_t act) {
    const Rows r(x_, "x");
    if (!codes_.is_cuda() || codes_.scalar_type() != at::kChar || codes_.dim() != 2 || codes_.size(1) != up16(r.C) || codes_.size(0) < 1)
        fail("weight codes must be a CUDA tensor of type int8, [N, " + std::to_string(up16(r.C)) + "] for x of " + std::to_string(r.C) + " channels");
    check_pair(x_, codes_);
    check_pair(x_, steps_);
    const int64_t D = codes_.size(0);
    if (steps_.scalar_type() != at::kFloat || steps_.dim() != 1 || steps_.size(0) != D) fail("weight scales must be float32, one for every row of the codes");
    check_bias(x_, b_, D, "bias");
    if (at::GradMode::is_enabled() && (trains(x_) || trains(steps_) || trains(b_)))
        fail("a layer in 8-bit integers has no gradients: call it without them (torch.no_grad, or on detached tensors)");
    py::gil_scoped_release nogil;
    const Place at(x_);
    const Tensor x = dense(x_), codes = dense(codes_), steps = dense(steps_), b = like(x, b_);
    Tensor y = at::empty(with_last(x, D), x.options());
    if (r.rows == 0) return y;
    const int dt = dtype_code(x);
    const size_t need = lib.int8_workspace_bytes((size_t)r.rows, as_int(r.C), as_int(D), dt);
    const Tensor ws = bytes(x, need);
    check(lib.int8_linear(ptr(x), ptr(codes), (const float *)ptr(steps), dptr(b), y.data_ptr(), ws.data_ptr(), need, (size_t)r.rows, as_int(r.C),
                          as_int(D), (int)act, dt, at.stream),
          "dwo_int8_linear");
    return y;
}

// ------------------------------------------------------------------------------------------------- top logits
std::tuple<Tensor, Tensor> top(const Tensor &x_, int64_t k) {
    const Rows r(x_, "logits");
    if (k < 1 || k > 1024 || k > r.C) throw py::value_error("k must be from 1 to 1024 and no more than there are classes");
    py::gil_scoped_release nogil;
    const Place at(x_);
    const Tensor x = dense(x_.detach());
    Tensor values = at::empty(with_last(x, k), x.options()), classes = at::empty(with_last(x, k), x.options().dtype(at::kLong));
    if (r.rows == 0) return {values, classes};
    const int dt = dtype_code(x);
    const size_t need = lib.top_workspace_bytes((size_t)r.rows, as_int(r.C), (int)k, dt);
    const Tensor ws = bytes(x, need);
    check(lib.top(ptr(x), values.data_ptr(), classes.data_ptr(), ws.data_ptr(), need, (size_t)r.rows, as_int(r.C), (int)k, dt, at.stream), "dwo_top");
    return {values, classes};
}

// ------------------------------------------------------------------------------------------------- distillation from top logits
// (loss, what the backward pass takes, number of rows that count or undefined)
std::tuple<Tensor, Tensor, Tensor> distill_forward(const Tensor &x, const Tensor &w, const Tensor &b, const Tensor &logits, const Tensor &classes,
                                                   double temperature, bool mean) {
    const Place at(x);
    const int64_t C = x.size(-1), rows = x.numel() / C, V = w.size(0), k = logits.size(-1);
    const auto f32 = x.options().dtype(at::kFloat);
    Tensor loss = mean ? at::empty({}, f32) : at::empty(without_last(x), f32);
    Tensor keep = at::empty({rows * (3 * k + 2)}, f32), count = mean ? at::empty({}, f32) : Tensor();
    if (rows == 0) {
        if (mean) loss.fill_(NAN), count.zero_();
        return {loss, keep, count};
    }
    const int dt = dtype_code(x);
    const size_t need = lib.distill_workspace_bytes((size_t)rows, as_int(C), as_int(V), as_int(k), 0, dt);
    const Tensor ws = bytes(x, need);
    check(lib.distill_forward(ptr(x), ptr(w), dptr(b), ptr(logits), ptr(classes), (float)temperature, (float *)keep.data_ptr(),
                              (float *)loss.data_ptr(), (float *)mptr(count), ws.data_ptr(), need, (size_t)rows, as_int(C), as_int(V), as_int(k), dt,
                              dtype_code(logits), at.stream),
          "dwo_distill_forward");
    return {loss, keep, count};
}
struct Distill : torch::autograd::Function<Distill> {
    static Tensor forward(Context *ctx, const Tensor &x_, const Tensor &w_, const OptTensor &b_, const Tensor &logits_, const Tensor &classes_,
                          double temperature, bool mean) {
        ctx->set_materialize_grads(false);
        const Place at(x_);
        const Tensor x = dense(x_), w = like(x, w_), b = like(x, b_);
        auto [loss, keep, count] = distill_forward(x, w, b, dense(logits_), dense(classes_), temperature, mean);
        ctx->save_for_backward({x, w, b, keep, count});
        ctx->saved_data["p"] = std::vector<int64_t>{logits_.size(-1), (int64_t)w_.scalar_type(), b_.has_value() ? (int64_t)b_->scalar_type() : -1};
        ctx->saved_data["t"] = temperature;
        return loss;
    }
    static List backward(Context *ctx, const List &grads) {
        List out(7);
        if (!grads[0].defined()) return out;
        const List s = ctx->get_saved_variables();
        const Tensor &x = s[0], &w = s[1], &b = s[2], &keep = s[3], &count = s[4];
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
            const size_t need = lib.distill_workspace_bytes((size_t)rows, as_int(C), as_int(V), as_int(p[0]), 1, dt);
            const Tensor ws = bytes(x, need);
            check(lib.distill_backward((const float *)ptr(up), ptr(x), ptr(w), dptr(b), (const float *)ptr(keep),
                                       (float)ctx->saved_data["t"].toDouble(), (const float *)dptr(count), mptr(dx), mptr(dw), mptr(db), ws.data_ptr(),
                                       need, (size_t)rows, as_int(C), as_int(V), as_int(p[0]), dt, dtype_code(w_type), at.stream),
                  "dwo_distill_backward");
        }
        out[0] = dx;
        if (ctx->needs_input_grad(1)) out[1] = dw;
        if (need_db) out[2] = as_type(db, (at::ScalarType)p[2]);
        return out;
    }
};
Tensor distill(const Tensor &x, const Tensor &w, const OptTensor &b, const Tensor &logits, const Tensor &classes, double temperature, bool mean) {
    const Rows r(x, "x");
    check_weight(x, w, -1, r.C, "weight");
    check_bias(x, b, w.size(0), "bias");
    check_glue(logits, "teacher_logits");
    check_pair(x, logits);
    check_pair(x, classes);
    if (logits.dim() != x.dim() || logits.sizes().slice(0, x.dim() - 1) != x.sizes().slice(0, x.dim() - 1) || logits.size(-1) < 1 || logits.size(-1) > 1024)
        fail("teacher_logits must have from 1 to 1024 entries for every row of x");
    if (classes.scalar_type() != at::kLong || classes.sizes() != logits.sizes()) fail("teacher_classes must be int64, one class for every teacher logit");
    if (!(temperature >= 1e-4 && temperature <= 1e4)) fail("temperature must be from 1e-4 to 1e4");
    if (at::GradMode::is_enabled() && trains(logits)) fail("the teacher's logits get no gradient: detach them");
    py::gil_scoped_release nogil;
    if (at::GradMode::is_enabled() && (trains(x) || trains(w) || trains(b)))
        return Distill::apply(x, w, b, logits, classes, temperature, mean);
    const Place at(x);
    const Tensor d = dense(x);
    return std::get<0>(distill_forward(d, like(d, w), like(d, b), dense(logits), dense(classes), temperature, mean));
}
