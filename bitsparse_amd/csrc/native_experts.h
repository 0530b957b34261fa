// Dropout and the experts' operators: the bodies of dropout.py's and
// experts.py's calls (part of native.cpp).
#pragma once

// ---------------------------------------------------------------------------
// dropout
// ---------------------------------------------------------------------------
// What a dropout is besides its operand.  `state`: [seed, offset] on the
// device, for a captured graph whose replays draw anew.
struct DropKind {
    int64_t below = 0;
    uint64_t seed = 0, offset = 0;
    Maybe state;
};

bs_drop drop_args(const DropKind& k, const Tensor& on)
{
    bs_drop d{k.seed, k.offset, nullptr, (int)k.below};
    if (k.state) {
        plain_on_gpu(*k.state, "drop.seed");
        TORCH_CHECK_TYPE(k.state->scalar_type() == at::kLong, "drop.seed: a tensor holds int64 [seed, offset], got ", k.state->scalar_type());
        TORCH_CHECK_VALUE(k.state->numel() == 2 && k.state->is_contiguous(), "drop.seed: expected a contiguous [seed, offset], got ", k.state->sizes());
        TORCH_CHECK(k.state->device() == on.device(), "drop.seed is on ", k.state->device(), ", the values on ", on.device());
        d.state = k.state->data_ptr<int64_t>();
    }
    return d;
}

Tensor dropped(const Tensor& x, const DropKind& k)
{
    plain_on_gpu(x, "x");
    const int type = row_type(x, "x");
    const c10::DeviceGuard guard(x.device());
    const bs_drop d = drop_args(k, x);
    Tensor out = at::empty(x.sizes(), x.options());
    if (x.numel() == 0) return out;
    const int64_t cols = x.dim() ? x.size(-1) : 1;
    const Tensor rows = as_rows(x.dim() ? x : x.reshape({1}), cols);
    check(L.bs_dropout(&d, rows.data_ptr(), type, rows.size(0), cols, row_stride(rows), out.data_ptr(), stream_of(x)), "bs_dropout");
    return out;
}

// (linear, and its own transpose: any order of derivatives)
struct Dropped : torch::autograd::Function<Dropped> {
    static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& x, const DropKind& k)
    {
        Tensor out = dropped(x, k);
        ctx->saved_data["below"] = k.below;
        ctx->saved_data["seed"] = (int64_t)k.seed;
        ctx->saved_data["offset"] = (int64_t)k.offset;
        ctx->saved_data["type"] = (int64_t)x.scalar_type();
        ctx->save_for_backward({k.state ? *k.state : Tensor()});
        return out;
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, const torch::autograd::variable_list& grads)
    {
        if (!grads[0].defined()) return {Tensor(), Tensor()};
        DropKind k{ctx->saved_data["below"].toInt(), (uint64_t)ctx->saved_data["seed"].toInt(), (uint64_t)ctx->saved_data["offset"].toInt(), {}};
        const Tensor state = ctx->get_saved_variables()[0];
        if (state.defined()) k.state = state;
        TORCH_CHECK_TYPE((int64_t)grads[0].scalar_type() == ctx->saved_data["type"].toInt(), "the gradient: unexpected dtype ", grads[0].scalar_type());
        if (at::GradMode::is_enabled() && grads[0].requires_grad()) return {Dropped::apply(grads[0], k), Tensor()};
        return {dropped(grads[0], k), Tensor()};
    }
};

Tensor dropout(const Tensor& x, int64_t below, uint64_t seed, uint64_t offset, const Maybe& state)
{
    const DropKind k{below, seed, offset, state};
    return at::GradMode::is_enabled() && x.requires_grad() ? Dropped::apply(x, k) : dropped(x, k);
}

// ---------------------------------------------------------------------------
// routing
// ---------------------------------------------------------------------------
struct RouteKind {
    Maybe bias;
    int64_t top_k, score, groups, top_groups, group_best;
    bool renormalize;
    double scale;
};

struct RouteCall {
    bs_route a{};
    Tensor logits, bias;
    RouteCall(const Tensor& l, const RouteKind& k)
    {
        plain_on_gpu(l, "logits");
        TORCH_CHECK_VALUE(l.dim() >= 1 && l.size(-1) > 0, "logits: expected [..., experts], got ", l.sizes());
        a.logits_type = row_type(l, "logits");
        const int64_t E = l.size(-1);
        logits = as_rows(l, E);
        auto narrow = [](int64_t v) { return (int)std::clamp<int64_t>(v, -1, 1 << 30); };
        a.tokens = logits.size(0), a.experts = narrow(E), a.top_k = narrow(k.top_k);
        a.logits = a.tokens ? logits.data_ptr() : nullptr, a.logits_stride = row_stride(logits);
        if (k.bias) {
            plain_on_gpu(*k.bias, "bias");
            TORCH_CHECK(k.bias->device() == l.device(), "bias is on ", k.bias->device(), ", logits on ", l.device());
            TORCH_CHECK_TYPE(k.bias->scalar_type() == at::kFloat, "bias must be float32, got ", k.bias->scalar_type());
            TORCH_CHECK_VALUE(k.bias->dim() == 1 && k.bias->size(0) == E, "bias: expected shape [", E, "], got ", k.bias->sizes());
            bias = k.bias->contiguous();
            a.bias = bias.data_ptr<float>();
        }
        a.score = narrow(k.score), a.groups = narrow(k.groups), a.top_groups = narrow(k.top_groups), a.group_best = narrow(k.group_best);
        a.renormalize = k.renormalize, a.scale = (float)k.scale;
    }
};

std::pair<Tensor, Tensor> route_forward(const Tensor& logits, const RouteKind& k)
{
    const c10::DeviceGuard guard(logits.device());
    RouteCall c(logits, k);
    TORCH_CHECK_VALUE(k.top_k >= 1 && k.top_k <= std::min<int64_t>(logits.size(-1), 64), "top_k must be in 1..64 and at most the number of experts, got ",
                      k.top_k, " of ", logits.size(-1));
    auto shape = logits.sizes().vec();
    shape.back() = k.top_k;
    const Tensor w = at::empty(shape, logits.options().dtype(at::kFloat)), chosen = at::empty(shape, logits.options().dtype(at::kInt));
    check(L.bs_route_forward(&c.a, w.numel() ? w.data_ptr<float>() : nullptr, chosen.numel() ? chosen.data_ptr<int32_t>() : nullptr, stream_of(logits)),
          "bs_route_forward");
    return {w, chosen};
}

struct RouteNode : torch::CustomClassHolder {
    RouteKind kind;
    c10::SmallVector<int64_t, 4> shape;
    at::TensorOptions options;
};

void no_second(const char* what)
{
    TORCH_CHECK_NOT_IMPLEMENTED(!at::GradMode::is_enabled(), "bitsparse_amd: ", what, " has no second derivative (create_graph)");
}
// (hooks on saved tensors may hand back others than were saved)
void as_saved(const Tensor& t, at::IntArrayRef sizes, at::ScalarType type, c10::Device device, const char* what)
{
    plain_on_gpu(t, what);
    TORCH_CHECK(t.device() == device && t.scalar_type() == type && t.sizes() == sizes, what, ": expected what was saved, ", type, " ", sizes,
                " on ", device, ", got ", t.scalar_type(), " ", t.sizes(), " on ", t.device());
}

struct Route : torch::autograd::Function<Route> {
    static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const Tensor& logits, const RouteKind& k)
    {
        const auto [w, chosen] = route_forward(logits, k);
        auto node = c10::make_intrusive<RouteNode>();
        node->kind = k, node->kind.bias.reset();        // (the choice is made)
        node->shape.assign(logits.sizes().begin(), logits.sizes().end());
        node->options = logits.options();
        ctx->saved_data["node"] = c10::IValue::make_capsule(node);
        ctx->save_for_backward({logits, chosen});
        ctx->mark_non_differentiable({chosen});
        ctx->set_materialize_grads(false);
        return {w, chosen};
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, const torch::autograd::variable_list& grads)
    {
        no_second("routing");
        if (!grads[0].defined()) return {Tensor(), Tensor()};
        const auto saved = ctx->get_saved_variables();
        const auto capsule = ctx->saved_data["node"].toCapsule();
        const RouteNode& node = static_cast<const RouteNode&>(*capsule);
        const c10::Device device = node.options.device();
        const c10::DeviceGuard guard(device);
        auto shape = std::vector<int64_t>(node.shape.begin(), node.shape.end());
        as_saved(saved[0], shape, node.options.dtype().toScalarType(), device, "logits");
        shape.back() = node.kind.top_k;
        as_saved(saved[1], shape, at::kInt, device, "the chosen experts");
        as_saved(grads[0], shape, at::kFloat, device, "the gradient of the weights");
        const RouteCall c(saved[0], node.kind);
        const Tensor d = at::empty(saved[0].sizes(), node.options);
        if (d.numel() == 0) return {d, Tensor()};
        const Tensor chosen = saved[1].contiguous(), g = grads[0].contiguous();
        check(L.bs_route_backward(&c.a, chosen.data_ptr<int32_t>(), g.data_ptr<float>(), d.data_ptr(), stream_of(d)), "bs_route_backward");
        return {d, Tensor()};
    }
};

std::vector<Tensor> route(const Tensor& logits, const Maybe& bias, int64_t top_k, int64_t score, int64_t groups, int64_t top_groups,
                          int64_t group_best, bool renormalize, double scale)
{
    const RouteKind k{bias ? Maybe(bias->detach()) : bias, top_k, score, groups, top_groups, group_best, renormalize, scale};
    if (at::GradMode::is_enabled() && logits.requires_grad()) return Route::apply(logits, k);
    const auto [w, chosen] = route_forward(logits, k);
    return {w, chosen};
}

// (offsets, order, place)
std::vector<Tensor> plan_experts(const Tensor& chosen, int64_t experts)
{
    plain_on_gpu(chosen, "experts");
    TORCH_CHECK_TYPE(chosen.scalar_type() == at::kInt, "experts must be int32, got ", chosen.scalar_type());
    TORCH_CHECK_VALUE(chosen.dim() >= 1 && chosen.size(-1) > 0, "experts: expected [..., top_k], got ", chosen.sizes());
    TORCH_CHECK_VALUE(experts >= 1 && experts <= 1024, "n_experts must be in 1..1024, got ", experts);
    const c10::DeviceGuard guard(chosen.device());
    const Tensor ids = chosen.contiguous();
    const Tensor offsets = at::empty({experts + 1}, ids.options()), order = at::empty({ids.numel()}, ids.options()),
                 place = at::empty(chosen.sizes(), ids.options());
    const int64_t need = L.bs_expert_plan_workspace_bytes(ids.numel(), (int)experts);
    Tensor ws;
    if (need) ws = at::empty({need}, ids.options().dtype(at::kByte));
    check(L.bs_expert_plan(ptr<int32_t>(ids), ids.numel(), (int)experts, offsets.data_ptr<int32_t>(), ptr<int32_t>(order), ptr<int32_t>(place),
                           raw(ws), need, stream_of(ids)),
          "bs_expert_plan");
    return {offsets, order, place};
}

// ---------------------------------------------------------------------------
// the experts' products
// ---------------------------------------------------------------------------
// A plan as the kernels read it.
struct Plan {
    Tensor offsets, order, place;       // [E + 1], [T k], [..., k]
    int64_t experts, rows, tokens, top_k;
    Plan(const Tensor& offsets_, const Tensor& order_, const Tensor& place_)
    {
        const struct { const Tensor& t; const char* what; } all[] = {{offsets_, "plan.offsets"}, {order_, "plan.order"}, {place_, "plan.place"}};
        for (const auto& i : all) {
            plain_on_gpu(i.t, i.what);
            TORCH_CHECK_TYPE(i.t.scalar_type() == at::kInt, i.what, " must be int32, got ", i.t.scalar_type());
            TORCH_CHECK(i.t.device() == offsets_.device(), i.what, " is on ", i.t.device(), ", plan.offsets on ", offsets_.device());
        }
        TORCH_CHECK_VALUE(offsets_.dim() == 1 && offsets_.size(0) >= 2 && offsets_.size(0) <= 1025,
                          "plan.offsets: expected the offsets of 1..1024 experts and the end, got ", offsets_.sizes());
        TORCH_CHECK_VALUE(place_.dim() >= 1 && place_.size(-1) > 0 && place_.size(-1) <= 64, "plan.place: expected [..., top_k] with top_k in 1..64, got ",
                          place_.sizes());
        TORCH_CHECK_VALUE(order_.dim() == 1 && order_.size(0) == place_.numel(), "plan.order: expected shape [", place_.numel(), "], got ", order_.sizes());
        TORCH_CHECK_VALUE(place_.numel() < (int64_t(1) << 31), "plan: 2^31 pairs or more");
        offsets = offsets_.contiguous(), order = order_.contiguous(), place = place_.contiguous();
        experts = offsets.size(0) - 1, rows = order.size(0), top_k = place.size(-1), tokens = rows / top_k;
    }
    bs_experts args(bool gather) const
    {
        return {rows, tokens, (int)experts, (int)top_k, offsets.data_ptr<int32_t>(), gather ? ptr<int32_t>(order) : nullptr};
    }
    const int32_t* used() const { return offsets.data_ptr<int32_t>() + experts; }
    std::vector<int64_t> token_shape(int64_t cols) const
    {
        std::vector<int64_t> s = place.sizes().vec();
        s.back() = cols;
        return s;
    }
};

void bf16_on(const Tensor& t, const char* what, const Plan& plan)
{
    plain_on_gpu(t, what);
    TORCH_CHECK_TYPE(t.scalar_type() == at::kBFloat16, what, " must be bfloat16, got ", t.scalar_type());
    TORCH_CHECK(t.device() == plan.offsets.device(), what, " is on ", t.device(), ", the plan on ", plan.offsets.device());
}

// rows as 16-byte loads take them: themselves, or a copy padded with zeros
struct Rows16 {
    Tensor t;
    int64_t stride;
    bool padded = false;
    explicit Rows16(const Tensor& rows)
    {
        const int64_t R = rows.size(0), C = rows.size(1), width = (C + 7) / 8 * 8;
        stride = R > 1 ? rows.stride(0) : width;
        if (C % 8 == 0 && stride % 8 == 0 && stride >= C && stride < (int64_t(1) << 22) && (uintptr_t)raw(rows) % 16 == 0) {
            t = rows;
            return;
        }
        t = at::empty({R, width}, rows.options());
        check(L.bs_pad_rows(raw(rows), R, C, row_stride(rows), raw(t), width, stream_of(rows)), "bs_pad_rows");
        stride = width;
        padded = true;
    }
};

// x's rows: the tokens' (gather) or the plan's
Tensor expert_operand(const Tensor& x, const Plan& plan, bool gather, const char* what)
{
    bf16_on(x, what, plan);
    TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) > 0, what, ": expected rows [..., D] with D > 0, got ", x.sizes());
    const Tensor rows = as_rows(x, x.size(-1));
    TORCH_CHECK_VALUE(rows.size(0) == (gather ? plan.tokens : plan.rows), what, ": expected ", gather ? plan.tokens : plan.rows,
                      gather ? " tokens" : " rows in the plan's order", ", got ", x.sizes());
    return rows;
}
// weights [E, N, D] as rows
Rows16 expert_weights(const Tensor& W)
{
    return Rows16(W.is_contiguous() ? W.view({W.size(0) * W.size(1), W.size(2)}) : W.contiguous().view({W.size(0) * W.size(1), W.size(2)}));
}
void check_weights(const Tensor& W, const Plan& plan, const char* what)
{
    bf16_on(W, what, plan);
    TORCH_CHECK_VALUE(W.dim() == 3 && W.size(0) == plan.experts && W.size(1) > 0 && W.size(2) > 0, what, ": expected [", plan.experts,
                      " experts, out, in], got ", W.sizes());
}

// A gathered operand.  `written`, and one of 4 GiB or more, which is past the
// loads' offsets: its rows are written out in the plan's order.
struct Gathered {
    Rows16 rows;
    bool gather;
    Gathered(const Tensor& x, const Plan& plan, bool gather_, bool written)
        : rows(gather_ && (written || too_far(x)) ? written_out(x, plan) : x), gather(gather_ && !written && !too_far(x))
    {
    }
    static bool too_far(const Tensor& x)
    {
        const int64_t width = (x.size(1) + 7) / 8 * 8;
        return x.size(0) * std::max(width, row_stride(x)) * 2 >= (int64_t(1) << 32) - 32;
    }
    static Tensor written_out(const Tensor& x, const Plan& plan)
    {
        Tensor t = at::empty({plan.rows, x.size(1)}, x.options());
        const bs_experts e = plan.args(false);
        check(L.bs_expert_combine_plan_backward(&e, raw(x), row_stride(x), nullptr, 0, nullptr, ptr<int32_t>(plan.place), x.size(1), raw(t), nullptr,
                                                stream_of(x)),
              "bs_expert_combine_plan_backward");
        return t;
    }
};

Tensor expert_product(const Rows16& w, const Gathered& a, const Plan& plan, int64_t in, int64_t out, int64_t act, double act_k)
{
    Tensor y = at::empty({plan.rows, out}, a.rows.t.options());
    if (plan.rows == 0) return y;
    const bs_experts e = plan.args(a.gather);
    check(L.bs_expert_linear(&e, raw(a.rows.t), a.rows.stride, raw(w.t), w.stride, in, out, (int)act, (float)act_k, raw(y), stream_of(y)),
          "bs_expert_linear");
    return y;
}
// in the plan's order
Tensor expert_product_dx(const Rows16& g, const Rows16& w, const Plan& plan, int64_t in, int64_t out, at::ScalarType type)
{
    Tensor dx = at::empty({plan.rows, in}, g.t.options().dtype(type));
    if (plan.rows == 0) return dx;
    const bs_experts e = plan.args(false);
    check(L.bs_expert_linear_dx(&e, raw(g.t), g.stride, raw(w.t), w.stride, in, out, raw(dx), type == at::kFloat ? BS_DT_F32 : BS_DT_BF16,
                                stream_of(dx)),
          "bs_expert_linear_dx");
    return dx;
}
// x: rows in the plan's order
Tensor expert_product_dw(const Rows16& g, const Rows16& x, const Plan& plan, int64_t in, int64_t out)
{
    Tensor dW = at::empty({plan.experts, out, in}, g.t.options());
    const bs_experts e = plan.args(false);
    check(L.bs_expert_linear_dw(&e, raw(g.t), g.stride, raw(x.t), x.stride, in, out, raw(dW), stream_of(dW)), "bs_expert_linear_dw");
    return dW;
}
// (operands checked, and the rows of x)
Tensor expert_operands(const Tensor& x, const Tensor& W, const Plan& plan, bool gather)
{
    const Tensor rows = expert_operand(x, plan, gather, "x");
    check_weights(W, plan, "W");
    TORCH_CHECK_VALUE(W.size(2) == rows.size(1), "W: expected ", rows.size(1), " columns, as x has, got ", W.sizes());
    return rows;
}
// sums over the choices of each token, in bf16
Tensor combined(const Tensor& y, const Tensor& weights, const Plan& plan)
{
    const c10::DeviceGuard guard(plan.offsets.device());
    Tensor out = at::empty(plan.token_shape(y.size(1)), y.options().dtype(at::kBFloat16));
    if (out.numel() == 0) return out;
    const bs_experts e = plan.args(false);
    check(L.bs_expert_combine_plan(&e, raw(y), y.scalar_type() == at::kFloat ? BS_DT_F32 : BS_DT_BF16, row_stride(y), ptr<float>(weights),
                                   ptr<int32_t>(plan.place), y.size(1), raw(out), stream_of(out)),
          "bs_expert_combine_plan");
    return out;
}

// the plan's tensors and an operator's other arguments, kept for a backward
struct ExpertsNode : torch::CustomClassHolder {
    bool gather = false, gathered = false, need[2] = {}, copied[2] = {};
    std::vector<int64_t> shape[2], operand[2], plan_shape[3];       // of what is saved, of the operands
    at::TensorOptions options;
};

void keep_plan(ExpertsNode& node, const Plan& p)
{
    const Tensor* all[3] = {&p.offsets, &p.order, &p.place};
    for (int i = 0; i < 3; i++) node.plan_shape[i] = all[i]->sizes().vec();
    node.options = p.offsets.options();
}
Plan kept_plan(const ExpertsNode& node, const torch::autograd::variable_list& saved, int at)
{
    static constexpr const char* names[3] = {"plan.offsets", "plan.order", "plan.place"};
    for (int i = 0; i < 3; i++) as_saved(saved[at + i], node.plan_shape[i], at::kInt, node.options.device(), names[i]);
    return Plan(saved[at], saved[at + 1], saved[at + 2]);
}

struct PlanTensors {
    Tensor offsets, order, place;
};

struct ExpertLinear : torch::autograd::Function<ExpertLinear> {
    static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& x, const Tensor& W, const PlanTensors& p, bool gather)
    {
        const Plan plan(p.offsets, p.order, p.place);
        const c10::DeviceGuard guard(plan.offsets.device());
        const Tensor rows = expert_operands(x, W, plan, gather);
        const Gathered a(rows, plan, gather, false);
        const Rows16 w = expert_weights(W);
        Tensor y = expert_product(w, a, plan, W.size(2), W.size(1), BS_ACT_NONE, 0.0);
        auto node = c10::make_intrusive<ExpertsNode>();
        node->gather = a.gather;        // (rows that were written out are rows)
        node->need[0] = x.requires_grad(), node->need[1] = W.requires_grad();
        node->gathered = gather;
        node->operand[0] = x.sizes().vec(), node->operand[1] = W.sizes().vec();
        // What a gradient that is asked for is formed of; of padded operands the copies, which the backward pass would make again.
        const bool copied = a.rows.padded || gather != a.gather;
        const Tensor keep_x = node->need[1] ? copied ? a.rows.t : x : Tensor(), keep_W = node->need[0] ? w.padded ? w.t : W : Tensor();
        if (keep_x.defined()) node->shape[0] = keep_x.sizes().vec();
        if (keep_W.defined()) node->shape[1] = keep_W.sizes().vec();
        node->copied[0] = copied, node->copied[1] = w.padded;
        keep_plan(*node, plan);
        ctx->saved_data["node"] = c10::IValue::make_capsule(node);
        ctx->save_for_backward({keep_x, keep_W, plan.offsets, plan.order, plan.place});
        return y;
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, const torch::autograd::variable_list& grads)
    {
        no_second("expert_linear");
        const auto saved = ctx->get_saved_variables();
        const auto capsule = ctx->saved_data["node"].toCapsule();
        const ExpertsNode& node = static_cast<const ExpertsNode&>(*capsule);
        const c10::Device device = node.options.device();
        const c10::DeviceGuard guard(device);
        torch::autograd::variable_list out(4);
        const Plan plan = kept_plan(node, saved, 2);
        const int64_t D = node.operand[1][2], N = node.operand[1][1];
        as_saved(grads[0], {plan.rows, N}, at::kBFloat16, device, "the gradient of y");
        const Rows16 g(as_rows(grads[0], N));
        if (ctx->needs_input_grad(0) && node.need[0]) {
            as_saved(saved[1], node.shape[1], at::kBFloat16, device, "W");
            const Rows16 w = node.copied[1] ? Rows16(saved[1].contiguous()) : expert_weights(saved[1]);
            // (a gathered token's rows are rounded once, in their sum)
            const Tensor dx = expert_product_dx(g, w, plan, D, N, node.gathered && plan.top_k > 1 ? at::kFloat : at::kBFloat16);
            out[0] = (node.gathered ? combined(dx, Tensor(), plan) : dx).view(node.operand[0]);
        }
        if (ctx->needs_input_grad(1) && node.need[1]) {
            as_saved(saved[0], node.shape[0], at::kBFloat16, device, "x");
            const Tensor x = as_rows(saved[0], node.shape[0].back());
            out[1] = expert_product_dw(g, Gathered(x, plan, node.gather && plan.rows, true).rows, plan, D, N);
        }
        return out;
    }
};

Tensor expert_product_act(const Tensor& x, const Tensor& W, const Tensor& offsets, const Tensor& order, const Tensor& place, bool gather,
                          int64_t act, double act_k)
{
    const Plan plan(offsets, order, place);
    const c10::DeviceGuard guard(plan.offsets.device());
    const Tensor rows = expert_operands(x, W, plan, gather);
    return expert_product(expert_weights(W), Gathered(rows, plan, gather, false), plan, W.size(2), W.size(1), act, act_k);
}

Tensor expert_linear(const Tensor& x, const Tensor& W, const Tensor& offsets, const Tensor& order, const Tensor& place, bool gather)
{
    if (at::GradMode::is_enabled() && (x.requires_grad() || W.requires_grad())) return ExpertLinear::apply(x, W, PlanTensors{offsets, order, place}, gather);
    return expert_product_act(x, W, offsets, order, place, gather, BS_ACT_NONE, 0.0);
}

// ---------------------------------------------------------------------------
// the weighted sum
// ---------------------------------------------------------------------------
struct CombineCall {
    Tensor y, w;
    CombineCall(const Tensor& y_, const Tensor& weights, const Plan& plan)
    {
        y = expert_operand(y_, plan, false, "y");
        plain_on_gpu(weights, "weights");
        TORCH_CHECK_TYPE(weights.scalar_type() == at::kFloat, "weights must be float32, got ", weights.scalar_type());
        TORCH_CHECK(weights.device() == plan.offsets.device(), "weights are on ", weights.device(), ", the plan on ", plan.offsets.device());
        TORCH_CHECK_VALUE(weights.sizes() == plan.place.sizes(), "weights: expected shape ", plan.place.sizes(), ", got ", weights.sizes());
        w = weights.contiguous();
    }
};

struct ExpertCombine : torch::autograd::Function<ExpertCombine> {
    static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& y, const Tensor& weights, const PlanTensors& p)
    {
        const Plan plan(p.offsets, p.order, p.place);
        const CombineCall c(y, weights, plan);
        Tensor out = combined(c.y, c.w, plan);
        auto node = c10::make_intrusive<ExpertsNode>();
        node->need[0] = y.requires_grad(), node->need[1] = weights.requires_grad();
        node->shape[0] = y.sizes().vec(), node->shape[1] = weights.sizes().vec();
        keep_plan(*node, plan);
        ctx->saved_data["node"] = c10::IValue::make_capsule(node);
        ctx->save_for_backward({node->need[1] ? y : Tensor(), node->need[0] ? weights : Tensor(), plan.offsets, plan.order, plan.place});
        return out;
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, const torch::autograd::variable_list& grads)
    {
        no_second("expert_combine");
        const auto saved = ctx->get_saved_variables();
        const auto capsule = ctx->saved_data["node"].toCapsule();
        const ExpertsNode& node = static_cast<const ExpertsNode&>(*capsule);
        const c10::Device device = node.options.device();
        const c10::DeviceGuard guard(device);
        const Plan plan = kept_plan(node, saved, 2);
        const int64_t D = node.shape[0].back();
        as_saved(grads[0], plan.token_shape(D), at::kBFloat16, device, "the gradient of the sum");
        const Tensor g = as_rows(grads[0], D);
        torch::autograd::variable_list out(3);
        Tensor y, w;
        if (ctx->needs_input_grad(0) && node.need[0]) {
            as_saved(saved[1], node.shape[1], at::kFloat, device, "weights");
            w = saved[1].contiguous();
            out[0] = at::empty(node.shape[0], grads[0].options());
        }
        if (ctx->needs_input_grad(1) && node.need[1]) {
            as_saved(saved[0], node.shape[0], at::kBFloat16, device, "y");
            y = as_rows(saved[0], D);
            out[1] = at::empty(node.shape[1], grads[0].options().dtype(at::kFloat));
        }
        if (plan.rows == 0 || (!out[0].defined() && !out[1].defined())) return out;
        const bs_experts e = plan.args(false);
        check(L.bs_expert_combine_plan_backward(&e, raw(g), row_stride(g), raw(y), y.defined() ? row_stride(y) : 0, ptr<float>(w),
                                                ptr<int32_t>(plan.place), D, raw(out[0]), ptr<float>(out[1]), stream_of(g)),
              "bs_expert_combine_plan_backward");
        return out;
    }
};

Tensor expert_combine(const Tensor& y, const Tensor& weights, const Tensor& offsets, const Tensor& order, const Tensor& place)
{
    if (at::GradMode::is_enabled() && (y.requires_grad() || weights.requires_grad()))
        return ExpertCombine::apply(y, weights, PlanTensors{offsets, order, place});
    const Plan plan(offsets, order, place);
    const CombineCall c(y, weights, plan);
    return combined(c.y, c.w, plan);
}

// ---------------------------------------------------------------------------
// a block of experts (experts.py's ExpertsRelu and ExpertsRelu2)
// ---------------------------------------------------------------------------
// The gradients of out = sum of w act(x W1^T) W2^T over a token's choices, of
// (x, W1, W2, weights) those that are wanted.  r: the saved relu(x W1^T)
// [rows, H], overwritten.  The result y of the second product is not needed:
// the weights' gradient is <dout W2, act>.
std::vector<std::optional<Tensor>> experts_backward(const Tensor& grad, const Tensor& x, const Tensor& W1, const Tensor& W2, const Tensor& weights,
                                                    const Tensor& offsets, const Tensor& order, const Tensor& place, const Tensor& r, bool square,
                                                    double k, std::vector<bool> need)
{
    const Plan plan(offsets, order, place);
    const c10::DeviceGuard guard(plan.offsets.device());
    // (those that this walk through the graph asks for; the node's edges are its tensors in order)
    if (const std::shared_ptr<torch::autograd::Node> node = torch::autograd::get_current_node(); node && node->name() == "_ExpertsBlockBackward")
        for (size_t i = 0; i < need.size(); i++) need[i] = need[i] && node->task_should_compute_output(i);
    TORCH_CHECK_VALUE(need.size() == 4, "four gradients, each wanted or not");
    const Tensor tokens = expert_operand(x, plan, true, "x");
    check_weights(W1, plan, "W1");
    check_weights(W2, plan, "W2");
    const int64_t H = W1.size(1), O = W2.size(1);
    const CombineCall w(r, weights, plan);
    TORCH_CHECK_VALUE(W1.size(2) == tokens.size(1) && W2.size(2) == H && r.dim() == 2 && r.size(1) == H && r.is_contiguous(),
                      "the operands are not those of the forward pass");
    as_saved(grad, plan.token_shape(O), at::kBFloat16, plan.offsets.device(), "the gradient");
    std::vector<std::optional<Tensor>> out(4);
    const Tensor g_tokens = as_rows(grad, O);
    // (before its weights, in the plan's order)
    const Rows16 dy(plan.rows ? Gathered::written_out(g_tokens, plan) : at::empty({0, O}, grad.options()));
    const Tensor dz = expert_product_dx(dy, expert_weights(W2), plan, H, O, at::kBFloat16);
    Tensor dw;
    if (need[3]) dw = at::zeros(weights.sizes(), weights.options());
    if (plan.rows)
        check(L.bs_experts_act_grad(raw(dz), raw(r), plan.rows, H, square, (float)k, ptr<float>(w.w), ptr<int32_t>(plan.order), plan.used(), plan.rows,
                                    ptr<float>(dw), stream_of(dz)),
              "bs_experts_act_grad");
    if (need[3]) out[3] = dw;
    if (need[2]) out[2] = expert_product_dw(dy, Rows16(r), plan, H, O);
    if (!need[0] && !need[1]) return out;
    const int64_t D = tokens.size(1);
    const Rows16 g(dz);
    if (need[0])
        out[0] = combined(expert_product_dx(g, expert_weights(W1), plan, D, H, plan.top_k > 1 ? at::kFloat : at::kBFloat16), Tensor(), plan).view(x.sizes());
    if (need[1]) out[1] = expert_product_dw(g, Gathered(tokens, plan, plan.rows > 0, true).rows, plan, D, H);
    return out;
}
