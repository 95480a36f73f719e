// 8-bit rows and what reads them, over at::Tensor, with autograd nodes.  The nodes keep codes and scales through the
// saved-tensor hooks; scales and softmax statistics go through them as bytes, so that a hook that stores floating activations
// in fewer bits leaves them alone.
#include "torch_rows8.h"
#include "torch_nodes.h"

#include <cmath>

namespace tango_host {

constexpr int64_t kMaxGroup = 1024, kMaxHeadWidth = 512;

static int type_code(const Tensor &t) {
    const auto s = t.scalar_type();
    return s == at::kFloat ? TANGO_FP32 : s == at::kBFloat16 ? TANGO_BF16 : s == at::kHalf ? TANGO_FP16 : -1;
}
static void require_matrix(const Tensor &t) {
    require(t.is_cuda() && t.layout() == at::kStrided && type_code(t) >= 0, "fp32, bf16 or fp16 CUDA tensor expected");
}
static void require_group(int64_t group) { require(group >= 1 && group <= kMaxGroup, "groups of 1 to 1024 columns"); }

static Tensor bytes(const Tensor &t) { return t.defined() ? t.view(at::kByte) : t; }
static Tensor numbers(const Tensor &t) { return t.contiguous().view(at::kFloat); }

static Rows8 alloc_rows8(int64_t rows, int64_t cols, int64_t group, const Tensor &like) {
    const int64_t groups = cols ? (cols + group - 1) / group : 0;
    return {at::empty({rows, tango_rows8_ld(cols, group)}, like.options().dtype(at::kChar)),
            at::empty({rows, groups}, like.options().dtype(at::kFloat))};
}

// Up to four matrices of one shape and type in one launch.  paired: the last two become one tensor of codes, interleaved, with
// their scales in pairs.
static std::vector<Rows8> pack_all(std::initializer_list<Tensor> tensors, int64_t group, bool paired = false) {
    const Tensor &first = *tensors.begin();
    const c10::cuda::CUDAGuard guard(first.device());
    std::vector<Matrix> x;
    std::vector<Rows8> out;
    tango_rows8_job jobs[4];
    for (const Tensor &t : tensors) x.push_back(matrix(t));
    const size_t apart = x.size() - (paired ? 2 : 0);
    for (size_t k = 0; k < apart; ++k) {
        out.push_back(alloc_rows8(x[k].rows, x[k].cols, group, first));
        jobs[k] = {ptr(x[k].t), x[k].ld, ptr<int8_t>(out[k].q), ptr<float>(out[k].scale), 1, 0};
    }
    if (paired) {
        const int64_t groups = (x[0].cols + group - 1) / group, run = tango_rows8_run(group);
        const Rows8 both{at::empty({x[0].rows, 2 * tango_rows8_ld(x[0].cols, group)}, first.options().dtype(at::kChar)),
                         at::empty({x[0].rows, groups, 2}, first.options().dtype(at::kFloat))};
        out.push_back(both);
        for (size_t k = apart; k < x.size(); ++k)
            jobs[k] = {ptr(x[k].t), x[k].ld, ptr<int8_t>(both.q) ? ptr<int8_t>(both.q) + (k - apart) * run : nullptr,
                       ptr<float>(both.scale) ? ptr<float>(both.scale) + (k - apart) : nullptr, 2, 1};
    }
    if (x[0].rows == 0 || x[0].cols == 0) return out;
    const int mode = settings().mode_quantize, n = (int)x.size();
    const uint64_t call = mode == TANGO_ROUND_STOCHASTIC ? next_call() : 0;
    for (int k = 1; k < n && call; ++k) next_call();
    check(tango_rows8_pack(jobs, n, x[0].rows, x[0].cols, group, type_code(first), mode, settings().seed, call, settings().step,
                           cuda_stream()), "pack8");
    count(1);
    return out;
}

Rows8 pack8(const Tensor &x, int64_t group) {
    require_matrix(x);
    require_group(group);
    const Raw raw;
    return pack_all({x}, group)[0];
}

Tensor unpack8(const Rows8 &r, at::IntArrayRef sizes, int64_t group, at::ScalarType type) {
    require_group(group);
    require(r.q.is_cuda() && r.q.scalar_type() == at::kChar && r.scale.scalar_type() == at::kFloat && r.scale.device() == r.q.device(),
            "int8 codes and fp32 scales on one CUDA device expected");
    const Raw raw;
    const c10::cuda::CUDAGuard guard(r.q.device());
    const Tensor out = at::empty(sizes, r.q.options().dtype(type));
    require_matrix(out);
    const Matrix m = matrix(out);
    if (m.rows == 0 || m.cols == 0) return out;
    const Tensor q = r.q.contiguous(), scale = r.scale.contiguous();
    require(q.numel() == m.rows * tango_rows8_ld(m.cols, group) && scale.numel() == m.rows * ((m.cols + group - 1) / group),
            "codes and scales do not belong to this shape");
    check(tango_rows8_unpack(ptr<int8_t>(q), ptr<float>(scale), m.rows, m.cols, group, type_code(out), ptr(out), m.ld, cuda_stream()),
          "unpack8");
    count(1);
    return out;
}

// ------------------------------------------------------------------------------------------------ activations
struct Activation8Backward : SavingNode {
    std::string name() const override { return "Activation8Backward"; }
    int act = 0;
    int64_t group = 0;
    std::vector<int64_t> sizes;
    at::ScalarType type = at::kFloat;
    variable_list backward(const variable_list &grads) override {
        const std::vector<Tensor> k = kept();
        if (!grads[0].defined() || !needs(0)) return variable_list(1);
        const c10::cuda::CUDAGuard guard(grads[0].device());
        const Matrix dy = matrix(grads[0].to(type));
        const Tensor dx = at::empty(sizes, grads[0].options().dtype(type));
        if (dx.numel() == 0) return {dx};
        const Tensor q = k[0].contiguous(), scale = numbers(k[1]);
        check(tango_act8_backward(act, ptr<int8_t>(q), ptr<float>(scale), dy.rows, dy.cols, group, type_code(dx), ptr(dy.t), dy.ld,
                                  ptr(dx), std::max<int64_t>(dy.cols, 1), cuda_stream()), "activation8_backward");
        count(1);
        return {dx};
    }
};

Tensor activation8_fn(const Tensor &x_, int act, int64_t group) {
    require_matrix(x_);
    require_group(group);
    Tensor y;
    Rows8 copy;
    const bool saves = torch::autograd::compute_requires_grad(x_);
    {
        const Raw raw;
        const c10::cuda::CUDAGuard guard(x_.device());
        const Matrix x = matrix(x_);
        y = at::empty(x_.sizes(), x_.options());
        if (saves) copy = alloc_rows8(x.rows, x.cols, group, x_);
        if (y.numel() > 0) {
            const int mode = settings().mode_quantize;
            const uint64_t call = saves && mode == TANGO_ROUND_STOCHASTIC ? next_call() : 0;
            const tango_rows8_job job{ptr(x.t), x.ld, ptr<int8_t>(copy.q), ptr<float>(copy.scale), 1, 0};
            check(tango_act8_forward(act, &job, x.rows, x.cols, group, type_code(x_), ptr(y), x.cols, mode, settings().seed, call,
                                     settings().step, cuda_stream()), "activation8");
            count(1);
        }
    }
    if (auto node = make_node<Activation8Backward>(x_)) {
        node->act = act; node->group = group; node->sizes = x_.sizes().vec(); node->type = x_.scalar_type();
        torch::autograd::set_history(y, node);
        node->keep({copy.q, bytes(copy.scale)});
    }
    return y;
}

// ------------------------------------------------------------------------------------------------ edge attention
// The row schedule of one direction and the workspace of its long rows.
struct EdgePlan {
    tango_edge_plan p{};
    Tensor ws;
    bool present = false;
    const tango_edge_plan *get() const { return present ? &p : nullptr; }
    int64_t bytes() const { return ws.defined() ? ws.numel() : 0; }
    int launches() const { return p.n_heavy > 0 ? 2 : 1; }
};
static EdgePlan edge_plan(const EdgeSchedule &s, int pass, int heads, int d, const Tensor &like) {
    EdgePlan plan;
    plan.present = s.present;
    if (!plan.present) return plan;
    plan.p.rows = ptr<int32_t>(s.rows); plan.p.n_long = s.n_long;
    if (s.n_heavy == 0) return plan;
    plan.p.units = ptr<int32_t>(s.units); plan.p.n_units = s.n_units;
    plan.p.heavy_first = ptr<int32_t>(s.heavy_first); plan.p.n_heavy = s.n_heavy;
    plan.ws = at::empty({tango_edge_attention_workspace_bytes(pass, s.n_units, heads, d)}, like.options().dtype(at::kByte));
    return plan;
}
static const int32_t *index_ptr(const Direction &d) { return ptr<int32_t>(d.indices.numel() > 0 ? d.indices : d.indptr); }
static tango_rows8 view(const Rows8 &r) { return {ptr<int8_t>(r.q), ptr<float>(r.scale)}; }

struct EdgeAttentionBackward : SavingNode {
    std::string name() const override { return "EdgeAttentionBackward"; }
    GraphPtr g;
    int heads = 0, d = 0;
    float scale = 1.f;
    at::ScalarType type = at::kFloat;
    variable_list backward(const variable_list &grads) override {
        const std::vector<Tensor> k = kept();
        if (!grads[0].defined()) return variable_list(3);
        const Tensor grad = grads[0].to(type);
        const c10::cuda::CUDAGuard guard(grad.device());
        const Tensor q8 = k[0].contiguous(), kv8 = k[1].contiguous();
        const Tensor sq = numbers(k[2]), skv = numbers(k[3]), stats = numbers(k[4]);
        const int64_t n = g->n_nodes;
        const auto out = [&] { return at::empty({n, heads, d}, grad.options()); };
        const Tensor dq = out();
        if (n == 0) return {dq, out(), out()};
        const Rows8 o8 = pack_all({grad}, d)[0];
        const bool sources = needs(1) || needs(2);
        Tensor record, qo8;       // what the second pass reads of a destination
        if (sources) {
            record = at::empty({n, heads, 4}, grad.options().dtype(at::kFloat));
            qo8 = at::empty_like(kv8);
        }
        tango_edge_operands x{ptr<int8_t>(q8), ptr<int8_t>(kv8), ptr<int8_t>(o8.q), ptr<float>(sq), ptr<float>(skv),
                              ptr<float>(o8.scale)};
        const int code = type_code(grad);
        {
            const Direction &in = g->dir(false);
            const EdgePlan plan = edge_plan(in.edge_sched, 1, heads, d, grad);
            check(tango_edge_attention_bwd_dst(ptr<int32_t>(in.indptr), index_ptr(in), n, plan.get(), heads, d, &x, scale,
                                               ptr<float>(stats), ptr(dq), code, ptr<float>(record), ptr<int8_t>(qo8), ptr(plan.ws),
                                               plan.bytes(), cuda_stream()), "edge_attention_bwd_dst");
            count(plan.launches());
        }
        if (!sources) return {dq, Tensor(), Tensor()};
        const Tensor dk = out(), dv = out();
        const Direction &from = g->dir(true);
        const EdgePlan plan = edge_plan(from.edge_sched, 2, heads, d, grad);
        check(tango_edge_attention_bwd_src(ptr<int32_t>(from.indptr), index_ptr(from), n, plan.get(), heads, d, ptr<int8_t>(kv8),
                                           ptr<float>(skv), ptr<int8_t>(qo8), ptr<float>(record), ptr(dk), ptr(dv), code, ptr(plan.ws), plan.bytes(), cuda_stream()),
              "edge_attention_bwd_src");
        count(plan.launches());
        return {needs(0) ? dq : Tensor(), needs(1) ? dk : Tensor(), needs(2) ? dv : Tensor()};
    }
};

static void require_heads(const Tensor &t) {
    require(t.dim() == 3, "[rows, heads, width] expected");
    require(t.size(1) >= 1 && t.size(1) <= 65535 && t.size(2) >= 1 && t.size(2) <= kMaxHeadWidth, "1 to 65535 heads of width 1 to 512 expected");
}

Tensor edge_attention_fn(const GraphPtr &g, const Tensor &q, const Tensor &k, const Tensor &v, double scale) {
    require_heads(q);
    for (const Tensor *t : {&q, &k, &v}) {
        require_matrix(*t);
        require(t->sizes() == q.sizes() && t->scalar_type() == q.scalar_type() && t->device() == q.device(),
                "q, k and v of one shape, type and device expected");
    }
    require(q.size(0) == g->n_nodes, "one row of q, k and v per node expected");
    require(g->csc->indptr.device() == q.device(), "graph and features must be on the same GPU");
    require(std::isfinite(scale), "finite scale expected");
    const int heads = (int)q.size(1), d = (int)q.size(2);
    const bool saves = torch::autograd::compute_requires_grad(q, k, v);
    Tensor out, stats;
    std::vector<Rows8> r;
    {
        const Raw raw;
        const c10::cuda::CUDAGuard guard(q.device());
        out = at::empty(q.sizes(), q.options().memory_format(at::MemoryFormat::Contiguous));
        r = pack_all({q, k, v}, d, true);
        if (saves) stats = floats({q.size(0), heads, 2}, q);
        if (q.size(0) > 0) {
            const Direction &in = g->dir(false);
            const EdgePlan plan = edge_plan(in.edge_sched, 0, heads, d, q);
            const tango_edge_operands x{ptr<int8_t>(r[0].q), ptr<int8_t>(r[1].q), nullptr, ptr<float>(r[0].scale),
                                        ptr<float>(r[1].scale), nullptr};
            check(tango_edge_attention(ptr<int32_t>(in.indptr), index_ptr(in), q.size(0), plan.get(), heads, d, &x, (float)scale, ptr(out),
                                       type_code(q), ptr<float>(stats), ptr(plan.ws), plan.bytes(), cuda_stream()),
                  "edge_attention");
            count(plan.launches());
        }
    }
    if (auto node = make_node<EdgeAttentionBackward>(q, k, v)) {
        node->g = g; node->heads = heads; node->d = d; node->scale = (float)scale; node->type = q.scalar_type();
        torch::autograd::set_history(out, node);
        node->keep({r[0].q, r[1].q, bytes(r[0].scale), bytes(r[1].scale), bytes(stats)});
    }
    return out;
}

Tensor edge_attention_rows(const GraphPtr &g, const Tensor &rows_, const Tensor &q, const Rows8 &k, const Rows8 &v, double scale) {
    require_heads(q);
    require_matrix(q);
    require(!torch::autograd::compute_requires_grad(q), "edge_attention_rows has no gradient: call it under torch.no_grad()");
    require(rows_.dim() == 1 && rows_.size(0) == q.size(0) && (rows_.scalar_type() == at::kLong || rows_.scalar_type() == at::kInt),
            "one int32 or int64 node id per query expected");
    require(g->csc->indptr.device() == q.device() && rows_.device() == q.device(), "graph, rows and queries must be on the same GPU");
    const int64_t heads = q.size(1), d = q.size(2), r = q.size(0), n = g->n_nodes;
    for (const Rows8 *t : {&k, &v}) {
        require(t->q.device() == q.device() && t->scale.device() == q.device(), "keys and values must be on the GPU of the queries");
        require(t->q.dim() == 2 && t->q.size(0) == n && t->q.size(1) == tango_rows8_ld(heads * d, d) && t->scale.numel() == n * heads,
                "keys and values packed with one row per node and one group per head expected");
    }
    require(std::isfinite(scale), "finite scale expected");
    const Raw raw;
    const c10::cuda::CUDAGuard guard(q.device());
    const Tensor out = at::empty(q.sizes(), q.options().memory_format(at::MemoryFormat::Contiguous));
    if (r == 0) return out;
    const Tensor rows = rows_.to(at::kLong).contiguous();
    const Matrix qm = matrix(q);
    const Direction &in = g->dir(false);
    const int splits = tango_edge_attention_rows_splits(r, in.edge_sched.present ? in.edge_sched.longest : g->n_edges());
    const int64_t bytes = tango_edge_attention_rows_workspace_bytes(r, splits, (int)heads, (int)d);
    if (bytes < 0) check((int)bytes, "edge_attention_rows");
    const Tensor ws = at::empty({bytes}, q.options().dtype(at::kByte));
    const int mode = settings().mode_quantize;
    const uint64_t call = mode == TANGO_ROUND_STOCHASTIC ? next_call() : 0;
    const tango_rows8 k8 = view(k), v8 = view(v);
    check(tango_edge_attention_rows(ptr<int32_t>(in.indptr), index_ptr(in), n, ptr<int64_t>(rows), r, splits, (int)heads, (int)d, ptr(qm.t),
                                    qm.ld, type_code(q), &k8, &v8, (float)scale, ptr(out), ptr(ws), bytes, mode, settings().seed, call,
                                    settings().step, cuda_stream()), "edge_attention_rows");
    count(splits > 1 ? 2 : 1);
    return out;
}

}  // namespace tango_host
