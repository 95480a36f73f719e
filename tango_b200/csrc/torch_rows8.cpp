// 8-bit rows and what reads them, over at::Tensor, with autograd nodes.  What a node keeps -- codes, scales, softmax statistics
// -- is one allocation of bytes, a saved tensor like any other (an allocation and a saved variable cost about a microsecond
// each, which a small graph's pass notices).
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

// Several arrays in one allocation, each on a 256-byte boundary.
struct Layout {
    int64_t bytes = 0;
    int64_t add(int64_t n) {
        const int64_t at = bytes;
        bytes += (n + 255) / 256 * 256;
        return at;
    }
};
static Tensor allocate(const Layout &l, const Tensor &like) { return at::empty({l.bytes}, like.options().dtype(at::kByte)); }
template <class T>
static T *part(const Tensor &t, int64_t at) {
    return reinterpret_cast<T *>(static_cast<char *>(t.data_ptr()) + at);
}

// The call number of a pack of n matrices: each draws with a number of its own when rounding is stochastic.
static uint64_t calls_of(int mode, int n) {
    if (mode != TANGO_ROUND_STOCHASTIC) return 0;
    const uint64_t call = next_call();
    for (int k = 1; k < n; ++k) next_call();
    return call;
}
static void pack(const tango_rows8_job *jobs, int n, const Matrix &x, int64_t group) {
    const int mode = settings().mode_quantize;
    check(tango_rows8_pack(jobs, n, x.rows, x.cols, group, type_code(x.t), mode, settings().seed, calls_of(mode, n), settings().step,
                           cuda_stream()), "pack8");
    count(1);
}

Rows8 pack8(const Tensor &x, int64_t group) {
    require_matrix(x);
    require_group(group);
    const Raw raw;
    const c10::cuda::CUDAGuard guard(x.device());
    const Matrix m = matrix(x);
    const int64_t groups = (m.cols + group - 1) / group;
    const Rows8 out{at::empty({m.rows, tango_rows8_ld(m.cols, group)}, x.options().dtype(at::kChar)),
                    at::empty({m.rows, groups}, x.options().dtype(at::kFloat))};
    if (m.rows == 0 || m.cols == 0) return out;
    const tango_rows8_job job{ptr(m.t), m.ld, ptr<int8_t>(out.q), ptr<float>(out.scale), 1, 0};
    pack(&job, 1, m, group);
    return out;
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
// What an activation keeps of a matrix: codes, then scales.
struct Copy8 {
    Layout l;
    int64_t codes, scales;
    Copy8(int64_t rows, int64_t cols, int64_t group)
        : codes(l.add(rows * tango_rows8_ld(cols, group))), scales(l.add(rows * ((cols + group - 1) / group) * 4)) {}
};

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
        const Tensor copy = k[0].contiguous();
        const Copy8 at(dy.rows, dy.cols, group);
        check(tango_act8_backward(act, part<int8_t>(copy, at.codes), part<float>(copy, at.scales), dy.rows, dy.cols, group,
                                  type_code(dx), ptr(dy.t), dy.ld, ptr(dx), dy.cols, cuda_stream()), "activation8_backward");
        count(1);
        return {dx};
    }
};

Tensor activation8_fn(const Tensor &x_, int act, int64_t group) {
    require_matrix(x_);
    require_group(group);
    Tensor y, copy;
    auto node = make_node<Activation8Backward>(x_);
    {
        const Raw raw;
        const c10::cuda::CUDAGuard guard(x_.device());
        const Matrix x = matrix(x_);
        const Copy8 at(x.rows, x.cols, group);
        y = at::empty(x_.sizes(), x_.options());
        if (node) copy = allocate(at.l, x_);
        if (y.numel() > 0) {
            const int mode = settings().mode_quantize;
            tango_rows8_job job{ptr(x.t), x.ld, nullptr, nullptr, 1, 0};
            if (node) { job.q = part<int8_t>(copy, at.codes); job.scales = part<float>(copy, at.scales); }
            check(tango_act8_forward(act, &job, x.rows, x.cols, group, type_code(x_), ptr(y), x.cols, mode, settings().seed,
                                     node ? calls_of(mode, 1) : 0, settings().step, cuda_stream()), "activation8");
            count(1);
        }
    }
    if (node) {
        node->act = act; node->group = group; node->sizes = x_.sizes().vec(); node->type = x_.scalar_type();
        torch::autograd::set_history(y, node);
        node->keep({copy});
    }
    return y;
}

// ------------------------------------------------------------------------------------------------ edge attention
// The row schedule of one direction.
struct EdgePlan {
    tango_edge_plan p{};
    bool present;
    EdgePlan(const EdgeSchedule &s) : present(s.present) {
        if (!present) return;
        p.rows = ptr<int32_t>(s.rows); p.n_long = s.n_long;
        p.units = ptr<int32_t>(s.units); p.n_units = s.n_units;
        p.heavy_first = ptr<int32_t>(s.heavy_first); p.n_heavy = s.n_heavy;
    }
    const tango_edge_plan *get() const { return present ? &p : nullptr; }
    int64_t workspace(int pass, int heads, int d) const { return tango_edge_attention_workspace_bytes(pass, p.n_units, heads, d); }
    int launches() const { return p.n_heavy > 0 ? 2 : 1; }
};
static const int32_t *index_ptr(const Direction &d) { return ptr<int32_t>(d.indices.numel() > 0 ? d.indices : d.indptr); }

// What the forward pass keeps: the 8-bit operands and the softmax statistics.
struct Kept8 {
    Layout l;
    int64_t q, kv, sq, skv, stats;
    Kept8(int64_t n, int64_t heads, int64_t d) {
        const int64_t ld = tango_rows8_ld(heads * d, d);
        q = l.add(n * ld); kv = l.add(2 * n * ld); sq = l.add(4 * n * heads); skv = l.add(8 * n * heads); stats = l.add(8 * n * heads);
    }
    tango_edge_operands operands(const Tensor &t) const {
        return {part<int8_t>(t, q), part<int8_t>(t, kv), nullptr, part<float>(t, sq), part<float>(t, skv), nullptr};
    }
};

struct EdgeAttentionBackward : SavingNode {
    std::string name() const override { return "EdgeAttentionBackward"; }
    GraphPtr g;
    int heads = 0, d = 0;
    float scale = 1.f;
    at::ScalarType type = at::kFloat;
    variable_list backward(const variable_list &grads) override {
        const std::vector<Tensor> k = kept();
        if (!grads[0].defined()) return variable_list(3);
        const Matrix grad = matrix(grads[0].to(type));
        const c10::cuda::CUDAGuard guard(grad.t.device());
        const int64_t n = g->n_nodes, ld = tango_rows8_ld((int64_t)heads * d, d);
        const auto out = [&] { return at::empty({n, heads, d}, grad.t.options()); };
        const Tensor dq = out();
        if (n == 0) return {dq, out(), out()};
        const Tensor saved = k[0].contiguous();
        const Kept8 in(n, heads, d);
        const bool sources = needs(1) || needs(2);
        const Direction &to = g->dir(false), &from = g->dir(true);
        const EdgePlan by_dst(to.edge_sched), by_src(from.edge_sched);
        // the gradient in 8 bits, what the second pass reads of a destination, and the workspace, which the passes share
        Layout l;
        const int64_t o = l.add(n * ld), so = l.add(4 * n * heads), record = l.add(sources ? 16 * n * heads : 0),
                      qo = l.add(sources ? 2 * n * ld : 0), ws_bytes = std::max(by_dst.workspace(1, heads, d), by_src.workspace(2, heads, d)),
                      ws = l.add(ws_bytes);
        const Tensor scratch = allocate(l, grad.t);
        const tango_rows8_job job{ptr(grad.t), grad.ld, part<int8_t>(scratch, o), part<float>(scratch, so), 1, 0};
        pack(&job, 1, grad, d);
        tango_edge_operands x = in.operands(saved);
        x.o = part<int8_t>(scratch, o); x.so = part<float>(scratch, so);
        const int code = type_code(grad.t);
        check(tango_edge_attention_bwd_dst(ptr<int32_t>(to.indptr), index_ptr(to), n, by_dst.get(), heads, d, &x, scale,
                                           part<float>(saved, in.stats), ptr(dq), code, sources ? part<float>(scratch, record) : nullptr,
                                           sources ? part<int8_t>(scratch, qo) : nullptr, part<void>(scratch, ws), ws_bytes,
                                           cuda_stream()), "edge_attention_bwd_dst");
        count(by_dst.launches());
        if (!sources) return {dq, Tensor(), Tensor()};
        const Tensor dk = out(), dv = out();
        check(tango_edge_attention_bwd_src(ptr<int32_t>(from.indptr), index_ptr(from), n, by_src.get(), heads, d, x.kv, x.skv,
                                           part<int8_t>(scratch, qo), part<float>(scratch, record), ptr(dk), ptr(dv), code,
                                           part<void>(scratch, ws), ws_bytes, cuda_stream()), "edge_attention_bwd_src");
        count(by_src.launches());
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
    require(std::isfinite((float)scale), "finite scale expected");
    const int heads = (int)q.size(1), d = (int)q.size(2);
    const int64_t n = q.size(0);
    Tensor out, saved;
    auto node = make_node<EdgeAttentionBackward>(q, k, v);
    {
        const Raw raw;
        const c10::cuda::CUDAGuard guard(q.device());
        out = at::empty(q.sizes(), q.options().memory_format(at::MemoryFormat::Contiguous));
        const Direction &in = g->dir(false);
        const EdgePlan plan(in.edge_sched);
        Kept8 at(n, heads, d);
        const int64_t ws_bytes = plan.workspace(0, heads, d);
        Tensor ws;
        int64_t ws_at = 0;
        if (node) ws = at::empty({ws_bytes}, q.options().dtype(at::kByte));
        else ws_at = at.l.add(ws_bytes);
        saved = allocate(at.l, q);
        if (!node) ws = saved;
        if (n > 0) {
            const Matrix m[3] = {matrix(q), matrix(k), matrix(v)};
            const tango_edge_operands x = at.operands(saved);
            const int64_t run = tango_rows8_run(d);
            int8_t *kv = part<int8_t>(saved, at.kv);
            float *skv = part<float>(saved, at.skv);
            const tango_rows8_job jobs[3] = {{ptr(m[0].t), m[0].ld, part<int8_t>(saved, at.q), part<float>(saved, at.sq), 1, 0},
                                             {ptr(m[1].t), m[1].ld, kv, skv, 2, 1}, {ptr(m[2].t), m[2].ld, kv + run, skv + 1, 2, 1}};
            pack(jobs, 3, m[0], d);
            check(tango_edge_attention(ptr<int32_t>(in.indptr), index_ptr(in), n, plan.get(), heads, d, &x, (float)scale, ptr(out),
                                       type_code(q), node ? part<float>(saved, at.stats) : nullptr, part<void>(ws, ws_at), ws_bytes,
                                       cuda_stream()), "edge_attention");
            count(plan.launches());
        }
    }
    if (node) {
        node->g = g; node->heads = heads; node->d = d; node->scale = (float)scale; node->type = q.scalar_type();
        torch::autograd::set_history(out, node);
        node->keep({saved});
    }
    return out;
}

static tango_rows8 view(const Rows8 &r) { return {ptr<int8_t>(r.q), ptr<float>(r.scale)}; }

Tensor edge_attention_rows(const GraphPtr &g, const Tensor &rows_, const Tensor &q, const Rows8 &k_, const Rows8 &v_, double scale) {
    // the kernel takes bare pointers: nothing but int8 codes and fp32 scales, dense, reaches it
    for (const Rows8 *t : {&k_, &v_})
        require(t->q.scalar_type() == at::kChar && t->scale.scalar_type() == at::kFloat, "keys and values of int8 codes and fp32 scales expected");
    require_heads(q);
    require_matrix(q);
    require(!torch::autograd::compute_requires_grad(q), "edge_attention_rows has no gradient: call it under torch.no_grad()");
    require(rows_.dim() == 1 && rows_.size(0) == q.size(0) && (rows_.scalar_type() == at::kLong || rows_.scalar_type() == at::kInt),
            "one int32 or int64 node id per query expected");
    require(g->csc->indptr.device() == q.device() && rows_.device() == q.device(), "graph, rows and queries must be on the same GPU");
    const int64_t heads = q.size(1), d = q.size(2), r = q.size(0), n = g->n_nodes;
    for (const Rows8 *t : {&k_, &v_}) {
        require(t->q.device() == q.device() && t->scale.device() == q.device(), "keys and values must be on the GPU of the queries");
        // (pack8 of a tensor without rows has no columns either)
        require(t->q.dim() == 2 && t->q.size(0) == n && t->scale.dim() == 2 && t->scale.size(0) == n &&
                    (n == 0 || (t->q.size(1) == tango_rows8_ld(heads * d, d) && t->scale.size(1) == heads)),
                "keys and values packed with one row per node and one group per head expected");
    }
    require(std::isfinite((float)scale), "finite scale expected");
    const Raw raw;
    const c10::cuda::CUDAGuard guard(q.device());
    const Rows8 k{k_.q.contiguous(), k_.scale.contiguous()}, v{v_.q.contiguous(), v_.scale.contiguous()};
    const Tensor out = at::empty(q.sizes(), q.options().memory_format(at::MemoryFormat::Contiguous));
    if (r == 0) return out;
    const Tensor rows = rows_.to(at::kLong).contiguous();
    const Matrix qm = matrix(q);
    const Direction &in = g->dir(false);
    const int splits = tango_edge_attention_rows_splits(r, g->longest >= 0 ? g->longest : g->n_edges());
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
