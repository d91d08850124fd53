// Symbolic reverse-mode autodiff: emits the backward pass as graph nodes so the
// gradient computation is scheduled, fused, memory-planned and run on the GPU like
// any forward graph.
//
// The vector-Jacobian products and their evaluation order restate the reference's
// eager Autodiff::compute_gradients (src/autodiff/gradient.cpp:52-332): nodes are
// visited in reverse topological order, contributions are accumulated with add in
// that order, and unbroadcast (gradient.cpp:10-50) sums leading axes, then
// singleton axes, then reshapes.  Ops the reference lacks (exp, neg, tanh, step,
// reshape, expand) get their standard derivatives.
#include <algorithm>
#include <cmath>
#include <unordered_map>

#include "ttb.hpp"

namespace ttb {

namespace {

struct Builder {
    Graph& g;

    int mk(int op, std::vector<int> in) {
        Node n;
        n.op = op;
        n.dtype = g.nodes[static_cast<size_t>(in[0])].dtype;
        n.in = std::move(in);
        n.id = g.next_id;
        infer_shape(g, n);
        return g.add(std::move(n));
    }
    int constant(std::vector<float> values, Shape s, int dtype) {
        Node n;
        n.op = TT_OP_CONSTANT;
        n.dtype = dtype;
        n.shape = std::move(s);
        n.cdata = std::move(values);
        n.id = g.next_id;
        return g.add(std::move(n));
    }
    int scalar(float v, int dtype) { return constant({v}, {}, dtype); }
    int view(int op, int a, const Shape s) {
        const Node& an = g.nodes[static_cast<size_t>(a)];
        if (an.shape == s) return a;
        Node n;
        n.op = op;
        n.dtype = an.dtype;
        n.in = {a};
        n.shape = s;
        n.id = g.next_id;
        return g.add(std::move(n));
    }
    int transpose(int a, int64_t d0, int64_t d1) {
        Node n;
        n.op = TT_OP_TRANSPOSE;
        n.dtype = g.nodes[static_cast<size_t>(a)].dtype;
        n.in = {a};
        n.dim0 = d0;
        n.dim1 = d1;
        n.id = g.next_id;
        infer_shape(g, n);
        return g.add(std::move(n));
    }
    int reduce_sum(int a, std::vector<int64_t> axes, bool keepdims) {
        Node n;
        n.op = TT_OP_REDUCE_SUM;
        n.dtype = g.nodes[static_cast<size_t>(a)].dtype;
        n.in = {a};
        n.axes = std::move(axes);
        n.keepdims = keepdims;
        n.id = g.next_id;
        infer_shape(g, n);
        return g.add(std::move(n));
    }
    Shape shape(int a) const { return g.nodes[static_cast<size_t>(a)].shape; }  // by value: g.nodes grows
    int dtype(int a) const { return g.nodes[static_cast<size_t>(a)].dtype; }

    // Autodiff::unbroadcast (gradient.cpp:10-50).
    int unbroadcast(int grad, const Shape target) {
        if (shape(grad) == target) return grad;
        if (target.empty()) return reduce_sum(grad, {}, false);
        int cur = grad;
        size_t gr = shape(grad).size(), tr = target.size();
        if (gr > tr) {
            std::vector<int64_t> lead;
            for (size_t i = 0; i < gr - tr; ++i) lead.push_back(static_cast<int64_t>(i));
            cur = reduce_sum(cur, lead, false);
        }
        std::vector<int64_t> single;
        for (size_t i = 0; i < tr; ++i)
            if (target[i] == 1 && shape(cur)[i] > 1) single.push_back(static_cast<int64_t>(i));
        if (!single.empty()) cur = reduce_sum(cur, single, true);
        if (shape(cur) != target) cur = view(TT_OP_RESHAPE, cur, target);
        return cur;
    }

    // Reduced axes replaced by 1, so the gradient broadcasts back (gradient.cpp:262-324).
    Shape kept_shape(const Node& red, const Shape& in_shape) {
        auto ax = normalized_axes(red, static_cast<int64_t>(in_shape.size()));
        Shape s;
        for (size_t i = 0; i < in_shape.size(); ++i)
            s.push_back(std::binary_search(ax.begin(), ax.end(), static_cast<int64_t>(i)) ? 1 : in_shape[i]);
        return s;
    }
};

}  // namespace

void append_gradients(Graph& g, int loss, const std::vector<int>& wrt, int seed) {
    if (loss < 0 || static_cast<size_t>(loss) >= g.nodes.size()) fail(TT_ERR_INVALID, "loss node out of range");
    if (seed != -1) {
        if (seed < 0 || static_cast<size_t>(seed) >= g.nodes.size()) fail(TT_ERR_INVALID, "seed node out of range");
        if (g.nodes[static_cast<size_t>(seed)].shape != g.nodes[static_cast<size_t>(loss)].shape)
            fail(TT_ERR_SHAPE, "the seed must have the loss's shape " + shape_str(g.nodes[static_cast<size_t>(loss)].shape) +
                                   ", got " + shape_str(g.nodes[static_cast<size_t>(seed)].shape));
        if (g.nodes[static_cast<size_t>(seed)].dtype != g.nodes[static_cast<size_t>(loss)].dtype)
            fail(TT_ERR_TYPE, "the seed must have the loss's dtype");
    }
    for (int w : wrt)
        if (w >= 0 && static_cast<size_t>(w) < g.nodes.size() && g.nodes[static_cast<size_t>(w)].dtype == TT_INT32)
            fail(TT_ERR_TYPE, "token ids have no gradient");
    const size_t nfwd = static_cast<size_t>(loss) + 1;  // nodes after the loss cannot reach it
    Builder b{g};
    std::unordered_map<int, int> grads;
    auto accumulate = [&](int target, int contrib) {
        auto it = grads.find(target);
        if (it == grads.end())
            grads[target] = contrib;
        else
            it->second = b.mk(TT_OP_ADD, {it->second, contrib});
    };

    // Gradients of scan states: of a whole GatedScan (grads) and of its last state alone
    // (last_grads), which enters the same backward scan as its first carry.
    std::unordered_map<int, int> last_grads;
    auto backward = [&](int op, std::vector<int> in, int64_t axis, std::vector<int64_t> has, std::vector<float> attr,
                        int64_t split = 0) {
        Node q;
        q.dim1 = split;
        q.op = op;
        q.in = std::move(in);
        q.dim0 = axis;
        q.axes = std::move(has);
        q.attr = std::move(attr);
        q.id = g.next_id;
        infer_shape(g, q);
        return g.add(std::move(q));
    };

    // Seed dL/dL = ones(loss.shape) (gradient.cpp:131), or the caller's seed.
    if (seed >= 0) {
        grads[loss] = seed;
    } else {
        int one = b.scalar(1.0f, b.dtype(loss));
        grads[loss] = b.view(TT_OP_EXPAND, one, b.shape(loss));
    }

    for (size_t ii = nfwd; ii-- > 0;) {
        int i = static_cast<int>(ii);
        auto git = grads.find(i);
        const auto lit = last_grads.find(i);
        if (git == grads.end() && lit == last_grads.end()) continue;
        const int gidx = git == grads.end() ? -1 : git->second;  // -1: a scan reached through its last state only
        const Node n = g.nodes[ii];  // copy: g.nodes grows below
        const int dt = n.dtype;
        switch (n.op) {
            case TT_OP_INPUT:
            case TT_OP_CONSTANT:
            case TT_OP_STEP:
                break;
            case TT_OP_ADD:
                accumulate(n.in[0], b.unbroadcast(gidx, b.shape(n.in[0])));
                accumulate(n.in[1], b.unbroadcast(gidx, b.shape(n.in[1])));
                break;
            case TT_OP_SUB: {
                accumulate(n.in[0], b.unbroadcast(gidx, b.shape(n.in[0])));
                int neg = b.mk(TT_OP_MUL, {gidx, b.scalar(-1.0f, dt)});
                accumulate(n.in[1], b.unbroadcast(neg, b.shape(n.in[1])));
                break;
            }
            case TT_OP_MUL: {
                int ga = b.mk(TT_OP_MUL, {gidx, n.in[1]});
                int gb = b.mk(TT_OP_MUL, {gidx, n.in[0]});
                accumulate(n.in[0], b.unbroadcast(ga, b.shape(n.in[0])));
                accumulate(n.in[1], b.unbroadcast(gb, b.shape(n.in[1])));
                break;
            }
            case TT_OP_DIV: {
                int ga = b.mk(TT_OP_DIV, {gidx, n.in[1]});
                accumulate(n.in[0], b.unbroadcast(ga, b.shape(n.in[0])));
                int bsq = b.mk(TT_OP_MUL, {n.in[1], n.in[1]});
                int negg = b.mk(TT_OP_MUL, {gidx, b.scalar(-1.0f, dt)});
                int negga = b.mk(TT_OP_MUL, {negg, n.in[0]});
                int gb = b.mk(TT_OP_DIV, {negga, bsq});
                accumulate(n.in[1], b.unbroadcast(gb, b.shape(n.in[1])));
                break;
            }
            case TT_OP_RELU: {
                int mask = b.mk(TT_OP_STEP, {n.in[0]});
                accumulate(n.in[0], b.mk(TT_OP_MUL, {gidx, mask}));
                break;
            }
            case TT_OP_SIGMOID: {
                int oms = b.mk(TT_OP_SUB, {b.view(TT_OP_EXPAND, b.scalar(1.0f, dt), n.shape), i});
                int ds = b.mk(TT_OP_MUL, {i, oms});
                accumulate(n.in[0], b.mk(TT_OP_MUL, {gidx, ds}));
                break;
            }
            case TT_OP_EXP:
                accumulate(n.in[0], b.mk(TT_OP_MUL, {gidx, i}));
                break;
            case TT_OP_NEG:
                accumulate(n.in[0], b.mk(TT_OP_NEG, {gidx}));
                break;
            case TT_OP_TANH: {
                int tt = b.mk(TT_OP_MUL, {i, i});
                int om = b.mk(TT_OP_SUB, {b.view(TT_OP_EXPAND, b.scalar(1.0f, dt), n.shape), tt});
                accumulate(n.in[0], b.mk(TT_OP_MUL, {gidx, om}));
                break;
            }
            case TT_OP_MATMUL: {
                int bt = b.transpose(n.in[1], -2, -1);
                int at = b.transpose(n.in[0], -2, -1);
                int ga = b.mk(TT_OP_MATMUL, {gidx, bt});
                int gb = b.mk(TT_OP_MATMUL, {at, gidx});
                accumulate(n.in[0], b.unbroadcast(ga, b.shape(n.in[0])));
                accumulate(n.in[1], b.unbroadcast(gb, b.shape(n.in[1])));
                break;
            }
            case TT_OP_TRANSPOSE:
                accumulate(n.in[0], b.transpose(gidx, n.dim0, n.dim1));
                break;
            case TT_OP_RESHAPE:
                accumulate(n.in[0], b.view(TT_OP_RESHAPE, gidx, b.shape(n.in[0])));
                break;
            case TT_OP_EXPAND:
                accumulate(n.in[0], b.unbroadcast(gidx, b.shape(n.in[0])));
                break;
            case TT_OP_REDUCE_SUM: {
                const Shape ash = b.shape(n.in[0]);
                int gs = n.keepdims ? gidx : b.view(TT_OP_RESHAPE, gidx, b.kept_shape(n, ash));
                accumulate(n.in[0], b.view(TT_OP_EXPAND, gs, ash));
                break;
            }
            case TT_OP_REDUCE_MEAN: {
                const Shape ash = b.shape(n.in[0]);
                int64_t gn = numel(b.shape(gidx));
                int64_t nred = numel(ash) / (gn > 0 ? gn : 1);
                if (nred <= 0) nred = 1;
                float factor = static_cast<float>(1.0 / static_cast<double>(nred));
                int scaled = b.mk(TT_OP_MUL, {gidx, b.scalar(factor, dt)});
                int gs = n.keepdims ? scaled : b.view(TT_OP_RESHAPE, scaled, b.kept_shape(n, ash));
                accumulate(n.in[0], b.view(TT_OP_EXPAND, gs, ash));
                break;
            }
            case TT_OP_SCAN_LAST: {
                auto l = last_grads.find(n.in[0]);
                if (l == last_grads.end()) last_grads[n.in[0]] = gidx;
                else l->second = b.mk(TT_OP_ADD, {l->second, gidx});
                break;
            }
            case TT_OP_GATED_SCAN: {
                // u[t] = g[t] + gate[t+1]*u[t+1] (g_last enters at the last step): dx = u,
                // dgate[t] = u[t]*h[t-1], dinit = gate[0]*u[0]
                std::vector<int> ops{n.in[0]};
                const bool has_last = lit != last_grads.end(), has_init = n.in.size() > 2;
                if (gidx >= 0) ops.push_back(gidx);
                if (has_last) ops.push_back(lit->second);
                const std::vector<int64_t> has{gidx >= 0, has_last, has_init};
                std::vector<int> gate_ops = ops;
                gate_ops.push_back(i);
                if (has_init) gate_ops.push_back(n.in[2]);
                // A gate shared by adjacent lanes (a head's channels): its gradient is summed over them in
                // the scan's launch, not stored in full and reduced.
                int gate = n.in[0];
                int64_t split = 0;
                {
                    const Node& e = g.nodes[static_cast<size_t>(gate)];
                    const Shape src = e.op == TT_OP_EXPAND ? b.shape(e.in[0]) : Shape{};
                    // (not where the expanded gate itself is a gradient target)
                    if (e.op == TT_OP_EXPAND && src.size() == e.shape.size() && std::find(wrt.begin(), wrt.end(), gate) == wrt.end()) {
                        size_t s = src.size();
                        while (s > static_cast<size_t>(n.dim0) + 1 && src[s - 1] == 1) --s;
                        const bool same = std::equal(src.begin(), src.begin() + static_cast<long>(s), e.shape.begin());
                        int64_t group = 1;
                        for (size_t d = s; d < src.size(); ++d) group *= e.shape[d];
                        if (same && group > 1) {
                            split = static_cast<int64_t>(s);
                            gate = e.in[0];
                        }
                    }
                }
                accumulate(gate, backward(BOP_SCAN_DGATE, gate_ops, n.dim0, has, {}, split));
                accumulate(n.in[1], backward(BOP_SCAN_DX, ops, n.dim0, has, {}));
                if (has_init) accumulate(n.in[2], backward(BOP_SCAN_DINIT, ops, n.dim0, has, {}));
                break;
            }
            case TT_OP_TOKEN_LOGPROB: case TT_OP_POLICY_LOSS: case TT_OP_PREFERENCE_LOSS: {
                // with respect to the logits; the other operands are data (constants)
                const int op = n.op == TT_OP_TOKEN_LOGPROB ? BOP_LOGPROB_GRAD
                               : n.op == TT_OP_POLICY_LOSS ? BOP_POLICY_GRAD : BOP_PREFERENCE_GRAD;
                std::vector<int> ops = n.in;
                ops.push_back(gidx);
                accumulate(n.in[0], backward(op, ops, 0, {}, n.attr));
                break;
            }
            case TT_OP_REDUCE_MAX:
                fail(TT_ERR_COMPILE, "reduce_max has no gradient in this backend");
            default:
                fail(TT_ERR_COMPILE, std::string("Unsupported op in backward pass: ") + op_name(n.op));
        }
    }

    for (int w : wrt) {
        if (w < 0 || static_cast<size_t>(w) >= nfwd) fail(TT_ERR_INVALID, "gradient target out of range");
        // A scan's states as the target: their last one's gradient is theirs too, at the axis's last step
        // (times 1 there and 0 before it: where it is not finite, so are its lane's steps before).
        const auto last = last_grads.find(w);
        if (last != last_grads.end()) {
            const Shape sh = b.shape(w);
            if (numel(sh) > 0) {
                const size_t axis = static_cast<size_t>(g.nodes[static_cast<size_t>(w)].dim0);
                Shape steps(sh.size(), 1), lane = sh;
                steps[axis] = sh[axis];
                lane[axis] = 1;
                std::vector<float> one(static_cast<size_t>(sh[axis]), 0.0f);
                one.back() = 1.0f;
                const int at = b.view(TT_OP_EXPAND, b.constant(std::move(one), steps, b.dtype(w)), sh);
                accumulate(w, b.mk(TT_OP_MUL, {b.view(TT_OP_EXPAND, b.view(TT_OP_RESHAPE, last->second, lane), sh), at}));
            }
            last_grads.erase(last);
        }
        auto it = grads.find(w);
        int out;
        if (it != grads.end()) {
            out = it->second;
        } else {
            out = b.view(TT_OP_EXPAND, b.scalar(0.0f, b.dtype(w)), b.shape(w));
        }
        // A gradient that is just a view of the seed or another value is still a
        // separate output buffer; the scheduler materialises views that are outputs.
        if (std::find(g.outputs.begin(), g.outputs.end(), out) != g.outputs.end() || out == w)
            out = b.view(TT_OP_RESHAPE, out, Shape{-1});  // placeholder fixed below
        g.outputs.push_back(out);
    }
    // Replace placeholders (reshape to [-1]) by a reshape to the node's own shape, which
    // the scheduler treats as a copy when the node is an output.
    for (int& o : g.outputs) {
        Node& n = g.nodes[static_cast<size_t>(o)];
        if (n.op == TT_OP_RESHAPE && n.shape.size() == 1 && n.shape[0] == -1)
            n.shape = g.nodes[static_cast<size_t>(n.in[0])].shape;
    }
}

}  // namespace ttb
