// Python entry points of the linear attention with a decay for each head and of what stands in front of it and behind it: rotary positions and the layer norm.
#include "block.h"

#include <optional>

namespace {

// ---- linear attention ------------------------------------------------------------------------------------------------------------------------
enum { LQ, LK, LV, LDECAY, LH0, LINEAR_INPUTS };

// Cuts long sequences into parts of `seg` tokens that run side by side, where there are too few chains (sequences x v-heads x kinds of results) for the SMs or where they fill
// them unevenly: the cheapest of all lengths of parts, against no cut, by what a stretch (128 tokens, in fp32 64) costs an SM in us (on the tensor cores more where all SMs draw on HBM and power than
// where few do).  A cut costs two more kernels, a pass over all parts but one that finds what they make of nothing (`kinds_before` of them), and the traffic of their states.
// In us, uncut / parts of so many stretches (what the rule takes in brackets), 128 channels: bf16 forward 32749 tokens x 32 heads 836 / 8 435 [29 378] 64 392; 8192 x 16 248 / [8 78] 16 118;
// 4096 x 2 113 / [2 32] 8 58; 2 x 2048 x 8 57 / [2 34] 4 40; 1024 x 16 [31] / 2 30; 8 x 4096 x 32 [257] / 16 410; backward 32749 x 32 [920] / 29 1019; 8192 x 16 244 / 8 183 [22 152];
// 4096 x 2 113 / [2 39] 8 64; 2 x 2048 x 8 [59] / 6 61; 4 x 1000 x 8 [35] / 4 82; fp32, parts of stretches of 64 tokens: forward 300 x 2 146 / [1 61];
// 700 x 2 [1 62] 2 101; 4096 x 8 1972 / [4 189] 16 668; 64 channels 4 x 1000 x 8 [2 74] 4 90; 2 x 700 x 2 [1 33] 2 50; forward and backward 16384 x 4 [1331] with parts of 64 allowed, 1600 without.
void cut_linear(MkdaSeqs& s, const Sequences& q, int64_t heads, int kinds, int kinds_before, int64_t K, int64_t V, at::ScalarType dt) {
    const bool tensor_cores = dt != at::kFloat && K % 8 == 0 && V % 8 == 0;
    const int64_t unit = dt == at::kFloat ? 64 : 128;      // tokens that parts are multiples of
    if (q.longest < 4 * unit || s.N == 0) return;
    const int64_t longest = (q.longest + unit - 1) / unit, most = std::max<int64_t>(longest, (s.TT + unit - 1) / unit), n_sm = sms(), state = heads * K * V;
    const double size = std::sqrt((double)K * V) / 128, launch = 16.0, state_us = 16.0 * K * V * kinds_before / 5e6;      // of a part and head
    const int64_t places = !tensor_cores && K <= 64 && V <= 64 ? 2 * n_sm : n_sm;      // narrow heads: two blocks to an SM, each half as slow again
    auto rounds = [&](int64_t items) { return (items + places - 1) / places; };
    auto shared = [&](int64_t items) { return places > n_sm && items > n_sm ? 1.5 : 1.0; };
    auto main = [&](int64_t items) { return !tensor_cores ? unit / 64 * 30.0 * size * shared(items) : items > n_sm / 2 ? 4.2 : 3.4; };
    auto before = [&](int64_t items) { return !tensor_cores ? unit / 64 * 11.0 * size * shared(items) : items > n_sm / 2 ? 1.9 : 1.4; };
    double best = std::max(longest * main(0), (double)most * heads * kinds / places * main(places));
    for (int64_t parts = 2; parts <= (tensor_cores ? (longest + 1) / 2 : longest); ++parts) {
        const int64_t seg = (longest + parts - 1) / parts, all = (most + seg - 1) / seg;      // parts with tokens, about
        if (s.N * parts * state * 4 > (int64_t)256 << 20) break;
        const int64_t items = all * heads * kinds, items_before = std::max<int64_t>(0, all - 1) * heads * kinds_before;
        const double us = (rounds(items) * main(items) + rounds(items_before) * before(items_before)) * seg + launch + (all + s.N) * heads * state_us + 0.002 * s.N * parts * heads;
        if (us < 0.97 * best) {
            best = us;
            s.seg = (int)(seg * unit);
            s.segs = (int)((longest + seg - 1) / seg);
        }
    }
}

// What a call hands to the library; the tensors behind the pointers are kept in `hold`.
struct LinearCall {
    MkdaLinearFwd p{};
    std::vector<Tensor> hold;
    LinearCall(const Sequences& q, const variable_list& t, double scale) {
        p.S = q.s; p.HK = (int)t[LQ].size(-2); p.HV = (int)t[LV].size(-2); p.K = (int)t[LQ].size(-1); p.V = (int)t[LV].size(-1);
        p.dtype = dtype_code(t[LQ]); p.scale = (float)scale;
        const bool tiles = t[LQ].scalar_type() != at::kFloat && p.K % 8 == 0 && p.V % 8 == 0;
        auto rows = [&](int i, const void*& ptr, long long& stride) {
            Rows r = rows_of(t[i], 2);
            // tiled copies want 16-byte boundaries and a stride that leads on: other rows are copied, so that results do not depend on where they lie
            const int64_t width = t[i].size(-1) * t[i].size(-2);
            if (tiles && (r.stride % 8 || r.stride < width || reinterpret_cast<uintptr_t>(r.t.data_ptr()) % 16)) r = {aligned(r.t), width};
            ptr = cptr(r.t);
            stride = r.stride;
            hold.push_back(r.t);
        };
        rows(LQ, p.q, p.q_stride); rows(LK, p.k, p.k_stride); rows(LV, p.v, p.v_stride);
        auto fp32 = [&](int i) {
            const Tensor v = param(t[i]);
            hold.push_back(v);
            return fptr(v);
        };
        p.log_decay = fp32(LDECAY);
        if ((int)t.size() > LH0) p.h0 = fp32(LH0);
    }
    Tensor parts(const at::Device& dev) const { return new_cuda({(int64_t)p.S.N * p.S.segs, p.HV, p.K, p.V}, at::kFloat, dev); }
};

variable_list linear_backward(const Sequences& q, double scale, const variable_list& s, const variable_list& grads) {
    reads_table(q);
    LinearCall call(q, s, scale);
    MkdaLinearBwd p{};
    const at::Device dev = s[LQ].device();
    cut_linear(call.p.S, q, call.p.HV, 3, 2, call.p.K, call.p.V, s[LQ].scalar_type());
    p.f = call.p;
    const Tensor dy = grads[0].defined() ? aligned(grads[0]) : at::zeros_like(s[LV], at::MemoryFormat::Contiguous);
    const Tensor dht = grads.size() > 1 && grads[1].defined() ? aligned(grads[1]) : Tensor();
    variable_list out(LINEAR_INPUTS);
    for (int i : {LQ, LK, LV}) out[i] = out_like(s[i], q.covers_all);
    if (s[LH0].defined()) out[LH0] = new_cuda(s[LH0].sizes(), at::kFloat, dev);
    Tensor seg_h, seg_g, part_q, part_k;
    if (p.f.S.seg) {
        seg_h = call.parts(dev);
        seg_g = call.parts(dev);
        p.f.seg_h = fmptr(seg_h); p.seg_g = fmptr(seg_g);
    }
    if (p.f.HV > p.f.HK) {
        part_q = new_cuda({(int64_t)q.s.TT, p.f.HV, p.f.K}, at::kFloat, dev);
        part_k = new_cuda({(int64_t)q.s.TT, p.f.HV, p.f.K}, at::kFloat, dev);
        p.part_q = fmptr(part_q); p.part_k = fmptr(part_k);
    }
    p.d_o = dy.data_ptr(); p.dht = fptr(dht); p.dq = out[LQ].data_ptr(); p.dk = out[LK].data_ptr(); p.dv = out[LV].data_ptr(); p.dh0 = fmptr(out[LH0]);
    p.end = (int)q.end;
    check_rc(mkda_linear_bwd(&p, stream()), "mkda_linear_bwd");
    return out;
}

// the checks that prompts and single tokens share; `lead` axes in front of the heads
PyObject* check_linear(const variable_list& t, int lead) {
    const Tensor &q = t[LQ], &k = t[LK], &v = t[LV], &d = t[LDECAY];
    REQUIRE(q.dim() == lead + 2 && float_type(q), lead == 2 ? "q must be [B, T, HK, K], bfloat16, float16 or float32" : "q must be [N, HK, K], bfloat16, float16 or float32");
    REQUIRE(k.scalar_type() == q.scalar_type() && v.scalar_type() == q.scalar_type(), "q, k and v must share a dtype");
    REQUIRE(k.sizes() == q.sizes(), "k must have the shape of q");
    REQUIRE(v.dim() == lead + 2, lead == 2 ? "v must be [B, T, HV, V]" : "v must be [N, HV, V]");
    for (int i = 0; i < lead; ++i) REQUIRE(v.size(i) == q.size(i), "q and v disagree on their leading axes");
    const int64_t HK = q.size(lead), HV = v.size(lead), K = q.size(lead + 1), V = v.size(lead + 1);
    REQUIRE(HK >= 1 && HV >= 1 && HV <= 65535 && HV % HK == 0, "the v-heads (at most 65535) must be a multiple of the q/k-heads");
    REQUIRE(K >= 1 && K <= MKDA_LINEAR_MAX_DIM && V >= 1 && V <= MKDA_LINEAR_MAX_DIM, "heads of 1 to 128 channels");
    REQUIRE(d.dim() == 1 && d.size(0) == HV && float_type(d), "log_decay must be [HV]");
    Py_RETURN_NONE;
}

// linear(q, k, v, log_decay, initial_state, table, dims, scale, want_last) -> (o, last or None)
PyObject* linear(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 9) return fail(PyExc_TypeError, "linear takes 9 arguments");
    variable_list t;
    if (!parse_tensors("linear_attention", a, LINEAR_INPUTS, 4, t)) return nullptr;
    if (!check_devices("linear_attention", t)) return nullptr;
    PyObject* ok = check_linear(t, 2);
    if (!ok) return nullptr;
    Py_DECREF(ok);
    const Tensor &v = t[LV], &h0 = t[LH0];
    REQUIRE(v.size(0) * v.size(1) <= MOST_TOKENS, "less than 2^31 tokens");
    const int64_t HV = v.size(2), K = t[LQ].size(3), V = v.size(3);
    Sequences q;
    if (!get_sequences(a[5], a[6], v.size(0), v.size(1), q)) return nullptr;
    REQUIRE(q.s.N <= 65535, "at most 65535 sequences");
    if (h0.defined()) {
        REQUIRE(h0.scalar_type() == at::kFloat, "initial_state must be float32");
        if (h0.dim() < 1 || h0.size(0) != q.s.N) return fail(PyExc_ValueError, count_error(q.s.N, h0.dim() ? h0.size(0) : 0));
        REQUIRE(h0.dim() == 4 && h0.size(1) == HV && h0.size(2) == K && h0.size(3) == V, "initial_state must be [N, HV, K, V]");
    }
    const double scale = a[7] == Py_None ? 1.0 / std::sqrt((double)K) : PyFloat_AsDouble(a[7]);
    const int want = PyObject_IsTrue(a[8]);
    if (PyErr_Occurred()) return nullptr;
    const bool grad = any_requires_grad(t);
    if (grad && t[LDECAY].requires_grad()) return fail(PyExc_RuntimeError, "linear_attention: log_decay has no gradient: pass log_decay.detach()");
    Tensor o, last;
    {
        pybind11::gil_scoped_release nogil;
        c10::cuda::CUDAGuard guard(v.device());
        reads_table(q);
        {
            at::AutoGradMode off(false);
            LinearCall call(q, t, scale);
            o = out_like(v, q.covers_all);
            if (want) last = new_cuda({q.s.N, HV, K, V}, at::kFloat, v.device());
            call.p.o = o.data_ptr(); call.p.ht = fmptr(last);
            cut_linear(call.p.S, q, HV, 1, 1, K, V, v.scalar_type());
            Tensor seg_h;
            if (call.p.S.seg) {
                seg_h = call.parts(v.device());
                call.p.seg_h = fmptr(seg_h);
            }
            library_call([&] { check_rc(mkda_linear_fwd(&call.p, stream()), "mkda_linear_fwd"); });
        }
        if (grad) {
            constexpr uint32_t Q = 1u << LQ, KK = 1u << LK, VV = 1u << LV, H = 1u << LH0;
            auto node = new_node("linear_attention", v.device(), t, {KK | VV | H, Q | VV, Q | KK, 0, Q}, [q, scale](const variable_list& s, const variable_list& g, const Need&) { return linear_backward(q, scale, s, g); });
            for (const Tensor& x : t) node->save(x);
            torch::autograd::set_history(o, node);
            if (last.defined()) torch::autograd::set_history(last, node);
        }
    }
    return pair(o, last);
    END_HANDLE_TH_ERRORS
}

// linear_step(q, k, v, log_decay, state, scale) -> o
PyObject* linear_step(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 6) return fail(PyExc_TypeError, "linear_step takes 6 arguments");
    variable_list t;
    if (!parse_tensors("linear_attention_step", a, LINEAR_INPUTS, LINEAR_INPUTS, t)) return nullptr;
    if (!check_devices("linear_attention_step", t)) return nullptr;
    PyObject* ok = check_linear(t, 1);
    if (!ok) return nullptr;
    Py_DECREF(ok);
    const Tensor v = t[LV], state = t[LH0];
    const int64_t N = v.size(0), HV = v.size(1), K = t[LQ].size(2), V = v.size(2);
    REQUIRE(N <= 65535, "at most 65535 sequences");
    REQUIRE(state.dim() == 4 && state.size(0) == N && state.size(1) == HV && state.size(2) == K && state.size(3) == V && state.scalar_type() == at::kFloat, "state must be float32 [N, HV, K, V]");
    if (!check_step("linear_attention_step", t, state)) return nullptr;
    const double scale = a[5] == Py_None ? 1.0 / std::sqrt((double)K) : PyFloat_AsDouble(a[5]);
    if (PyErr_Occurred()) return nullptr;
    Tensor o;
    {
        pybind11::gil_scoped_release nogil;
        c10::cuda::CUDAGuard guard(v.device());
        at::AutoGradMode off(false);
        t.pop_back();
        const LinearCall call(Sequences(), t, scale);
        const MkdaLinearFwd& f = call.p;
        o = out_like(v, true);
        MkdaLinearStep p{};
        p.N = (int)N; p.HK = f.HK; p.HV = f.HV; p.K = f.K; p.V = f.V; p.dtype = f.dtype; p.scale = f.scale;
        p.q = f.q; p.k = f.k; p.v = f.v; p.q_stride = f.q_stride; p.k_stride = f.k_stride; p.v_stride = f.v_stride;
        p.log_decay = f.log_decay; p.state = fmptr(state); p.o = o.data_ptr();
        library_call([&] { check_rc(mkda_linear_step(&p, stream()), "mkda_linear_step"); });
        changed(state);
    }
    return THPVariable_Wrap(o);
    END_HANDLE_TH_ERRORS
}

// ---- rotary positions ------------------------------------------------------------------------------------------------------------------------
struct RotaryPlan {
    int64_t tokens = 0, dim = 0;
    int heads_q = 0, heads_k = 0;
    MkdaRotary p{};
};
// q or k (either may be undefined) turned; `plan` has everything but the tensors
void rotate(const RotaryPlan& plan, const Tensor& positions, const Tensor& inv_freq, const Tensor& q, const Tensor& k, Tensor& q_out, Tensor& k_out, bool inverse) {
    MkdaRotary p = plan.p;
    const Rows rq = rows_of(q, 2), rk = rows_of(k, 2);
    auto half = [&](const Rows& r, int heads, int& h, const void*& from, long long& stride, void*& to, Tensor& out) {
        if (!r.t.defined()) return;
        h = heads; from = cptr(r.t); stride = r.stride;
        out = new_cuda(r.t.sizes(), r.t.scalar_type(), r.t.device());
        to = out.data_ptr();
    };
    half(rq, plan.heads_q, p.heads_q, p.q, p.q_stride, p.q_out, q_out);
    half(rk, plan.heads_k, p.heads_k, p.k, p.k_stride, p.k_out, k_out);
    p.inverse = inverse; p.positions = cptr(positions); p.inv_freq = fptr(inv_freq);
    check_rc(mkda_rotary(&p, stream()), "mkda_rotary");
}

// rotary(q, k or None, positions, inv_freq, axes or None, interleaved) -> (q, k or None)
PyObject* rotary(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 6) return fail(PyExc_TypeError, "rotary takes 6 arguments");
    variable_list t(4);
    for (int i = 0; i < 4; ++i) {
        if (!tensor_arg(a[i], t[i])) return nullptr;
        if (i != 1 && !t[i].defined()) { PyErr_Format(PyExc_TypeError, "rotary: argument %d must be a tensor", i + 1); return nullptr; }
    }
    if (!check_devices("rotary", t)) return nullptr;
    const Tensor &q = t[0], &k = t[1], &pos = t[2], &freq = t[3];
    REQUIRE(q.dim() >= 2 && float_type(q), "q must be [.., H, D], bfloat16, float16 or float32");
    const int64_t D = q.size(-1), F = freq.numel(), lead = q.dim() - 2;
    REQUIRE(D >= 1 && D <= MKDA_ROTARY_MAX_DIM, "heads of 1 to 512 channels");
    REQUIRE(freq.dim() == 1 && freq.scalar_type() == at::kFloat && 2 * F <= D, "inv_freq must be float32, one for each pair of turned channels");
    REQUIRE(q.size(-2) >= 1 && q.size(-2) <= 65536, "1 to 65536 heads");
    int64_t tokens = 1;
    for (int64_t i = 0; i < lead; ++i) tokens *= q.size(i);
    REQUIRE(tokens <= MOST_TOKENS, "less than 2^31 tokens");
    if (k.defined()) {
        REQUIRE(k.scalar_type() == q.scalar_type() && k.dim() == q.dim() && k.size(-1) == D && k.size(-2) >= 1 && k.size(-2) <= 65536, "k must be [.., H, D] of the type of q");
        for (int64_t i = 0; i < lead; ++i) REQUIRE(k.size(i) == q.size(i), "q and k disagree on their leading axes");
    }
    REQUIRE(pos.scalar_type() == at::kInt || pos.scalar_type() == at::kLong, "positions must be int32 or int64");
    RotaryPlan plan;
    plan.p.axes = 1;
    const int64_t extra = a[4] != Py_None;
    REQUIRE(pos.dim() == lead + extra, extra ? "positions must be [axes, ..] with the leading axes of q behind" : "positions must have the leading axes of q");
    for (int64_t i = 0; i < lead; ++i) REQUIRE(pos.size(i + extra) == q.size(i), "q and positions disagree on their leading axes");
    if (extra) {
        REQUIRE(pos.size(0) >= 1 && pos.size(0) <= 255, "1 to 255 axes");
        plan.p.axes = (int)pos.size(0);
        PyObject* seq = PySequence_Fast(a[4], "axes must be a sequence of whole numbers");
        if (!seq) return nullptr;
        const Py_ssize_t count = PySequence_Fast_GET_SIZE(seq);
        bool good = count == F;
        for (Py_ssize_t f = 0; good && f < count; ++f) {
            const long axis = PyLong_AsLong(PySequence_Fast_GET_ITEM(seq, f));
            if (PyErr_Occurred()) { Py_DECREF(seq); return nullptr; }
            good = axis >= 0 && axis < plan.p.axes;
            if (good) plan.p.axis_of[f >> 2] |= (int)((unsigned)axis << (8 * (f & 3)));
        }
        Py_DECREF(seq);
        REQUIRE(good, "axes must name the axis of each frequency");
    }
    const int interleaved = PyObject_IsTrue(a[5]);
    if (PyErr_Occurred()) return nullptr;
    const bool grad = any_requires_grad(t);
    if (grad && freq.requires_grad()) return fail(PyExc_RuntimeError, "rotary: inv_freq has no gradient: pass inv_freq.detach()");
    plan.tokens = tokens; plan.dim = D; plan.heads_q = (int)q.size(-2); plan.heads_k = k.defined() ? (int)k.size(-2) : 0;
    plan.p.tokens = (int)tokens; plan.p.dim = (int)D; plan.p.freqs = (int)F; plan.p.interleaved = interleaved; plan.p.dtype = dtype_code(q); plan.p.positions_64 = pos.scalar_type() == at::kLong;
    Tensor q_out, k_out;
    {
        pybind11::gil_scoped_release nogil;
        c10::cuda::CUDAGuard guard(q.device());
        {
            at::AutoGradMode off(false);
            const Tensor at_ = pos.contiguous(), fr = freq.contiguous();
            library_call([&] { rotate(plan, at_, fr, q, k, q_out, k_out, false); });
        }
        if (grad) {
            // linear in q and k: their gradients are functions of the incoming ones alone
            auto node = new_node("rotary", q.device(), {q, k}, {0, 0}, [plan](const variable_list& s, const variable_list& g, const Need& need) {
                const Tensor at_ = s[0].contiguous(), fr = s[1].contiguous();
                variable_list out(2);
                const Tensor dq = g[0].defined() && need(0) ? g[0] : Tensor(), dk = g.size() > 1 && g[1].defined() && need(1) ? g[1] : Tensor();
                rotate(plan, at_, fr, dq, dk, out[0], out[1], true);
                return out;
            });
            node->save(pos);
            node->save(freq);
            torch::autograd::set_history(q_out, node);
            if (k.defined()) torch::autograd::set_history(k_out, node);
        }
    }
    return pair(q_out, k_out);
    END_HANDLE_TH_ERRORS
}

// ---- layer norm ------------------------------------------------------------------------------------------------------------------------------
// inputs x, weight, bias, residual; saved: what was normalised, the weight, mean and 1 / sqrt(var + eps); the bias' size and type
struct LayerNormCall {
    int groups;
    bool residual, bias;
    at::ScalarType dt, res_dt, bias_dt;
};
variable_list layer_norm_backward(const LayerNormCall& c, const variable_list& s, const variable_list& grads, const Need& need) {
    const Rows r = rows_of(s[0]);
    const Tensor &w = s[1], stats = aligned(s[2]);
    const int64_t H = s[0].size(-1), rows = row_count(s[0]);
    const at::Device dev = s[0].device();
    const Tensor dy = grads[0].defined() ? aligned(grads[0]) : at::zeros(s[0].sizes(), s[0].options().dtype(c.dt));
    const Tensor dsum = grads.size() > 1 && grads[1].defined() ? aligned(grads[1]) : Tensor();
    const Tensor wc = aligned(w);
    variable_list out(4);
    out[0] = new_cuda(s[0].sizes(), c.dt, dev);
    if (c.residual) out[3] = c.res_dt == c.dt ? out[0] : new_cuda(s[0].sizes(), c.res_dt, dev);      // one gradient for both where they share a type
    if (w.defined()) out[1] = new_cuda(w.sizes(), w.scalar_type(), dev);
    if (c.bias) out[2] = new_cuda({H}, c.bias_dt, dev);
    Tensor part;
    if ((w.defined() && need(1)) || (c.bias && need(2))) part = new_cuda({mkda_layer_norm_bwd_part_rows((int)rows, (int)H, c.groups), 2, H}, at::kFloat, dev);
    MkdaLayerNormBwd p{};
    p.rows = (int)rows; p.width = (int)H; p.groups = c.groups; p.dtype = dtype_code(out[0]);
    p.s = r.t.data_ptr(); p.s_stride = r.stride; p.s_dtype = dtype_code(r.t); p.weight = cptr(wc); p.weight_dtype = w.defined() ? dtype_code(w) : MKDA_F32; p.stats = fptr(stats);
    p.dy = dy.data_ptr(); p.dsum = cptr(dsum); p.dx = out[0].data_ptr(); p.dres = c.residual && c.res_dt != c.dt ? out[3].data_ptr() : nullptr;
    p.part_rows = part.defined() ? (int)part.size(0) : 0; p.part = fmptr(part);
    check_rc(mkda_layer_norm_bwd(&p, stream()), "mkda_layer_norm_bwd");
    if (part.defined()) {
        MkdaSumRows q{};
        const int count = rows ? p.part_rows : 0;          // without rows nothing has been written
        if (w.defined()) q.job[0] = {fptr(part), count, 1, 2 * H, H, (int)H, (int)H, 0, 0, 1, out[1].data_ptr(), dtype_code(out[1])};
        if (c.bias) q.job[1] = {fptr(part) + H, count, 1, 2 * H, H, (int)H, (int)H, 0, 0, 1, out[2].data_ptr(), dtype_code(out[2])};
        check_rc(mkda_sum_rows(&q, stream()), "mkda_sum_rows");
    }
    return out;
}

// layer_norm(x, weight, bias, residual, groups, eps) -> (y, residual sum or None)
PyObject* layer_norm(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 6) return fail(PyExc_TypeError, "layer_norm takes 6 arguments");
    variable_list t;
    if (!parse_tensors("layer_norm", a, 4, 1, t)) return nullptr;
    const Tensor &x = t[0], &w = t[1], &b = t[2], &res = t[3];
    if (!check_devices("layer_norm", t)) return nullptr;
    REQUIRE(x.dim() >= 1 && float_type(x), "x must be [.., H], bfloat16, float16 or float32");
    const int64_t H = x.size(-1), rows = row_count(x), groups = PyLong_AsLong(a[4]);
    const double eps = PyFloat_AsDouble(a[5]);
    if (PyErr_Occurred()) return nullptr;
    REQUIRE(groups >= 1 && groups <= 65535 && H >= 1 && H % groups == 0, "the channels must be a multiple of the groups, at most 65535");
    REQUIRE(H / groups <= MKDA_NORM_MAX_WIDTH && H <= MOST_CHANNELS, "1 to 32768 channels to a group");
    REQUIRE(rows <= MOST_TOKENS, "less than 2^31 rows");
    REQUIRE(!w.defined() || (w.dim() == 1 && w.size(0) == H && float_type(w)), "weight must be [H]");
    REQUIRE(!b.defined() || (b.dim() == 1 && b.size(0) == H && float_type(b)), "bias must be [H]");
    REQUIRE(!res.defined() || res.sizes() == x.sizes(), "residual must have the shape of x");
    REQUIRE(!res.defined() || res.scalar_type() == x.scalar_type() || res.scalar_type() == at::kFloat, "residual must have the type of x, or be float32");
    const bool grad = any_requires_grad(t);
    Tensor y, sum, stats;
    {
        pybind11::gil_scoped_release nogil;
        c10::cuda::CUDAGuard guard(x.device());
        {
            at::AutoGradMode off(false);
            const Rows xr = rows_of(x), rr = rows_of(res);
            const Tensor wc = aligned(w), bc = aligned(b);
            y = new_cuda(x.sizes(), x.scalar_type(), x.device());
            if (res.defined()) sum = new_cuda(x.sizes(), res.scalar_type(), x.device());
            if (grad) stats = new_cuda({rows, groups, 2}, at::kFloat, x.device());
            MkdaLayerNormFwd p{};
            p.rows = (int)rows; p.width = (int)H; p.groups = (int)groups; p.dtype = dtype_code(x); p.res_dtype = res.defined() ? dtype_code(res) : MKDA_F32; p.eps = (float)eps;
            p.x = xr.t.data_ptr(); p.x_stride = xr.stride; p.residual = cptr(rr.t); p.res_stride = rr.stride;
            p.weight = cptr(wc); p.weight_dtype = w.defined() ? dtype_code(w) : MKDA_F32; p.bias = cptr(bc); p.bias_dtype = b.defined() ? dtype_code(b) : MKDA_F32;
            p.sum = mptr(sum); p.y = y.data_ptr(); p.stats = fmptr(stats);
            library_call([&] { check_rc(mkda_layer_norm_fwd(&p, stream()), "mkda_layer_norm_fwd"); });
        }
        if (grad) {
            const bool has = res.defined();
            const LayerNormCall c{(int)groups, has, b.defined(), x.scalar_type(), has ? res.scalar_type() : x.scalar_type(), b.defined() ? b.scalar_type() : at::kFloat};
            constexpr uint32_t X = 1, WT = 2, RES = 8;
            auto node = new_node("layer_norm", x.device(), t, {X | WT | RES, X | RES, 0, X | WT | RES}, [c](const variable_list& s, const variable_list& g, const Need& need) {
                return layer_norm_backward(c, s, g, need);
            });
            node->state_linear = true;                     // a sum
            torch::autograd::set_history(y, node);
            if (has) torch::autograd::set_history(sum, node);
            node->save(has ? sum : x, has);
            node->save(w);
            node->save(stats);
        }
    }
    return pair(y, sum);
    END_HANDLE_TH_ERRORS
}

}  // namespace

PyMethodDef mkda_host::mixer_methods[] = {
    {"linear", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(linear)), METH_FASTCALL, "linear attention with a decay for each head"},
    {"linear_step", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(linear_step)), METH_FASTCALL, "one token of a linear attention"},
    {"rotary", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(rotary)), METH_FASTCALL, "rotary positions"},
    {"layer_norm", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(layer_norm)), METH_FASTCALL, "layer norm"},
    {nullptr, nullptr, 0, nullptr}};
