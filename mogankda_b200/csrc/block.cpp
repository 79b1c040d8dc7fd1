// Python entry points and autograd node of the operators around the layer: short causal convolution, selective scan, RMS norm.  Checks, buffers and
// launches are native for the same reason as the layer's (binding.cpp): a call on a few tokens is nothing but host work.
#include "block.h"

namespace {

// ---- convolution ---------------------------------------------------------------------------------------------------------------------------
MkdaConvFwd conv_call(const Sequences& q, const Rows& x, const Tensor& w, const Tensor& bias, const Tensor& state, int silu) {
    MkdaConvFwd p{};
    p.S = q.s; p.D = (int)w.size(0); p.W = (int)w.size(1); p.dtype = dtype_code(x.t); p.silu = silu; p.x = x.t.data_ptr(); p.x_stride = x.stride;
    p.weight = fptr(w); p.bias = fptr(bias); p.state = cptr(state);
    return p;
}

variable_list conv_backward(const Sequences& q, int silu, const variable_list& s, const variable_list& grads) {
    reads_table(q);
    const Tensor &x0 = s[0], w = param(s[1]), bias = param(s[2]), state = aligned(s[3]);
    const Rows x = rows_of(x0);
    const int64_t D = w.size(0), W = w.size(1), TT = q.s.TT;
    const Tensor dy = grads[0].defined() ? aligned(grads[0]) : at::zeros_like(x0, at::MemoryFormat::Contiguous);
    const Tensor dlast = grads.size() > 1 && grads[1].defined() ? aligned(grads[1]) : Tensor();
    const int64_t rows = mkda_conv_bwd_part_rows((int)TT, (int)D);
    const Tensor part = new_cuda({rows, (W + 1) * D}, at::kFloat, x0.device());
    variable_list out(4);
    out[0] = out_like(x0, q.covers_all);
    out[1] = new_cuda(s[1].sizes(), s[1].scalar_type(), x0.device());
    if (s[2].defined()) out[2] = new_cuda(s[2].sizes(), s[2].scalar_type(), x0.device());
    if (state.defined()) out[3] = new_cuda(state.sizes(), state.scalar_type(), x0.device());
    const MkdaConvFwd f = conv_call(q, x, w, bias, state, silu);
    MkdaConvBwd p{};
    p.S = f.S; p.D = f.D; p.W = f.W; p.dtype = f.dtype; p.silu = silu; p.x = f.x; p.x_stride = f.x_stride; p.weight = f.weight; p.bias = f.bias; p.state = f.state;
    p.dy = dy.data_ptr(); p.dlast = cptr(dlast); p.dx = out[0].data_ptr(); p.dstate = mptr(out[3]); p.part_rows = (int)rows; p.part = fmptr(part);
    check_rc(mkda_conv_bwd(&p, stream()), "mkda_conv_bwd");
    MkdaSumRows r{};
    r.job[0] = {fptr(part), (int)rows, 1, (W + 1) * D, W * D, (int)D, (int)D, 0, 1, W, out[1].data_ptr(), dtype_code(out[1])};
    if (out[2].defined()) r.job[1] = {fptr(part) + W * D, (int)rows, 1, (W + 1) * D, D, (int)D, (int)D, 0, 0, 1, out[2].data_ptr(), dtype_code(out[2])};
    check_rc(mkda_sum_rows(&r, stream()), "mkda_sum_rows");
    return out;
}

#define CONV_PARAMS(W_, D_) \
    REQUIRE((W_).dim() == 2 && (W_).size(0) == (D_) && (W_).size(1) >= 2 && (W_).size(1) <= 4, "weight must be [D, W] with 2 to 4 taps"); \
    REQUIRE(float_type(W_), "weight must be bfloat16, float16 or float32")

// conv(x, weight, bias, initial_state, table, dims, silu, want_last) -> (y, last or None)
PyObject* conv(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 8) return fail(PyExc_TypeError, "conv takes 8 arguments");
    variable_list t;
    if (!parse_tensors("causal_conv1d", a, 4, 2, t)) return nullptr;
    const Tensor &x = t[0], &w = t[1], &bias = t[2], &state = t[3];
    if (!check_devices("causal_conv1d", t)) return nullptr;
    REQUIRE(x.dim() == 3 && float_type(x), "x must be [B, T, D], bfloat16, float16 or float32");
    const int64_t D = x.size(2);
    REQUIRE(D >= 1 && D <= MOST_CHANNELS && x.size(0) * x.size(1) <= MOST_TOKENS, "x must have 1 to 2^24 channels and less than 2^31 tokens");
    CONV_PARAMS(w, D);
    REQUIRE(!bias.defined() || (bias.dim() == 1 && bias.size(0) == D && float_type(bias)), "bias must be [D]");
    Sequences q;
    if (!get_sequences(a[4], a[5], x.size(0), x.size(1), q)) return nullptr;
    if (state.defined()) {
        REQUIRE(state.scalar_type() == x.scalar_type(), "initial_state must have the type of x");
        if (state.dim() < 1 || state.size(0) != q.s.N) return fail(PyExc_ValueError, count_error(q.s.N, state.dim() ? state.size(0) : 0));
        REQUIRE(state.dim() == 3 && state.size(1) == w.size(1) - 1 && state.size(2) == D, "initial_state must be [N, W - 1, D]");
    }
    const int silu = (int)PyLong_AsLong(a[6]), want = PyObject_IsTrue(a[7]);
    if (PyErr_Occurred()) return nullptr;
    Tensor y, last;
    {
        pybind11::gil_scoped_release nogil;
        c10::cuda::CUDAGuard guard(x.device());
        reads_table(q);
        const bool grad = any_requires_grad(t);
        {
            at::AutoGradMode off(false);
            const Rows xr = rows_of(x);
            const Tensor wf = param(w), bf = param(bias), sf = aligned(state);
            y = out_like(x, q.covers_all);
            if (want) last = new_cuda({q.s.N, w.size(1) - 1, D}, x.scalar_type(), x.device());
            MkdaConvFwd p = conv_call(q, xr, wf, bf, sf, silu);
            p.y = y.data_ptr(); p.last = mptr(last);
            library_call([&] { check_rc(mkda_conv_fwd(&p, stream()), "mkda_conv_fwd"); });
        }
        if (grad) {
            constexpr uint32_t X = 1, WT = 2, BIAS = 4, ST = 8, ALL = X | WT | BIAS | ST;
            const std::vector<uint32_t> depends = silu ? std::vector<uint32_t>(4, ALL) : std::vector<uint32_t>{WT, X | ST, 0, WT};      // linear but for the product of weight and tokens
            auto node = new_node("causal_conv1d", x.device(), t, depends, [q, silu](const variable_list& s, const variable_list& g, const Need&) { return conv_backward(q, silu, s, g); });
            node->state_linear = true;                     // tokens and states as they are
            for (const Tensor& v : t) node->save(v);
            torch::autograd::set_history(y, node);
            if (last.defined()) torch::autograd::set_history(last, node);
        }
    }
    return pair(y, last);
    END_HANDLE_TH_ERRORS
}

// conv_step(x, state, weight, bias, silu) -> y
PyObject* conv_step(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 5) return fail(PyExc_TypeError, "conv_step takes 5 arguments");
    variable_list t;
    if (!parse_tensors("causal_conv1d_step", a, 4, 3, t)) return nullptr;
    const Tensor &x = t[0], &state = t[1], &w = t[2], &bias = t[3];
    if (!check_devices("causal_conv1d_step", t)) return nullptr;
    REQUIRE(x.dim() == 2 && float_type(x) && x.size(1) >= 1 && x.size(1) <= MOST_CHANNELS, "x must be [N, D], bfloat16, float16 or float32");
    const int64_t N = x.size(0), D = x.size(1);
    REQUIRE(N <= 65535, "at most 65535 sequences");
    CONV_PARAMS(w, D);
    REQUIRE(!bias.defined() || (bias.dim() == 1 && bias.size(0) == D && float_type(bias)), "bias must be [D]");
    REQUIRE(state.dim() == 3 && state.size(0) == N && state.size(1) == w.size(1) - 1 && state.size(2) == D && state.scalar_type() == x.scalar_type(),
            "state must be [N, W - 1, D] of the type of x");
    if (!check_step("causal_conv1d_step", t, state)) return nullptr;
    const int silu = (int)PyLong_AsLong(a[4]);
    if (PyErr_Occurred()) return nullptr;
    Tensor y;
    {
        pybind11::gil_scoped_release nogil;
        c10::cuda::CUDAGuard guard(x.device());
        at::AutoGradMode off(false);
        const Rows xr = rows_of(x);
        const Tensor wf = param(w), bf = param(bias);
        y = out_like(x, true);
        MkdaConvStep p{};
        p.N = (int)N; p.D = (int)D; p.W = (int)w.size(1); p.dtype = dtype_code(x); p.silu = silu; p.x = xr.t.data_ptr(); p.x_stride = xr.stride;
        p.weight = fptr(wf); p.bias = fptr(bf); p.state = state.data_ptr(); p.y = y.data_ptr();
        library_call([&] { check_rc(mkda_conv_step(&p, stream()), "mkda_conv_step"); });
        changed(state);
    }
    return THPVariable_Wrap(y);
    END_HANDLE_TH_ERRORS
}

// ---- scan ------------------------------------------------------------------------------------------------------------------------------------
enum { SX, SDT, SA, SB, SC, SSKIP, SZ, SBIAS, SH0, SCAN_INPUTS };

// Cuts long sequences into parts that run side by side where there are fewer blocks than places for them (`places` per SM).  The pass over the parts that comes first takes `pre` of
// the time of the main pass over them, and both start anew, about 128 tokens' time.  Whole / cut in us, 8192 tokens, first pass included: forward
// x 256 channels 274 / 40, x 1024 278 / 132, x 2048 280 / 254; backward x 256 970 / 77, x 1024 1059 / 254, x 2048 1064 / 520, x 4096 1066 / 911;
// 600 tokens x 512 25 / 14 and 75 / 27.
// Every sequence has a row of blocks for each part that the longest one has, and a block without tokens takes its SM 0.9 us in each of the two kernels, in the backward pass (whose
// main kernel has fewer rows) half of that: the time of `nothing` tokens.  One document of 4096 tokens beside 512 of 8, x 256 channels: forward 140 / 534, backward 540 / 614; beside
// 296 of 8 backward 534 / 474; 8192 beside 64 of 64 forward 276 / 150.
void cut(MkdaSeqs& s, const Sequences& q, int blocks, int64_t P, int64_t D, int places, double pre, double nothing) {
    if (q.longest < 400 || s.N == 0) return;
    const double side_by_side = blocks * std::max(1.0, (double)s.TT / q.longest);      // blocks that are busy as long as the longest sequence runs
    const int64_t want = (int64_t)(places * sms() / side_by_side);
    if (want < 2) return;
    const int64_t seg = std::max<int64_t>(128, ((q.longest + want - 1) / want + 63) / 64 * 64), segs = (q.longest + seg - 1) / seg;
    const int64_t empty = std::max<int64_t>(0, s.N * (segs - 1) - s.TT / seg);      // parts without tokens, at least
    if ((1 + pre) * seg + 128 + nothing * empty * blocks / sms() >= q.longest || s.N * segs * D * P * 4 > (int64_t)256 << 20) return;
    s.seg = (int)seg;
    s.segs = (int)segs;
}

// What a scan call hands to the library; the tensors behind the pointers are kept in `hold`.
struct ScanCall {
    MkdaScanFwd p{};
    std::vector<Tensor> hold;
    ScanCall(const Sequences& q, const variable_list& t, int softplus) {
        p.S = q.s; p.D = (int)t[SX].size(-1); p.NST = (int)t[SA].size(1);
        const int inner = t[SB].dim() - (t[SX].dim() - 1);         // [.., N] or [.., G, N]
        p.G = inner == 2 ? (int)t[SB].size(-2) : 1;
        p.dtype = dtype_code(t[SX]); p.softplus = softplus;
        auto rows = [&](int i, int in, const void*& ptr, long long& stride) {
            const Rows r = rows_of(t[i], in);
            ptr = cptr(r.t);
            stride = r.stride;
            hold.push_back(r.t);
        };
        rows(SX, 1, p.x, p.x_stride); rows(SDT, 1, p.dt, p.dt_stride); rows(SB, inner, p.B, p.B_stride); rows(SC, inner, p.C, p.C_stride);
        if (t[SZ].defined()) rows(SZ, 1, p.z, p.z_stride);
        auto fp32 = [&](int i) {
            const Tensor v = param(t[i]);
            hold.push_back(v);
            return fptr(v);
        };
        p.A = fp32(SA); p.skip = fp32(SSKIP); p.dt_bias = fp32(SBIAS);
        if ((int)t.size() > SH0) p.h0 = fp32(SH0);
    }
};

// The backward pass leaves dB and dC per block of channels, 8 P bytes per token and block.  Where that is more than 1 GiB, it runs over ranges of blocks whose sums are added up in
// between.  A range has the blocks that are resident at once, two per SM, so that ranges take as many waves as one launch would.
struct Ranges { int count, blocks; };      // blocks of each group
Ranges ranges_of_blocks(const Sequences& q, int per, int G, int64_t P) {
    if (q.longest == 0 || (double)per * G * q.s.TT * P * 8 <= (double)(1 << 30)) return {1, per};
    const double side_by_side = G * std::max(1.0, (double)q.s.TT / q.longest);
    const int most = std::max(1, (int)std::ceil(2 * sms() / side_by_side)), count = (per + most - 1) / most;
    const int blocks = (per + count - 1) / count, ranges = (per + blocks - 1) / blocks;      // of equal size
    return blocks + ranges < per ? Ranges{ranges, blocks} : Ranges{1, per};
}

variable_list scan_backward(const Sequences& q, int softplus, const variable_list& s, const variable_list& grads) {
    reads_table(q);
    const variable_list in(s.begin(), s.begin() + SCAN_INPUTS);
    const Tensor ckpt = aligned(s[SCAN_INPUTS]);
    const ScanCall call(q, in, softplus);
    const Tensor& x = in[SX];
    const at::Device dev = x.device();
    const int64_t TT = q.s.TT, D = call.p.D, N = call.p.NST, G = call.p.G, P = mkda_scan_padded_states((int)N);
    const Tensor dy = grads[0].defined() ? aligned(grads[0]) : at::zeros_like(x, at::MemoryFormat::Contiguous);
    const Tensor dht = grads.size() > 1 && grads[1].defined() ? aligned(grads[1]) : Tensor();
    MkdaScanBwd p{};
    p.f = call.p;
    p.f.ckpt = fmptr(ckpt);
    p.dy = dy.data_ptr(); p.dht = fptr(dht);
    variable_list out(SCAN_INPUTS);
    for (int i : {SX, SDT, SZ})
        if (in[i].defined()) out[i] = out_like(in[i], q.covers_all);
    for (int i : {SB, SC}) out[i] = out_like(in[i], q.covers_all);
    for (int i : {SA, SSKIP, SBIAS, SH0})
        if (in[i].defined()) out[i] = new_cuda(in[i].sizes(), in[i].scalar_type(), dev);
    p.dx = out[SX].data_ptr(); p.ddt = out[SDT].data_ptr(); p.dz = mptr(out[SZ]); p.dh0 = fmptr(out[SH0]);
    p.channel_blocks = mkda_scan_bwd_channel_blocks((int)D, (int)G, (int)N);
    const int per = p.channel_blocks / (int)G;
    const Ranges ranges = ranges_of_blocks(q, per, (int)G, P);
    cut(p.f.S, q, ranges.blocks * (int)G, P, D, 2, 0.4, 9);
    const int64_t rows = p.f.S.seg ? (int64_t)q.s.N * p.f.S.segs : q.s.N;
    Tensor seg_g, seg_d;
    if (p.f.S.seg) {
        seg_g = new_cuda({rows, D, P}, at::kFloat, dev);
        seg_d = new_cuda({rows, D}, at::kFloat, dev);
        p.seg_g = fmptr(seg_g); p.seg_d = fmptr(seg_d);
    }
    // sequences are dealt to rows of blocks: enough of them for 16 blocks per SM; each leaves a row of sums for A, D and dt_bias
    p.slots = (int)std::max<int64_t>(1, std::min<int64_t>(rows, (16 * sms() + ranges.blocks * G - 1) / (ranges.blocks * G)));
    while (p.f.S.seg && std::gcd(p.slots, q.s.N) > 1) --p.slots;      // part k of sequence i is number k N + i: the parts of a sequence go to different rows
    const Tensor pB = new_cuda({G * ranges.blocks, TT * P}, at::kFloat, dev), pC = new_cuda({G * ranges.blocks, TT * P}, at::kFloat, dev);
    Tensor sB, sC;                                         // of each range, [G][ranges][TT P]
    if (ranges.count > 1) {
        sB = new_cuda({G * ranges.count, TT * P}, at::kFloat, dev);
        sC = new_cuda({G * ranges.count, TT * P}, at::kFloat, dev);
    }
    const Tensor pA = new_cuda({p.slots, D * P}, at::kFloat, dev);
    Tensor pskip, pbias;
    if (out[SSKIP].defined()) pskip = new_cuda({p.slots, D}, at::kFloat, dev);
    if (out[SBIAS].defined()) pbias = new_cuda({p.slots, D}, at::kFloat, dev);
    p.part_B = fmptr(pB); p.part_C = fmptr(pC); p.part_A = fmptr(pA); p.part_skip = fmptr(pskip); p.part_bias = fmptr(pbias);
    // sums over `rows` rows of each group, of the tokens that lie in sequences
    auto tokens = [&](const Tensor& part, int rows, const Tensor& o) {
        return MkdaSumJob{fptr(part), rows, (int)G, TT * P, q.end * P, (int)P, (int)N, N, G * N, 1, o.data_ptr(), dtype_code(o)};
    };
    auto range = [&](const Tensor& part, int rows, const Tensor& o, int r) {
        return MkdaSumJob{fptr(part), rows, (int)G, TT * P, q.end * P, (int)P, (int)P, ranges.count * TT * P, P, 1, fmptr(o) + r * TT * P, MKDA_F32};
    };
    auto channels = [&](const Tensor& part, const Tensor& o, int64_t pad, int64_t width) {
        return MkdaSumJob{fptr(part), p.slots, 1, D * pad, D * pad, (int)pad, (int)width, 0, width, 1, o.data_ptr(), dtype_code(o)};
    };
    for (int r = 0; r < ranges.count; ++r) {
        p.first_block = r * ranges.blocks;
        p.blocks = std::min(ranges.blocks, per - p.first_block);
        check_rc(mkda_scan_bwd(&p, stream()), "mkda_scan_bwd");
        if (ranges.count == 1 || q.end == 0) continue;
        MkdaSumRows part{};
        part.job[0] = range(pB, p.blocks, sB, r);
        part.job[1] = range(pC, p.blocks, sC, r);
        check_rc(mkda_sum_rows(&part, stream()), "mkda_sum_rows");
    }
    MkdaSumRows r{};
    r.job[0] = tokens(ranges.count > 1 ? sB : pB, ranges.count > 1 ? ranges.count : per, out[SB]);
    r.job[1] = tokens(ranges.count > 1 ? sC : pC, ranges.count > 1 ? ranges.count : per, out[SC]);
    r.job[2] = channels(pA, out[SA], P, N);
    if (pskip.defined()) r.job[3] = channels(pskip, out[SSKIP], 1, 1);
    if (pbias.defined()) r.job[4] = channels(pbias, out[SBIAS], 1, 1);
    check_rc(mkda_sum_rows(&r, stream()), "mkda_sum_rows");
    return out;
}

// what each input's gradient is a function of: the result is linear in x and the entering state together, in B, in C and in D
std::vector<uint32_t> scan_depends() {
    auto but = [](std::initializer_list<int> none) {
        uint32_t m = (1u << SCAN_INPUTS) - 1;
        for (int i : none) m &= ~(1u << i);
        return m;
    };
    std::vector<uint32_t> d(SCAN_INPUTS);
    d[SX] = but({SX, SH0});
    d[SDT] = d[SA] = d[SBIAS] = but({SSKIP});
    d[SB] = but({SB, SSKIP, SH0});
    d[SC] = but({SC, SSKIP});
    d[SSKIP] = 1u << SX | 1u << SZ;
    d[SZ] = but({});
    d[SH0] = but({SX, SB, SSKIP, SH0});
    return d;
}

// the checks that prompts and single tokens share; `lead` axes in front of the channels
PyObject* check_scan(const variable_list& t, int lead) {
    const Tensor &x = t[SX], &A = t[SA], &B = t[SB], &C = t[SC];
    REQUIRE(x.dim() == lead + 1 && float_type(x) && x.size(lead) >= 1, lead == 2 ? "x must be [B, T, D], bfloat16, float16 or float32" : "x must be [N, D], bfloat16, float16 or float32");
    const int64_t D = x.size(lead);
    REQUIRE(D <= MOST_CHANNELS, "at most 2^24 channels");
    for (int i : {SDT, SB, SC, SZ}) REQUIRE(!t[i].defined() || t[i].scalar_type() == x.scalar_type(), "x, dt, B, C and z must share a dtype");
    for (int i : {SDT, SZ}) REQUIRE(!t[i].defined() || t[i].sizes() == x.sizes(), "dt and z must have the shape of x");
    REQUIRE(A.dim() == 2 && A.size(0) == D && float_type(A), "A must be [D, N]");
    REQUIRE(A.size(1) >= 1 && A.size(1) <= MKDA_SCAN_MAX_STATES, "1 to 64 states per channel");
    REQUIRE((B.dim() == lead + 1 || B.dim() == lead + 2) && B.sizes() == C.sizes() && B.size(-1) == A.size(1), "B and C must be [.., N] or [.., G, N]");
    for (int d = 0; d < lead; ++d) REQUIRE(B.size(d) == x.size(d), "x and B disagree on their leading axes");
    REQUIRE(B.dim() == lead + 1 || (B.size(lead) >= 1 && D % B.size(lead) == 0), "the channels must be a multiple of the groups");
    for (int i : {SSKIP, SBIAS}) REQUIRE(!t[i].defined() || (t[i].dim() == 1 && t[i].size(0) == D && float_type(t[i])), "D and dt_bias must be [D]");
    Py_RETURN_NONE;
}

// scan(x, dt, A, B, C, D, z, dt_bias, initial_state, table, dims, softplus, want_last) -> (y, last or None)
PyObject* scan(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 13) return fail(PyExc_TypeError, "scan takes 13 arguments");
    variable_list t;
    if (!parse_tensors("selective_scan", a, SCAN_INPUTS, 5, t)) return nullptr;
    if (!check_devices("selective_scan", t)) return nullptr;
    PyObject* ok = check_scan(t, 2);
    if (!ok) return nullptr;
    Py_DECREF(ok);
    const Tensor &x = t[SX], &h0 = t[SH0];
    REQUIRE(x.size(0) * x.size(1) <= MOST_TOKENS, "less than 2^31 tokens");
    const int64_t D = x.size(2), NST = t[SA].size(1);
    Sequences q;
    if (!get_sequences(a[9], a[10], x.size(0), x.size(1), q)) return nullptr;
    if (h0.defined()) {
        REQUIRE(h0.scalar_type() == at::kFloat, "initial_state must be float32");
        if (h0.dim() < 1 || h0.size(0) != q.s.N) return fail(PyExc_ValueError, count_error(q.s.N, h0.dim() ? h0.size(0) : 0));
        REQUIRE(h0.dim() == 3 && h0.size(1) == D && h0.size(2) == NST, "initial_state must be [N, D, states]");
    }
    const int softplus = PyObject_IsTrue(a[11]), want = PyObject_IsTrue(a[12]);
    if (PyErr_Occurred()) return nullptr;
    Tensor y, last, ckpt;
    {
        pybind11::gil_scoped_release nogil;
        c10::cuda::CUDAGuard guard(x.device());
        reads_table(q);
        const bool grad = any_requires_grad(t);
        {
            at::AutoGradMode off(false);
            ScanCall call(q, t, softplus);
            y = out_like(x, q.covers_all);
            if (want) last = new_cuda({q.s.N, D, NST}, at::kFloat, x.device());
            if (grad) ckpt = new_cuda({std::max<int64_t>(q.checkpoints, 1), D, mkda_scan_padded_states((int)NST)}, at::kFloat, x.device());
            call.p.y = y.data_ptr(); call.p.ht = fmptr(last); call.p.ckpt = fmptr(ckpt);
            const int64_t P = mkda_scan_padded_states((int)NST);
            cut(call.p.S, q, mkda_scan_bwd_channel_blocks((int)D, call.p.G, (int)NST), P, D, 1, 0.75, 54);      // the forward kernel has the same blocks
            Tensor seg_h, seg_d;
            if (call.p.S.seg) {
                const int64_t rows = (int64_t)q.s.N * call.p.S.segs;
                seg_h = new_cuda({rows, D, P}, at::kFloat, x.device());
                seg_d = new_cuda({rows, D}, at::kFloat, x.device());
                call.p.seg_h = fmptr(seg_h); call.p.seg_d = fmptr(seg_d);
            }
            library_call([&] { check_rc(mkda_scan_fwd(&call.p, stream()), "mkda_scan_fwd"); });
        }
        if (grad) {
            auto node = new_node("selective_scan", x.device(), t, scan_depends(), [q, softplus](const variable_list& s, const variable_list& g, const Need&) { return scan_backward(q, softplus, s, g); });
            for (const Tensor& v : t) node->save(v);
            node->save(ckpt);
            torch::autograd::set_history(y, node);
            if (last.defined()) torch::autograd::set_history(last, node);
        }
    }
    return pair(y, last);
    END_HANDLE_TH_ERRORS
}

// scan_step(x, dt, A, B, C, D, z, dt_bias, state, softplus) -> y
PyObject* scan_step(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 10) return fail(PyExc_TypeError, "scan_step takes 10 arguments");
    variable_list t;
    if (!parse_tensors("selective_scan_step", a, SCAN_INPUTS, 5, t)) return nullptr;
    const Tensor &x = t[SX], state = t[SH0];
    if (!state.defined()) return fail(PyExc_TypeError, "selective_scan_step: the state must be a tensor");
    if (!check_devices("selective_scan_step", t)) return nullptr;
    PyObject* ok = check_scan(t, 1);
    if (!ok) return nullptr;
    Py_DECREF(ok);
    const int64_t N = x.size(0), D = x.size(1), NST = t[SA].size(1);
    REQUIRE(N <= 65535, "at most 65535 sequences");
    REQUIRE(state.dim() == 3 && state.size(0) == N && state.size(1) == D && state.size(2) == NST && state.scalar_type() == at::kFloat, "state must be float32 [N, D, states]");
    if (!check_step("selective_scan_step", t, state)) return nullptr;
    const int softplus = PyObject_IsTrue(a[9]);
    if (PyErr_Occurred()) return nullptr;
    Tensor y;
    {
        pybind11::gil_scoped_release nogil;
        c10::cuda::CUDAGuard guard(x.device());
        at::AutoGradMode off(false);
        t.pop_back();
        const ScanCall call(Sequences(), t, softplus);
        const MkdaScanFwd& f = call.p;
        y = out_like(x, true);
        MkdaScanStep p{};
        p.N = (int)N; p.D = f.D; p.NST = f.NST; p.G = f.G; p.dtype = f.dtype; p.softplus = softplus; p.x = f.x; p.dt = f.dt; p.z = f.z; p.B = f.B; p.C = f.C;
        p.x_stride = f.x_stride; p.dt_stride = f.dt_stride; p.z_stride = f.z_stride; p.B_stride = f.B_stride; p.C_stride = f.C_stride;
        p.A = f.A; p.skip = f.skip; p.dt_bias = f.dt_bias; p.state = fmptr(state); p.y = y.data_ptr();
        library_call([&] { check_rc(mkda_scan_step(&p, stream()), "mkda_scan_step"); });
        changed(state);
    }
    return THPVariable_Wrap(y);
    END_HANDLE_TH_ERRORS
}

// ---- norm ------------------------------------------------------------------------------------------------------------------------------------
// inputs x, weight, residual; saved: what was normalised and the weight
variable_list norm_backward(double eps, at::ScalarType dt, bool residual, at::ScalarType res_dt, const variable_list& s, const variable_list& grads, const Need& need) {
    const Rows r = rows_of(s[0]);
    const Tensor& w = s[1];
    const int64_t H = s[0].size(-1), rows = row_count(s[0]);
    const at::Device dev = s[0].device();
    const Tensor dy = grads[0].defined() ? aligned(grads[0]) : at::zeros(s[0].sizes(), s[0].options().dtype(dt));
    const Tensor dsum = grads.size() > 1 && grads[1].defined() ? aligned(grads[1]) : Tensor();
    const Tensor wc = aligned(w);
    variable_list out(3);
    out[0] = new_cuda(s[0].sizes(), dt, dev);
    if (residual) out[2] = res_dt == dt ? out[0] : new_cuda(s[0].sizes(), res_dt, dev);      // one gradient for both where they share a type
    Tensor part;
    if (w.defined()) {
        out[1] = new_cuda(w.sizes(), w.scalar_type(), dev);
        if (need(1)) part = new_cuda({mkda_norm_bwd_part_rows((int)rows, (int)H), H}, at::kFloat, dev);
    }
    MkdaNormBwd p{};
    p.rows = (int)rows; p.width = (int)H; p.dtype = dtype_code(out[0]); p.eps = (float)eps;
    p.s = r.t.data_ptr(); p.s_stride = r.stride; p.s_dtype = dtype_code(r.t); p.weight = cptr(wc); p.weight_dtype = w.defined() ? dtype_code(w) : MKDA_F32;
    p.dy = dy.data_ptr(); p.dsum = cptr(dsum); p.dx = out[0].data_ptr(); p.dres = residual && res_dt != dt ? out[2].data_ptr() : nullptr;
    p.part_rows = part.defined() ? (int)part.size(0) : 0; p.part = fmptr(part);
    check_rc(mkda_norm_bwd(&p, stream()), "mkda_norm_bwd");
    if (part.defined()) {
        MkdaSumRows q{};
        q.job[0] = {fptr(part), p.part_rows, 1, H, H, (int)H, (int)H, 0, 0, 1, out[1].data_ptr(), dtype_code(out[1])};
        check_rc(mkda_sum_rows(&q, stream()), "mkda_sum_rows");
    }
    return out;
}

// norm(x, weight, residual, eps, e4m3, group) -> (y, residual sum or None), or (e4m3, scale, residual sum or None)
PyObject* norm(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 6) return fail(PyExc_TypeError, "norm takes 6 arguments");
    variable_list t;
    if (!parse_tensors("rms_norm", a, 3, 1, t)) return nullptr;
    const Tensor &x = t[0], &w = t[1], &res = t[2];
    if (!check_devices("rms_norm", t)) return nullptr;
    REQUIRE(x.dim() >= 1 && float_type(x), "x must be [.., H], bfloat16, float16 or float32");
    const int64_t H = x.size(-1), rows = row_count(x);
    REQUIRE(H >= 1 && H <= MKDA_NORM_MAX_WIDTH, "rows of 1 to 32768 channels");
    REQUIRE(rows <= MOST_TOKENS, "less than 2^31 rows");
    REQUIRE(!w.defined() || (w.dim() == 1 && w.size(0) == H && float_type(w)), "weight must be [H]");
    REQUIRE(!res.defined() || res.sizes() == x.sizes(), "residual must have the shape of x");
    REQUIRE(!res.defined() || res.scalar_type() == x.scalar_type() || res.scalar_type() == at::kFloat, "residual must have the type of x, or be float32");
    const double eps = PyFloat_AsDouble(a[3]);
    const int e4m3 = PyObject_IsTrue(a[4]), group = (int)PyLong_AsLong(a[5]);
    if (PyErr_Occurred()) return nullptr;
    REQUIRE(!group || H % group == 0, "a scale per 128 channels needs rows of a multiple of 128 channels");
    const bool grad = any_requires_grad(t);
    if (grad && e4m3) return fail(PyExc_RuntimeError, "rms_norm: an output in 8 bits has no gradient: call it under torch.no_grad()");
    Tensor y, sum, scale;
    {
        pybind11::gil_scoped_release nogil;
        c10::cuda::CUDAGuard guard(x.device());
        {
            at::AutoGradMode off(false);
            const Rows xr = rows_of(x), rr = rows_of(res);
            const Tensor wc = aligned(w);
            y = new_cuda(x.sizes(), e4m3 ? at::kFloat8_e4m3fn : x.scalar_type(), x.device());
            if (res.defined()) sum = new_cuda(x.sizes(), res.scalar_type(), x.device());
            if (e4m3) {
                std::vector<int64_t> sz(x.sizes().begin(), x.sizes().end());
                sz.back() = group ? H / group : 1;
                scale = new_cuda(sz, at::kFloat, x.device());
            }
            MkdaNormFwd p{};
            p.rows = (int)rows; p.width = (int)H; p.dtype = dtype_code(x); p.res_dtype = res.defined() ? dtype_code(res) : MKDA_F32; p.eps = (float)eps;
            p.x = xr.t.data_ptr(); p.x_stride = xr.stride; p.residual = cptr(rr.t); p.res_stride = rr.stride; p.weight = cptr(wc); p.weight_dtype = w.defined() ? dtype_code(w) : MKDA_F32;
            p.sum = mptr(sum); p.y = y.data_ptr(); p.out_e4m3 = e4m3; p.group = group; p.scale = fmptr(scale);
            library_call([&] { check_rc(mkda_norm_fwd(&p, stream()), "mkda_norm_fwd"); });
        }
        if (grad) {
            const bool has = res.defined();
            const at::ScalarType dt = x.scalar_type(), rdt = has ? res.scalar_type() : dt;
            constexpr uint32_t X = 1, WT = 2, RES = 4;
            auto node = new_node("rms_norm", x.device(), t, {X | WT | RES, X | RES, X | WT | RES}, [eps, dt, has, rdt](const variable_list& s, const variable_list& g, const Need& need) {
                return norm_backward(eps, dt, has, rdt, s, g, need);
            });
            node->state_linear = true;                     // a sum
            torch::autograd::set_history(y, node);
            if (has) torch::autograd::set_history(sum, node);
            node->save(has ? sum : x, has);
            node->save(w);
        }
    }
    if (!e4m3) return pair(y, sum);
    PyObject* py = THPVariable_Wrap(y);
    PyObject* ps = THPVariable_Wrap(scale);
    PyObject* pr = Py_None;
    if (sum.defined()) pr = THPVariable_Wrap(sum);
    else Py_INCREF(pr);
    PyObject* r = py && ps && pr ? PyTuple_Pack(3, py, ps, pr) : nullptr;
    Py_XDECREF(py);
    Py_XDECREF(ps);
    Py_XDECREF(pr);
    return r;
    END_HANDLE_TH_ERRORS
}

}  // namespace

PyMethodDef mkda_host::block_methods[] = {
    {"conv", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(conv)), METH_FASTCALL, "causal convolution"},
    {"conv_step", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(conv_step)), METH_FASTCALL, "one token of a causal convolution"},
    {"scan", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(scan)), METH_FASTCALL, "selective scan"},
    {"scan_step", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(scan_step)), METH_FASTCALL, "one token of a selective scan"},
    {"norm", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(norm)), METH_FASTCALL, "RMS norm"},
    {nullptr, nullptr, 0, nullptr}};
