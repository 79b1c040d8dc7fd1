"""Performance cases of the operators around the delta-rule layer: the short causal convolution in front of it, the selective scan and
the RMS norm with the residual's addition, as training and serving programs call them.

A case is a dict of plain values:

  op        "conv", "conv_step", "scan", "scan_step" or "norm"
  train     forward and backward with dense upstream gradients, else forward only under ``no_grad``
  rows, tokens, docs, doc_seed
            ``rows`` x ``tokens`` with docs = 0; docs > 0: one row of ``tokens`` packed documents with lognormal lengths (median
            ``docs``, sigma 1), addressed by ``cu_seqlens``
  width     channels; dtype of the activations
  taps, bias, act                         the convolution's kernel size and options
  states, groups, skip, gate, softplus    the scan's states per channel, groups of B and C, ``D``, ``z`` and ``dt_softplus`` with ``dt_bias``
  state_in, state_out                     initial states given, final states wanted
  residual, quant                         the norm's residual stream ("" or its type) and output ("", "row" or "group": e4m3 with one scale
                                          per row or per 128 channels)
"""
import math
import random

import torch

own = False
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
#: token-channels of the largest listed cases: a convolution, a scan forward only and with its backward pass, a norm
MOST = {"conv": 32749 * 8192, "scan": 8192 * 4096, "scan_train": 2 * 2048 * 4096, "norm": 65536 * 2048}


def _case(**kw):
    c = dict(op="conv", train=False, rows=1, tokens=1, docs=0, doc_seed=0, width=4096, dtype="bf16", state_in=False, state_out=False)
    if kw["op"].startswith("conv"):
        c.update(taps=4, bias=False, act="silu")
    elif kw["op"].startswith("scan"):
        c.update(states=16, groups=1, skip=True, gate=True, softplus=True)
    else:
        c.update(residual="bf16", quant="")
    c.update(kw)
    return c


def listed():
    return [
        # one more token for each of eight running sequences, through the convolution of 32 heads of 128: latency
        _case(name="conv_step_b8", op="conv_step", rows=8, width=4096),
        # q, k and v of 16 + 16 + 32 heads in one convolution over a long prompt of odd length, state kept for decoding
        _case(name="conv_prefill_32k", op="conv", tokens=32749, width=8192, state_out=True),
        # the same layer trained on packed documents
        _case(name="conv_train_packed_8k", op="conv", train=True, tokens=8192, docs=500, doc_seed=1, width=4096, bias=True),
        # continued rows in fp32 with an odd number of channels, three taps, no activation
        _case(name="conv_train_fp32_4x1000", op="conv", train=True, rows=4, tokens=1000, width=1001, dtype="fp32", taps=3, act="", bias=True,
              state_in=True, state_out=True),
        # one more token for each of 64 running sequences: the states are read and written
        _case(name="scan_step_b64", op="scan_step", rows=64, width=4096),
        # a short prompt of one user
        _case(name="scan_prompt_t77", op="scan", tokens=77, width=2048, state_out=True),
        # a long prompt
        _case(name="scan_prefill_8k", op="scan", tokens=8192, width=4096, state_out=True),
        # a training batch of two rows
        _case(name="scan_train_2x2k", op="scan", train=True, rows=2, tokens=2048, width=4096),
        # packed documents that continue from states, two groups of B and C, no gate, fp32
        _case(name="scan_train_packed_fp32", op="scan", train=True, tokens=4001, docs=300, doc_seed=2, width=1024, dtype="fp32", groups=2,
              gate=False, state_in=True, state_out=True),
        # eight tokens of a decoding batch in front of an 8-bit projection
        _case(name="norm_decode_8_e4m3", op="norm", tokens=8, width=4096, quant="row"),
        # a training batch, residual stream in bf16
        _case(name="norm_train_8k", op="norm", train=True, tokens=8192, width=4096),
        # a long packed prompt in front of an 8-bit projection that takes a scale per 128 channels
        _case(name="norm_prefill_64k_e4m3", op="norm", tokens=65536, width=2048, quant="group"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng):
    """One more case: an operator, a direction and a size over the whole range, the options drawn independently."""
    op = rng.choice(("conv", "conv", "scan", "scan", "norm", "norm", "conv_step", "scan_step"))
    kw = dict(op=op, dtype=rng.choice(("bf16", "bf16", "bf16", "fp16", "fp32")), doc_seed=rng.randrange(1 << 20))
    kw["width"] = rng.choice((128 * rng.randint(1, 32), 8 * rng.randint(8, 512), rng.randint(64, 4096)))
    if op.startswith("conv"):
        kw.update(taps=rng.choice((2, 3, 4, 4)), bias=rng.random() < 0.5, act=rng.choice(("silu", "silu", "")))
    elif op.startswith("scan"):
        kw.update(skip=rng.random() < 0.8, gate=rng.random() < 0.7, softplus=rng.random() < 0.8, states=rng.choice((16, 16, 16, 8, 32, rng.randint(1, 16))))
        kw["groups"] = rng.choice([g for g in (1, 1, 2, 4) if kw["width"] % g == 0])
    if op.endswith("step"):
        kw["rows"] = _log_int(rng, 1, 256)
        return _case(**kw)
    kw["train"] = rng.random() < 0.5
    if op == "norm":
        kw["quant"] = "" if kw["train"] else rng.choice(("", "row", "group"))
        if kw["quant"] == "group":
            kw["width"] = 128 * rng.randint(1, 32)
        kw["residual"] = rng.choice(("", kw["dtype"], kw["dtype"], "fp32"))
        kw["tokens"] = _log_int(rng, 1, MOST["norm"] // kw["width"] // (1 if kw["dtype"] != "fp32" and not kw["train"] else 4))
        return _case(**kw)
    most = MOST["conv"] // (1 if kw["dtype"] != "fp32" and not kw["train"] else 4) if op == "conv" else MOST["scan_train" if kw["train"] else "scan"] * 16 // max(16, kw["states"])
    shape = rng.choice(("one", "rows", "packed"))
    kw["rows"] = rng.choice((2, 3, 4, 8)) if shape == "rows" else 1
    kw["tokens"] = _log_int(rng, 1, min(most // kw["width"] // kw["rows"], 8192 if op == "scan" else 65536))
    if shape == "packed":
        kw["docs"] = _log_int(rng, 4, 1000)
    kw["state_in"], kw["state_out"] = rng.random() < 0.4, rng.random() < 0.5
    return _case(**kw)


def _bounds(c):
    """Boundaries of the packed documents, None without packing."""
    if not c["docs"]:
        return None
    g, cu = random.Random(c["doc_seed"]), [0]
    while cu[-1] < c["tokens"]:
        cu.append(min(cu[-1] + max(int(g.lognormvariate(math.log(c["docs"]), 1.0)), 1), c["tokens"]))
    return cu


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda").manual_seed(seed)
    B, T, D, dt = c["rows"], c["tokens"], c["width"], DTYPES[c["dtype"]]
    cu = _bounds(c)
    n = B if cu is None else len(cu) - 1

    def r(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    def uniform(*shape):
        return torch.rand(*shape, generator=g, device="cuda")

    t = {}
    step = c["op"].endswith("step")
    lead = (B,) if step else (B, T)
    if c["op"].startswith("conv"):
        K = c["taps"]
        t["x"], t["weight"] = r(*lead, D).to(dt), (uniform(D, K) * 2 - 1) * K ** -0.5
        if c["bias"]:
            t["bias"] = 0.1 * r(D)
        if step:
            t["state"] = r(B, K - 1, D).to(dt)
        elif c["state_in"]:
            t["initial_state"] = r(n, K - 1, D).to(dt)
        last = (n, K - 1, D)
    elif c["op"].startswith("scan"):
        N, G = c["states"], c["groups"]
        t["x"] = r(*lead, D).to(dt)
        step_size = torch.exp(uniform(D) * math.log(100.0) + math.log(1e-3))      # 0.001 .. 0.1
        if c["softplus"]:
            t["dt"], t["dt_bias"] = (0.5 * r(*lead, D)).to(dt), step_size + torch.log(-torch.expm1(-step_size))
        else:
            t["dt"] = (step_size * torch.exp(0.5 * r(*lead, D))).to(dt)
        t["A"] = -torch.arange(1, N + 1, device="cuda") * torch.exp(0.1 * r(D, N))
        t["B"], t["C"] = r(*lead, G, N).to(dt), r(*lead, G, N).to(dt)
        if c["skip"]:
            t["D"] = 1 + 0.1 * r(D)
        if c["gate"]:
            t["z"] = r(*lead, D).to(dt)
        if step:
            t["state"] = 0.2 * r(B, D, N)
        elif c["state_in"]:
            t["initial_state"] = 0.2 * r(n, D, N)
        last = (n, D, N)
    else:
        t["x"], t["weight"] = r(T, D).to(dt), 1 + 0.1 * r(D)
        if c["residual"]:
            t["residual"] = (2 * r(T, D)).to(DTYPES[c["residual"]])
    s = dict(case=c, leaves=t, cu=None if cu is None else torch.tensor(cu, dtype=torch.int32, device="cuda"))
    if c["train"]:
        for x in t.values():
            x.requires_grad_(True)
        s["dy"] = r(*t["x"].shape).to(dt)
        if c["op"] == "norm":
            s["dlast"] = r(T, D).to(t["residual"].dtype) if c["residual"] else None
        else:
            s["dlast"] = (0.1 * r(*last)).to(dt if c["op"] == "conv" else torch.float32) if c["state_out"] else None
    return s


# ---- the framework's calls -----------------------------------------------------------------------------------------------------------------
def _own(s):
    import mogankda_b200 as mk
    c, t = s["case"], s["leaves"]
    get = t.get
    if c["op"] == "conv_step":
        y = mk.causal_conv1d_step(t["x"], t["state"], t["weight"], get("bias"), activation=c["act"] or None)
        return dict(y=y, state=t["state"])
    if c["op"] == "scan_step":
        y = mk.selective_scan_step(t["x"], t["dt"], t["A"], t["B"], t["C"], t["state"], get("D"), get("z"), get("dt_bias"), dt_softplus=c["softplus"])
        return dict(y=y, state=t["state"])
    if c["op"] == "conv":
        y, last = mk.causal_conv1d(t["x"], t["weight"], get("bias"), activation=c["act"] or None, initial_state=get("initial_state"),
                                   output_final_state=c["state_out"], cu_seqlens=s["cu"])
    elif c["op"] == "scan":
        y, last = mk.selective_scan(t["x"], t["dt"], t["A"], t["B"], t["C"], get("D"), get("z"), get("dt_bias"), dt_softplus=c["softplus"],
                                    initial_state=get("initial_state"), output_final_state=c["state_out"], cu_seqlens=s["cu"])
    elif c["quant"]:
        got = mk.rms_norm(t["x"], t["weight"], residual=get("residual"), out_dtype=torch.float8_e4m3fn, scale_group=128 if c["quant"] == "group" else None)
        return dict(zip(("y", "scale", "last"), got))
    else:
        got = mk.rms_norm(t["x"], t["weight"], residual=get("residual"))
        y, last = got if c["residual"] else (got, None)
    if not c["train"]:
        return dict(y=y, last=last)
    outs, ups = ((y, last), (s["dy"], s["dlast"])) if last is not None else ((y,), (s["dy"],))
    grads = torch.autograd.grad(outs, list(t.values()), ups)
    return dict({"d" + n: d for n, d in zip(t, grads)}, y=y.detach(), last=None if last is None else last.detach())


# ---- the plain forms: fp32, rounded once at the end ----------------------------------------------------------------------------------------
def _silu(x):
    return x * torch.sigmoid(x)


def _dsilu(x):
    e = torch.sigmoid(x)
    return e * (1 + x * (1 - e))


def _cu(s):
    c = s["case"]
    return s["cu"].long() if s["cu"] is not None else torch.arange(c["rows"] + 1, device="cuda") * c["tokens"]


def _conv(s):
    c, t = s["case"], s["leaves"]
    K, D, n_tok = c["taps"], c["width"], c["rows"] * c["tokens"]
    cu = _cu(s)
    n = len(cu) - 1
    x, w = t["x"].reshape(n_tok, D).float(), t["weight"].float()
    init = t["initial_state"].reshape(n * (K - 1), D).float() if c["state_in"] else x.new_zeros(n * (K - 1), D)
    rows = torch.cat([init, x])                                     # row of token p of sequence q: n (K - 1) + p, of its state: q (K - 1) + j
    tok = torch.arange(n_tok, device="cuda")
    seq = torch.searchsorted(cu, tok, right=True) - 1
    start, end = cu[:-1], cu[1:]

    def row(q, p):
        return torch.where(p >= start[q], n * (K - 1) + p, q * (K - 1) + p - start[q] + K - 1)

    taps = torch.arange(K, device="cuda")
    xs = rows[row(seq[:, None], tok[:, None] - K + 1 + taps)]       # [tokens, K, D]
    pre = (xs * w.t()).sum(1)
    if c["bias"]:
        pre = pre + t["bias"].float()
    y = _silu(pre) if c["act"] else pre
    q, j = torch.arange(n, device="cuda")[:, None], torch.arange(K - 1, device="cuda")
    at = row(q, end[:, None] - K + 1 + j)                           # [n, K - 1]: rows that the final states hold
    out = dict(y=y.view_as(t["x"]).to(t["x"].dtype), last=rows[at].to(t["x"].dtype) if c["state_out"] else None)
    if not c["train"]:
        return out
    dpre = s["dy"].reshape(n_tok, D).float()
    if c["act"]:
        dpre = dpre * _dsilu(pre)
    padded = torch.cat([dpre, dpre.new_zeros(1, D)])

    def back(q, p):                                                 # gradient of the rows at positions p of the sequences q
        to = p[..., None] + K - 1 - taps
        return (padded[torch.where((to >= start[q][..., None]) & (to < end[q][..., None]), to, n_tok)] * w.t()).sum(-2)

    drows = torch.cat([back(q, start[:, None] - K + 1 + j).reshape(-1, D), back(seq, tok)])
    if c["state_out"]:
        drows.index_add_(0, at.reshape(-1), s["dlast"].reshape(-1, D).float())
    out.update(dx=drows[n * (K - 1):].view_as(t["x"]).to(t["x"].dtype), dweight=(dpre[:, None] * xs).sum(0).t().to(t["weight"].dtype))
    if c["bias"]:
        out["dbias"] = dpre.sum(0).to(t["bias"].dtype)
    if c["state_in"]:
        out["dinitial_state"] = drows[:n * (K - 1)].view_as(t["initial_state"]).to(t["x"].dtype)
    return out


def _conv_step(s):
    c, t = s["case"], s["leaves"]
    rows = torch.cat([t["state"], t["x"][:, None]], 1)
    pre = (rows.float() * t["weight"].float().t()).sum(1)
    if c["bias"]:
        pre = pre + t["bias"].float()
    t["state"].copy_(rows[:, 1:])
    return dict(y=(_silu(pre) if c["act"] else pre).to(t["x"].dtype), state=t["state"])


def _linear_scan(a, b):
    """h[t] = a[t] h[t - 1] + b[t] along the first axis, from zero: neighbours joined, half the length solved, the even places filled in."""
    n = a.shape[0]
    if n == 1:
        return b
    m = n // 2 * 2
    odd = _linear_scan(a[1:m:2] * a[0:m:2], b[1:m:2] + a[1:m:2] * b[0:m:2])
    h = torch.empty_like(b)
    h[1:m:2] = odd
    h[0] = b[0]
    h[2::2] = b[2::2] + a[2::2] * odd[:(n - 1) // 2]
    return h


def _scan(s):
    c, t = s["case"], s["leaves"]
    D, N, G, n_tok = c["width"], c["states"], c["groups"], c["rows"] * c["tokens"]
    cu = _cu(s)
    some = torch.nonzero(cu[1:] > cu[:-1]).view(-1)                 # sequences that are not empty
    first, final = cu[some], cu[some + 1] - 1
    flat = {k: t[k].reshape(n_tok, -1).float() for k in ("x", "dt", "z") if k in t}
    x, raw, A = flat["x"], flat["dt"], t["A"].float()
    if c["softplus"]:
        raw = raw + t["dt_bias"].float()
    d = torch.clamp(raw, min=0) + torch.log1p(torch.exp(-raw.abs())) if c["softplus"] else raw

    def spread(v):                                                  # [tokens, G, N] -> [tokens, D, N]
        return v.reshape(n_tok, G, 1, N).float().expand(n_tok, G, D // G, N).reshape(n_tok, D, N)

    a = torch.exp(d[:, :, None] * A)
    b = (d * x)[:, :, None] * spread(t["B"])
    if c["state_in"]:
        b[first] += a[first] * t["initial_state"][some].float()
    cut = a.clone()
    cut[first] = 0
    h = _linear_scan(cut, b)
    del b
    y0 = (h * spread(t["C"])).sum(-1)
    if c["skip"]:
        y0 = y0 + t["D"].float() * x
    y = y0 * _silu(flat["z"]) if c["gate"] else y0
    out = dict(y=y.view_as(t["x"]).to(t["x"].dtype), last=None)
    if c["state_out"]:
        last = t["initial_state"].detach().float().clone() if c["state_in"] else x.new_zeros(len(cu) - 1, D, N)
        last[some] = h[final]
        out["last"] = last
    if not c["train"]:
        return out
    dy = s["dy"].reshape(n_tok, D).float()
    if c["gate"]:
        out["dz"] = (dy * y0 * _dsilu(flat["z"])).view_as(t["x"]).to(t["x"].dtype)
        dy = dy * _silu(flat["z"])
    g = dy[:, :, None] * spread(t["C"])
    if c["state_out"]:
        g[final] += s["dlast"][some]
    after = torch.cat([cut[1:], torch.zeros_like(cut[:1])])         # the decay that takes the state of this token to the next one's
    g = _linear_scan(after.flip(0), g.flip(0)).flip(0)
    del after

    def gathered(v):                                                # [tokens, D, N] -> [tokens, G, N]
        return v.view(n_tok, G, D // G, N).sum(2)

    out["dC"] = gathered(dy[:, :, None] * h).view_as(t["C"]).to(t["x"].dtype)
    out["dB"] = gathered((d * x)[:, :, None] * g).view_as(t["B"]).to(t["x"].dtype)
    gb = (g * spread(t["B"])).sum(-1)
    before = torch.cat([torch.zeros_like(h[:1]), h[:-1]])
    before[first] = t["initial_state"][some].float() if c["state_in"] else 0.0
    if c["state_in"]:
        dinit = torch.zeros_like(t["initial_state"]) if not c["state_out"] else s["dlast"].clone()
        dinit[some] = a[first] * g[first]
        out["dinitial_state"] = dinit
    e = g * a * before
    del g, a, before, h, cut
    draw_ = x * gb + (e * A).sum(-1)
    out["dA"] = (e * d[:, :, None]).sum(0).to(t["A"].dtype)
    dx = d * gb
    if c["skip"]:
        dx = dx + t["D"].float() * dy
        out["dD"] = (dy * x).sum(0).to(t["D"].dtype)
    if c["softplus"]:
        draw_ = draw_ * torch.sigmoid(raw)
        out["ddt_bias"] = draw_.sum(0).to(t["dt_bias"].dtype)
    out.update(dx=dx.view_as(t["x"]).to(t["x"].dtype), ddt=draw_.view_as(t["dt"]).to(t["dt"].dtype))
    return out


def _scan_step(s):
    c, t = s["case"], s["leaves"]
    D, N, G, n = c["width"], c["states"], c["groups"], c["rows"]
    x, d = t["x"].float(), t["dt"].float()
    if c["softplus"]:
        d = d + t["dt_bias"].float()
        d = torch.clamp(d, min=0) + torch.log1p(torch.exp(-d.abs()))

    def spread(v):
        return v[:, :, None].float().expand(n, G, D // G, N).reshape(n, D, N)

    h = torch.exp(d[:, :, None] * t["A"]) * t["state"] + (d * x)[:, :, None] * spread(t["B"])
    t["state"].copy_(h)
    y = (h * spread(t["C"])).sum(-1)
    if c["skip"]:
        y = y + t["D"] * x
    if c["gate"]:
        y = y * _silu(t["z"].float())
    return dict(y=y.to(t["x"].dtype), state=t["state"])


def _norm(s):
    c, t = s["case"], s["leaves"]
    x, w = t["x"].float(), t["weight"].float()
    last = None
    if c["residual"]:                                               # the residual stream, in its type: what is normalised is what it holds
        last = (x + t["residual"].float()).to(t["residual"].dtype)
        x = last.float()
    r = torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6)
    y = x * r * w
    if c["quant"]:
        v = y.view(c["tokens"], -1, 128) if c["quant"] == "group" else y.view(c["tokens"], 1, -1)
        scale = torch.clamp(v.abs().amax(-1, keepdim=True), min=torch.finfo(torch.float32).tiny * 448) / 448
        q = (v / scale).view_as(y).to(torch.float8_e4m3fn)
        return dict(y=q, scale=scale.squeeze(-1), last=last)
    out = dict(y=y.to(t["x"].dtype), last=last)
    if not c["train"]:
        return out
    dy = s["dy"].float()
    dn = dy * w
    ds = r * (dn - x * r * r * (dn * x).mean(-1, keepdim=True))
    if c["residual"]:
        ds = ds + s["dlast"].float()
        out["dresidual"] = ds.to(t["residual"].dtype)
    out.update(dx=ds.to(t["x"].dtype), dweight=(dy * x * r).sum(0).to(t["weight"].dtype))
    return out


def run(state):
    op, train = state["case"]["op"], state["case"]["train"]
    if own:
        with torch.set_grad_enabled(train):
            return _own(state)
    with torch.no_grad():
        return {"conv": _conv, "conv_step": _conv_step, "scan": _scan, "scan_step": _scan_step, "norm": _norm}[op](state)


# ---- the definitions in 64 bits: sequence by sequence and token by token, gradients by torch's differentiation ------------------------------------
def exact(case, seed):
    c, s = case, prepare(case, seed)
    t = {k: v.detach().double().requires_grad_(c["train"]) for k, v in s["leaves"].items()}
    cu = _bounds(c)
    spans = [(b, 0, c["tokens"]) for b in range(c["rows"])] if cu is None else [(0, p, q) for p, q in zip(cu[:-1], cu[1:])]

    def scan_token(x, dt, B, C, z, h):          # one token of each row: x, dt, z [rows, D], B and C [rows, G, N], h [rows, D, N]
        d = torch.nn.functional.softplus(dt + t["dt_bias"], threshold=1000) if c["softplus"] else dt
        per = c["width"] // c["groups"]
        h = torch.exp(d.unsqueeze(-1) * t["A"]) * h + (d * x).unsqueeze(-1) * B.repeat_interleave(per, 1)
        y = torch.einsum("bdn,bdn->bd", h, C.repeat_interleave(per, 1))
        y = y + t["D"] * x if c["skip"] else y
        return (y * torch.nn.functional.silu(z) if c["gate"] else y), h

    def scan():
        ys, hs = [], []
        for i, (b, p, q) in enumerate(spans if cu is not None else [(0, 0, c["tokens"])]):
            b, i = (slice(None), slice(None)) if cu is None else (slice(0, 1), slice(i, i + 1))      # equal rows go together
            h = t["initial_state"][i] if c["state_in"] else t["x"].new_zeros(c["rows"], c["width"], c["states"])
            part = {k: t[k][b, p:q].unbind(1) for k in ("x", "dt", "B", "C", "z") if k in t}
            for j in range(q - p):
                y, h = scan_token(part["x"][j], part["dt"][j], part["B"][j], part["C"][j], part["z"][j] if c["gate"] else None, h)
                ys.append(y)
            hs.append(h)
        return torch.stack(ys, 1), torch.cat(hs) if c["state_out"] else None

    def conv():
        ys, last = [], []
        for i, (b, p, q) in enumerate(spans):
            head = t["initial_state"][i] if c["state_in"] else t["x"].new_zeros(c["taps"] - 1, c["width"])
            seq = torch.cat([head, t["x"][b, p:q]])
            y = torch.nn.functional.conv1d(seq.t()[None], t["weight"][:, None], t.get("bias"), groups=c["width"])[0].t()
            ys.append(torch.nn.functional.silu(y) if c["act"] else y)
            last.append(seq[q - p:])
        return torch.cat(ys).view_as(t["x"]), torch.stack(last) if c["state_out"] else None

    def norm():
        v, last = t["x"], None
        if c["residual"]:
            v = v + t["residual"]
            last = v = v + (v.detach().to(s["leaves"]["residual"].dtype).double() - v.detach())      # rounded; its derivative is one
        return v / torch.sqrt(torch.mean(v * v, -1, keepdim=True) + 1e-6) * t["weight"], last

    with torch.set_grad_enabled(c["train"]):
        if c["op"] == "conv_step":
            rows = torch.cat([t["state"], t["x"][:, None]], 1)
            y = torch.einsum("bkd,dk->bd", rows, t["weight"]) + t.get("bias", 0)
            return dict(y=torch.nn.functional.silu(y) if c["act"] else y, state=rows[:, 1:])
        if c["op"] == "scan_step":
            y, h = scan_token(t["x"], t["dt"], t["B"], t["C"], t.get("z"), t["state"])
            return dict(y=y, state=h)
        y, last = {"conv": conv, "scan": scan, "norm": norm}[c["op"]]()
    if c["op"] == "norm" and c["quant"]:
        parts = y.reshape(c["tokens"], -1, 128 if c["quant"] == "group" else c["width"])
        scale = parts.abs().amax(-1) / 448
        return dict(y=(parts / scale[..., None]).view_as(y), scale=scale, last=last)
    if not c["train"]:
        return dict(y=y, last=last)
    outs, ups = ((y, last), (s["dy"].double(), s["dlast"].double())) if last is not None else ((y,), (s["dy"].double(),))
    grads = torch.autograd.grad(outs, list(t.values()), ups, allow_unused=True)
    grads = {"d" + n: torch.zeros_like(t[n]) if d is None else d for n, d in zip(t, grads)}
    return dict(grads, y=y.detach(), last=None if last is None else last.detach())


def work(case):
    """Each input read once, each output written once (a backward pass: upstream gradients in, one gradient per input out); the operations of
    the definitions, an exponential as one, no recomputation."""
    c = case
    n, D = c["rows"] * c["tokens"], c["width"]
    e = DTYPES[c["dtype"]].itemsize
    cu = _bounds(c)
    seqs = c["rows"] if cu is None else len(cu) - 1
    if c["op"] == "norm":
        stream = DTYPES[c["residual"]].itemsize if c["residual"] else 0
        inputs = n * D * (e + stream) + 4 * D
        outputs = n * D * ((1 if c["quant"] else e) + stream)
        if c["quant"]:
            outputs += 4 * n * (D // 128 if c["quant"] == "group" else 1)
        return {"bytes": (inputs + outputs) * (2 if c["train"] else 1), "flops": n * D * (16 if c["train"] else 6)}
    if c["op"].startswith("conv"):
        K = c["taps"]
        state = seqs * (K - 1) * D * e
        inputs, outputs = n * D * e + 4 * D * (K + c["bias"]), n * D * e
        flops = n * D * (2 * K + 6) * (3 if c["train"] else 1)
    else:
        N = c["states"]
        state = 4 * seqs * D * N
        inputs = n * e * ((3 if c["gate"] else 2) * D + 2 * c["groups"] * N) + 4 * D * (N + c["skip"] + c["softplus"])
        outputs = n * D * e
        flops = n * D * (7 * N + 12) * (3 if c["train"] else 1)
    step = c["op"].endswith("step")
    inputs += state * (step or c["state_in"])
    outputs += state * (step or c["state_out"])
    return {"bytes": (inputs + outputs) * (2 if c["train"] else 1), "flops": flops}
