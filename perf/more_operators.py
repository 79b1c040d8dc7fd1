"""Performance cases of the linear attention with a decay for each head and of what stands in front of it and behind it in a block of a model: rotary
positions with several axes, and the layer norm of rows or of each head's part of them; as training and serving programs call them.

A case is a dict of plain values:

  op        "linear", "linear_step", "norm" or "rotary"
  train     forward and backward with dense upstream gradients, else forward only under ``no_grad``
  rows, tokens, docs, doc_seed
            ``rows`` x ``tokens`` with docs = 0; docs > 0: one row of ``tokens`` packed documents with lognormal lengths (median
            ``docs``, sigma 1), addressed by ``cu_seqlens``
  dtype     of the activations
  heads, kv_heads
            linear: v-heads, and the q/k-heads that they share in groups; rotary: heads of q, and of k
  dim, v_dim                              channels of a head of q and k, and of v
  state_in, state_out                     initial states given, final states wanted
  width, groups, affine, residual         the norm's channels, the parts of a row that are normalised by themselves, "", "weight" or "both"
                                          (weight and bias), and the type of its residual stream ("" without)
  axes, rotated, interleaved, far         position axes, rotated channels of a head, pairs of neighbours instead of halves, the first position
"""
import math
import random

import torch

own = False
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
#: token-channels of the largest listed cases, of the v-heads: forward only, with a backward pass; of a norm; of q in a rotary call
MOST = {"linear": 32749 * 32 * 128, "linear_train": 8192 * 16 * 128, "norm": 65536 * 2048, "rotary": 32749 * 32 * 128}
CHUNK = 128


def _case(**kw):
    c = dict(op="linear", train=False, rows=1, tokens=1, docs=0, doc_seed=0, dtype="bf16")
    if kw["op"].startswith("linear"):
        c.update(heads=16, kv_heads=0, dim=128, v_dim=128, state_in=False, state_out=False)
    elif kw["op"] == "norm":
        c.update(width=4096, groups=1, affine="both", residual="")
    else:
        c.update(heads=32, kv_heads=8, dim=128, axes=1, rotated=128, interleaved=False, far=0)
    c.update(kw)
    if c["op"].startswith("linear") and not c["kv_heads"]:
        c["kv_heads"] = c["heads"]
    return c


def listed():
    return [
        # one more token for each of 64 running sequences: the states are read and written
        _case(name="linear_step_b64", op="linear_step", rows=64, heads=32),
        # a short prompt of one user: latency
        _case(name="linear_prompt_t77", op="linear", tokens=77, heads=16, state_out=True),
        # a long prompt of odd length, two v-heads to a head of q and k
        _case(name="linear_prefill_32k", op="linear", tokens=32749, heads=32, kv_heads=16, state_out=True),
        # packed documents in training
        _case(name="linear_train_packed_8k", op="linear", train=True, tokens=8192, docs=500, doc_seed=1, heads=16),
        # continued rows in fp32 with smaller heads
        _case(name="linear_train_fp32_4x1000", op="linear", train=True, rows=4, tokens=1000, heads=8, dim=64, v_dim=64, dtype="fp32", state_in=True, state_out=True),
        # the norm of a decoding batch, with the residual's addition: latency
        _case(name="norm_decode_8", op="norm", tokens=8, residual="bf16"),
        # a training batch, residual stream in bf16
        _case(name="norm_train_8k", op="norm", train=True, tokens=8192, residual="bf16"),
        # the outputs of 32 heads in training, each head by itself, odd number of tokens
        _case(name="norm_heads_train_8k", op="norm", train=True, tokens=8191, groups=32, affine="weight"),
        # a long packed prompt
        _case(name="norm_prefill_64k", op="norm", tokens=65536, width=2048, dtype="fp16"),
        # queries and keys of a decoding batch, far into their sequences
        _case(name="rotary_decode_64", op="rotary", rows=64, tokens=1, far=100000),
        # time, height and width of a video's tokens in training
        _case(name="rotary_video_train_8k", op="rotary", train=True, tokens=8192, heads=16, kv_heads=16, axes=3),
        # a long prompt of odd length, half of each head's channels turned, in neighbouring pairs
        _case(name="rotary_prefill_32k", op="rotary", tokens=32749, rotated=64, interleaved=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng):
    """One more case: an operator, a direction and a size over the whole range, the options drawn independently."""
    op = rng.choice(("linear", "linear", "linear", "linear_step", "norm", "norm", "rotary", "rotary"))
    kw = dict(op=op, dtype=rng.choice(("bf16", "bf16", "bf16", "fp16", "fp32")), doc_seed=rng.randrange(1 << 20), train=op != "linear_step" and rng.random() < 0.5)
    if op.startswith("linear"):
        kw["kv_heads"] = rng.choice((1, 2, 4, 8, 16, 16, rng.randint(1, 24)))
        kw["heads"] = kw["kv_heads"] * rng.choice((1, 1, 1, 2))
        kw["dim"] = rng.choice((128, 128, 128, 64, 8 * rng.randint(4, 16)))
        kw["v_dim"] = rng.choice((kw["dim"], kw["dim"], 128, 64))
        if op == "linear_step":
            kw["rows"] = _log_int(rng, 1, 64)
            return _case(**kw)
        most = MOST["linear_train" if kw["train"] else "linear"] // (4 if kw["dtype"] == "fp32" else 1) // (kw["heads"] * 128)
        shape = rng.choice(("one", "rows", "packed"))
        kw["rows"] = rng.choice((2, 3, 4, 8)) if shape == "rows" else 1
        kw["tokens"] = _log_int(rng, 1, min(max(most // kw["rows"], 16), 32768))
        if shape == "packed":
            kw["docs"] = _log_int(rng, 32, 2000)
        kw["state_in"], kw["state_out"] = rng.random() < 0.4, rng.random() < 0.5
        return _case(**kw)
    if op == "norm":
        kw["groups"] = rng.choice((1, 1, 1, 8, 16, 32))
        kw["width"] = kw["groups"] * rng.choice((64, 128, 128, 8 * rng.randint(4, 32))) if kw["groups"] > 1 else rng.choice((128 * rng.randint(1, 64), 8 * rng.randint(8, 1024), rng.randint(64, 8192)))
        kw["affine"] = rng.choice(("", "weight", "both", "both"))
        kw["residual"] = rng.choice(("", "", kw["dtype"], kw["dtype"], "fp32"))
        kw["tokens"] = _log_int(rng, 1, min(MOST["norm"] // kw["width"] // (1 if kw["dtype"] != "fp32" and not kw["train"] else 4), 65536))
        return _case(**kw)
    kw["dim"] = rng.choice((128, 128, 64, 2 * rng.randint(20, 96)))
    kw["rotated"] = rng.choice((kw["dim"], kw["dim"], 2 * rng.randint(1, kw["dim"] // 2)))
    kw["interleaved"] = rng.random() < 0.4
    kw["axes"] = rng.choice((1, 1, 2, 3))
    kw["heads"], kw["kv_heads"] = rng.choice((8, 16, 32, rng.randint(1, 40))), rng.choice((0, 1, 4, 8, 16))
    kw["far"] = rng.choice((0, 0, 1000, 1000000))
    most = MOST["rotary"] // (4 if kw["dtype"] == "fp32" or kw["train"] else 1) // ((kw["heads"] + kw["kv_heads"]) * 128)
    kw["rows"] = rng.choice((1, 1, 2, 8))
    kw["tokens"] = _log_int(rng, 1, min(max(most // kw["rows"], 1), 32768))
    return _case(**kw)


def _bounds(c):
    """Boundaries of the packed documents, None without packing."""
    if not c["docs"]:
        return None
    g, cu = random.Random(c["doc_seed"]), [0]
    while cu[-1] < c["tokens"]:
        cu.append(min(cu[-1] + max(int(g.lognormvariate(math.log(c["docs"]), 1.0)), 1), c["tokens"]))
    return cu


def _axes(c):
    """The axis of each frequency: neighbouring parts of nearly equal size, the last axis' the largest."""
    n = c["rotated"] // 2
    return [min(f * c["axes"] // max(n, 1), c["axes"] - 1) for f in range(n)]


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda").manual_seed(seed)
    B, T, dt = c["rows"], c["tokens"], DTYPES[c["dtype"]]
    cu = _bounds(c)
    n = B if cu is None else len(cu) - 1

    def r(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    t, s = {}, dict(case=c, cu=None if cu is None else torch.tensor(cu, dtype=torch.int32, device="cuda"))
    if c["op"].startswith("linear"):
        H, HK, K, V = c["heads"], c["kv_heads"], c["dim"], c["v_dim"]
        lead = (B,) if c["op"] == "linear_step" else (B, T)
        t["q"], t["k"], t["v"] = r(*lead, HK, K).to(dt), r(*lead, HK, K).to(dt), r(*lead, H, V).to(dt)
        # memories of a few tokens up to many thousands, over the heads
        s["log_decay"] = -torch.exp2(-10 * (torch.arange(H, device="cuda") + 1) / H) * torch.exp(0.1 * r(H))
        if c["op"] == "linear_step":
            t["state"] = r(B, H, K, V)
        elif c["state_in"]:
            t["initial_state"] = r(n, H, K, V)
        ups = dict(dy=r(*lead, H, V).to(dt)) if c["train"] else {}
        if c["train"] and c["state_out"]:
            ups["dlast"] = 0.1 * r(n, H, K, V)
    elif c["op"] == "norm":
        W = c["width"]
        t["x"] = (r(T, W) + 0.5 * r(T, 1)).to(dt)
        if c["affine"]:
            t["weight"] = 1 + 0.1 * r(W)
        if c["affine"] == "both":
            t["bias"] = 0.1 * r(W)
        if c["residual"]:
            t["residual"] = (2 * r(T, W)).to(DTYPES[c["residual"]])
        ups = dict(dy=r(T, W).to(dt)) if c["train"] else {}
        if c["train"] and c["residual"]:
            ups["dlast"] = r(T, W).to(t["residual"].dtype)
    else:
        D, n_f = c["dim"], c["rotated"] // 2
        t["q"] = r(B, T, c["heads"], D).to(dt)
        if c["kv_heads"]:
            t["k"] = r(B, T, c["kv_heads"], D).to(dt)
        s["inv_freq"] = (10000.0 ** (-torch.arange(n_f, device="cuda", dtype=torch.float64) / max(n_f, 1))).float()
        at = torch.arange(T, device="cuda")[None] + c["far"] + torch.randint(0, 64, (B, 1), generator=g, device="cuda")
        if c["axes"] == 1:
            s["positions"] = at
        elif c["axes"] == 2:
            s["positions"] = torch.stack([at // 64, at % 64])
        else:
            s["positions"] = torch.stack([at // 1024, at // 32 % 32, at % 32])
        s["axes"] = None if c["axes"] == 1 else _axes(c)
        ups = dict(dy=r(*t["q"].shape).to(dt)) if c["train"] else {}
        if c["train"] and c["kv_heads"]:
            ups["dlast"] = r(*t["k"].shape).to(dt)
    if c["train"]:
        for x in t.values():
            x.requires_grad_(True)
    return dict(s, leaves=t, dy=ups.get("dy"), dlast=ups.get("dlast"))


# ---- the framework's calls -----------------------------------------------------------------------------------------------------------------
def _own(s):
    import mogankda_b200 as mk
    c, t = s["case"], s["leaves"]
    get = t.get
    if c["op"] == "linear_step":
        y = mk.linear_attention_step(t["q"], t["k"], t["v"], s["log_decay"], t["state"])
        return dict(y=y, last=t["state"])
    if c["op"] == "linear":
        y, last = mk.linear_attention(t["q"], t["k"], t["v"], s["log_decay"], initial_state=get("initial_state"), output_final_state=c["state_out"], cu_seqlens=s["cu"])
    elif c["op"] == "norm":
        got = mk.layer_norm(t["x"], get("weight"), get("bias"), residual=get("residual"), groups=c["groups"])
        y, last = got if c["residual"] else (got, None)
    else:
        got = mk.rotary(t["q"], get("k"), s["positions"], s["inv_freq"], axes=s["axes"], interleaved=c["interleaved"])
        y, last = got if c["kv_heads"] else (got, None)
    if not c["train"]:
        return dict(y=y, last=last)
    outs, ups = ((y, last), (s["dy"], s["dlast"])) if last is not None else ((y,), (s["dy"],))
    grads = torch.autograd.grad(outs, list(t.values()), ups)
    return dict({"d" + n: d for n, d in zip(t, grads)}, y=y.detach(), last=None if last is None else last.detach())


# ---- the plain forms: fp32, rounded once at the end ----------------------------------------------------------------------------------------
def _chunks(s):
    """The chunks of all sequences: sequence, first token and length of each, the tokens of each [chunks, CHUNK] (the last row stands for none), and the boundaries."""
    c = s["case"]
    cu = s["cu"].long() if s["cu"] is not None else torch.arange(c["rows"] + 1, device="cuda") * c["tokens"]
    per = (cu[1:] - cu[:-1] + CHUNK - 1) // CHUNK
    seq = torch.repeat_interleave(torch.arange(len(per), device="cuda"), per)
    first = cu[seq] + (torch.arange(len(seq), device="cuda") - (torch.cumsum(per, 0) - per)[seq]) * CHUNK
    length = torch.minimum(cu[seq + 1] - first, torch.full_like(first, CHUNK))
    j = torch.arange(CHUNK, device="cuda")
    rows = torch.where(j < length[:, None], first[:, None] + j, c["rows"] * c["tokens"])
    return dict(cu=cu, seq=seq, first=first, length=length, rows=rows)


def _mix(ch, gamma, a, b, c, state, back):
    """out[i] = sum_j exp(gamma |i - j|) (a[i] . b[j]) c[j] over j <= i (``back``: j >= i) of the same sequence, and what ``state`` [sequences, H, .., ..] in front
    of it (behind it) adds; a, b, c [tokens, H, .].  Returns out and the state behind (in front of) each sequence."""
    rate = gamma.double()

    def decay(n):                                                   # [H, ..] of a number of tokens
        return torch.exp(rate.view(-1, *(1,) * n.dim()) * n.clamp(min=0)).float()

    def chunked(x):                                                 # [H, chunks, CHUNK, .]
        return torch.cat([x, x.new_zeros(1, *x.shape[1:])])[ch["rows"]].permute(2, 0, 1, 3)

    H = a.shape[1]
    seq, first, length, cu = ch["seq"], ch["first"], ch["length"], ch["cu"]
    end = first + length
    j = torch.arange(CHUNK, device="cuda")
    away = j - j[:, None] if back else j[:, None] - j
    A, B, C = chunked(a), chunked(b), chunked(c)
    out = ((A @ B.transpose(-1, -2)) * torch.where(away >= 0, decay(away), 0.0)[:, None]) @ C
    left = (length[:, None] - 1 - j).clamp(min=0)                   # tokens of the chunk behind j
    sums = (B * decay(j + 1 if back else left).reshape(H, -1, CHUNK, 1)).transpose(-1, -2) @ C
    # from the chunks in front (behind) and from the state to each chunk's border, and to the sequence's other end
    other = first > first[:, None] if back else first < first[:, None]
    gap = first - end[:, None] if back else first[:, None] - end    # tokens between this chunk and the other one
    to_chunk = torch.where((seq == seq[:, None]) & other, decay(gap), 0.0)
    near = torch.einsum("hcd,hdn->hcn", to_chunk, sums.flatten(2))
    n_seq = len(cu) - 1
    to_end = torch.where(seq == torch.arange(n_seq, device="cuda")[:, None], decay(first[None, :] - cu[:-1, None] if back else cu[1:, None] - end[None, :]), 0.0)
    last = torch.einsum("hsd,hdn->shn", to_end, sums.flatten(2)).reshape(n_seq, *sums.shape[:1], *sums.shape[2:])
    if state is not None:
        near = near + decay(cu[seq + 1] - end if back else first - cu[seq])[..., None] * state[seq].transpose(0, 1).flatten(2)
        last = last + decay(cu[1:] - cu[:-1]).t()[..., None, None] * state
    out = out + (A * decay(left if back else j + 1).reshape(H, -1, CHUNK, 1)) @ near.view_as(sums)
    flat = torch.zeros(a.shape[0] + 1, H, c.shape[-1], device="cuda")
    flat[ch["rows"].reshape(-1)] = out.permute(1, 2, 0, 3).reshape(-1, H, c.shape[-1])
    return flat[:-1], last


def _linear(s):
    c, t = s["case"], s["leaves"]
    n_tok, H, HK, K, V = c["rows"] * c["tokens"], c["heads"], c["kv_heads"], c["dim"], c["v_dim"]
    scale, per = K ** -0.5, H // HK
    ch, gamma = _chunks(s), s["log_decay"]
    q = t["q"].reshape(n_tok, HK, K).float().repeat_interleave(per, 1) * scale
    k, v = t["k"].reshape(n_tok, HK, K).float().repeat_interleave(per, 1), t["v"].reshape(n_tok, H, V).float()
    state = t["initial_state"].float() if c["state_in"] else None
    y, last = _mix(ch, gamma, q, k, v, state, False)
    out = dict(y=y.view_as(t["v"]).to(t["v"].dtype), last=last if c["state_out"] else None)
    if not c["train"]:
        return out
    do = s["dy"].reshape(n_tok, H, V).float()
    up = s["dlast"] if c["state_out"] else None
    dq, _ = _mix(ch, gamma, do, v, k, None if state is None else state.transpose(-1, -2), False)
    dk, _ = _mix(ch, gamma, v, do, q, None if up is None else up.transpose(-1, -2), True)
    dv, dstate = _mix(ch, gamma, k, q, do, up, True)

    def shared(x):
        return x.view(n_tok, HK, per, K).sum(2).view_as(t["q"]).to(t["q"].dtype)

    out.update(dq=shared(dq * scale), dk=shared(dk), dv=dv.view_as(t["v"]).to(t["v"].dtype))
    if c["state_in"]:
        out["dinitial_state"] = dstate
    return out


def _linear_step(s):
    c, t = s["case"], s["leaves"]
    per = c["heads"] // c["kv_heads"]
    q, k = (t[n].float().repeat_interleave(per, 1) for n in ("q", "k"))
    h = torch.exp(s["log_decay"])[:, None, None] * t["state"] + k[..., None] * t["v"].float()[..., None, :]
    t["state"].copy_(h)
    return dict(y=((q * c["dim"] ** -0.5)[..., None] * h).sum(-2).to(t["v"].dtype), last=t["state"])


def _norm(s):
    c, t = s["case"], s["leaves"]
    T, W, G = c["tokens"], c["width"], c["groups"]
    x, last = t["x"].float(), None
    if c["residual"]:                                               # the residual stream, in its type: what is normalised is what it holds
        last = (x + t["residual"].float()).to(t["residual"].dtype)
        x = last.float()
    x = x.view(T, G, W // G)
    d = x - x.mean(-1, keepdim=True)
    r = torch.rsqrt(d.square().mean(-1, keepdim=True) + 1e-5)
    xh = (d * r).view(T, W)
    y = xh * t["weight"] if c["affine"] else xh
    if c["affine"] == "both":
        y = y + t["bias"]
    out = dict(y=y.to(t["x"].dtype), last=last)
    if not c["train"]:
        return out
    dy = s["dy"].float()
    dn = (dy * t["weight"] if c["affine"] else dy).view(T, G, W // G)
    h = xh.view_as(dn)
    ds = (r * (dn - dn.mean(-1, keepdim=True) - h * (dn * h).mean(-1, keepdim=True))).view(T, W)
    if c["residual"]:
        ds = ds + s["dlast"].float()
        out["dresidual"] = ds.to(t["residual"].dtype)
    out["dx"] = ds.to(t["x"].dtype)
    if c["affine"]:
        out["dweight"] = (dy * xh).sum(0)
    if c["affine"] == "both":
        out["dbias"] = dy.sum(0)
    return out


def _turned(x, cos, sin, interleaved):
    n = cos.shape[-1]
    x = x.float()
    part, rest = x[..., :2 * n], x[..., 2 * n:]
    a, b = (part[..., 0::2], part[..., 1::2]) if interleaved else (part[..., :n], part[..., n:])
    a, b = a * cos - b * sin, a * sin + b * cos
    return torch.cat([torch.stack([a, b], -1).flatten(-2) if interleaved else torch.cat([a, b], -1), rest], -1)


def _rotary(s):
    c, t = s["case"], s["leaves"]
    at = s["positions"] if c["axes"] == 1 else s["positions"][torch.tensor(s["axes"], device="cuda", dtype=torch.long)].permute(1, 2, 0)
    angle = (at[..., None] if c["axes"] == 1 else at).double() * s["inv_freq"].double()      # 32 bits lose the angles of far positions
    cos, sin = torch.cos(angle).float()[:, :, None], torch.sin(angle).float()[:, :, None]
    names = [n for n in ("q", "k") if n in t]
    out = dict(zip(("y", "last"), [_turned(t[n], cos, sin, c["interleaved"]).to(t[n].dtype) for n in names]))
    if c["train"]:
        out.update({"d" + n: _turned(s[u], cos, -sin, c["interleaved"]).to(t[n].dtype) for n, u in zip(names, ("dy", "dlast"))})
    return dict(out, last=out.get("last"))


def run(state):
    op, train = state["case"]["op"], state["case"]["train"]
    if own:
        with torch.set_grad_enabled(train):
            return _own(state)
    with torch.no_grad():
        return {"linear": _linear, "linear_step": _linear_step, "norm": _norm, "rotary": _rotary}[op](state)


# ---- the definitions in 64 bits: every pair of tokens of a sequence, gradients by torch's differentiation ----------------------------------------
def _exact_linear(c, s, t):
    cu = _bounds(c)
    H, HK = c["heads"], c["kv_heads"]
    per, scale, rate = H // HK, c["dim"] ** -0.5, s["log_decay"].double()
    flat = {k: v.detach().reshape(-1, *v.shape[2:]) for k, v in t.items() if k in "qkv"}
    spans = [(b * c["tokens"], (b + 1) * c["tokens"]) for b in range(c["rows"])] if cu is None else list(zip(cu[:-1], cu[1:]))
    y = torch.zeros_like(flat["v"])
    grads = {"d" + k: torch.zeros_like(v) for k, v in flat.items()} if c["train"] else {}
    lasts = torch.zeros(len(spans), H, c["dim"], c["v_dim"], dtype=torch.float64, device="cuda")
    dinit = torch.zeros_like(lasts)
    for n, (p, e) in enumerate(spans):
        T = e - p
        at = torch.arange(T, device="cuda", dtype=torch.float64)
        some = max(1, (1 << 27) // max(T * T, 1))                   # heads at a time; a head in blocks of rows where there are many tokens
        block = T if T <= 8192 else 2048
        for h0 in range(0, H, some):
            hs = torch.arange(h0, min(h0 + some, H), device="cuda")
            part = {k: flat[k][p:e][:, hs // per if k != "v" else hs].transpose(0, 1).clone().requires_grad_(c["train"]) for k in "qkv"}      # [heads, T, .]
            g = rate[hs][:, None]
            init = t["initial_state"].detach()[n][hs].clone().requires_grad_(c["train"]) if c["state_in"] else None
            tail = part["k"] * torch.exp(g * (T - 1 - at))[..., None]
            last = tail.transpose(1, 2) @ part["v"]
            if init is not None:
                last = last + torch.exp(g * T)[..., None] * init
            lasts[n, hs] = last.detach()
            ups, outs = [], []
            for i in range(0, T, max(block, 1)):
                m = min(i + block, T)
                gap = at[i:m, None] - at[None, :m]
                w = torch.where(gap >= 0, torch.exp(g[..., None] * gap.clamp(min=0)), 0.0)
                o = (part["q"][:, i:m] @ part["k"][:, :m].transpose(1, 2) * w) @ part["v"][:, :m]
                if init is not None:
                    o = o + torch.exp(g * (at[i:m] + 1))[..., None] * (part["q"][:, i:m] @ init)
                y[p + i:p + m, hs] = (scale * o.detach()).transpose(0, 1)
                outs.append(scale * o)
                ups.append(s["dy"].reshape(-1, H, c["v_dim"])[p + i:p + m][:, hs].transpose(0, 1).double() if c["train"] else None)
            if not c["train"]:
                continue
            if c["state_out"]:
                outs.append(last)
                ups.append(s["dlast"][n, hs].double())
            leaves = list(part.values()) + ([init] if init is not None else [])
            got = torch.autograd.grad(outs, leaves, ups, allow_unused=True) if outs else [None] * len(leaves)
            for k, d in zip("qkv", got):
                if d is not None and T:
                    grads["d" + k][p:e].index_add_(1, hs // per if k != "v" else hs, d.transpose(0, 1))
            if init is not None and got[3] is not None:
                dinit[n, hs] = got[3]
    out = dict({k: d.view_as(t[k[1:]]) for k, d in grads.items()}, y=y.view_as(t["v"]), last=lasts if c["state_out"] else None)
    return dict(out, dinitial_state=dinit) if c["train"] and c["state_in"] else out


def exact(case, seed):
    c, s = case, prepare(case, seed)
    t = {k: v.detach().double().requires_grad_(c["train"]) for k, v in s["leaves"].items()}
    if c["op"] == "linear":
        return _exact_linear(c, s, t)
    if c["op"] == "linear_step":
        per = c["heads"] // c["kv_heads"]
        q, k = t["q"].repeat_interleave(per, 1), t["k"].repeat_interleave(per, 1)
        state = torch.exp(s["log_decay"].double()).view(1, -1, 1, 1) * t["state"] + torch.einsum("bhk,bhv->bhkv", k, t["v"])
        return dict(y=torch.einsum("bhk,bhkv->bhv", q, state) * c["dim"] ** -0.5, last=state)

    def norm():
        v, last = t["x"], None
        if c["residual"]:
            v = v + t["residual"]
            last = v = v + (v.detach().to(s["leaves"]["residual"].dtype).double() - v.detach())      # rounded; its derivative is one
        g = v.reshape(c["tokens"], c["groups"], -1)
        var, mean = torch.var_mean(g, -1, correction=0, keepdim=True)
        y = ((g - mean) / torch.sqrt(var + 1e-5)).reshape(c["tokens"], -1)
        return y * t.get("weight", 1.0) + t.get("bias", 0.0), last

    def rotary():
        n = c["rotated"] // 2
        pos = s["positions"][None] if c["axes"] == 1 else s["positions"]
        angle = torch.stack([pos[a].double() * s["inv_freq"][f].double() for f, a in enumerate(_axes(c))], -1)
        turn = torch.polar(torch.ones_like(angle), angle)[:, :, None]

        def one(x):
            pairs = x[..., :2 * n].unflatten(-1, (n, 2)) if c["interleaved"] else x[..., :2 * n].unflatten(-1, (2, n)).transpose(-1, -2)
            z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
            z = z if c["interleaved"] else z.transpose(-1, -2)
            return torch.cat([z.flatten(-2), x[..., 2 * n:]], -1)

        return one(t["q"]), one(t["k"]) if "k" in t else None

    with torch.set_grad_enabled(c["train"]):
        y, last = {"norm": norm, "rotary": rotary}[c["op"]]()
    if not c["train"]:
        return dict(y=y, last=last)
    outs, ups = ((y, last), (s["dy"].double(), s["dlast"].double())) if last is not None else ((y,), (s["dy"].double(),))
    grads = torch.autograd.grad(outs, list(t.values()), ups)
    return dict({"d" + n: d for n, d in zip(t, grads)}, y=y.detach(), last=None if last is None else last.detach())


def work(case):
    """Each input read once, each output written once (a backward pass: upstream gradients in, one gradient per input out); the operations of
    the definitions, no recomputation."""
    c = case
    n, e = c["rows"] * c["tokens"], DTYPES[c["dtype"]].itemsize
    twice = 2 if c["train"] else 1
    if c["op"] == "norm":
        W = c["width"]
        stream = DTYPES[c["residual"]].itemsize if c["residual"] else 0
        params = 4 * W * {"": 0, "weight": 1, "both": 2}[c["affine"]]
        return {"bytes": (2 * n * W * (e + stream) + params) * twice, "flops": n * W * (20 if c["train"] else 8)}
    if c["op"] == "rotary":
        heads = c["heads"] + c["kv_heads"]
        return {"bytes": 2 * n * heads * c["dim"] * e * twice + 8 * n * c["axes"] + 2 * c["rotated"], "flops": 3 * n * heads * c["rotated"] * twice}
    K, V, H = c["dim"], c["v_dim"], c["heads"]
    step = c["op"] == "linear_step"
    cu = _bounds(c)
    state = 4 * (c["rows"] if cu is None else len(cu) - 1) * H * K * V
    n = c["rows"] if step else n
    inputs = n * e * (2 * c["kv_heads"] * K + H * V) + state * (step or c["state_in"])
    outputs = n * e * H * V + state * (step or c["state_out"])
    return {"bytes": (inputs + outputs) * twice + 4 * H, "flops": n * H * 5 * K * V * (3 if c["train"] else 1)}
