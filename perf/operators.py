"""The operators of an INT8 expert layer with grouped routing, as cases to measure.

Four operators:

* ``route``: expert selection from router logits. Scores are sigmoid or
  softmax, a per-expert balance bias is added for the selection only, experts
  come in groups of which the best few are kept, and the weights of the K
  selected experts are renormalised and scaled.
* ``norm``: root-mean-square norm with the residual's addition before it and
  an e4m3 copy of its output (one scale per token and 128 columns) after it.
* ``gate_up`` / ``down``: the two grouped products of an expert layer with
  int8 weights (one scale per expert and output channel) and int8 activations
  (one scale per token), from and to bf16 rows.
* ``norm_linear``: the norm with an int8 output (one scale per token) and the
  dense int8 product that reads it.

``run`` computes them in plain torch, or, with ``own`` set, through the
package's entry points.
"""

import torch

own = False

EPS = 1e-6
E4M3_MAX = 448.0


# --------------------------------------------------------------------------- cases
def listed():
    return [
        # one sequence decoding: a single token's selection, all latency
        {"name": "route_t1", "op": "route", "T": 1, "E": 256, "K": 8, "groups": 8, "keep": 4, "top": 2,
         "scoring": "sigmoid", "bias": True, "dtype": "float32", "masked": 0, "scale": 2.5, "norm": True},
        # a long prefill batch with the balance bias
        {"name": "route_prefill", "op": "route", "T": 16384, "E": 256, "K": 8, "groups": 8, "keep": 4, "top": 2,
         "scoring": "sigmoid", "bias": True, "dtype": "float32", "masked": 0, "scale": 2.5, "norm": True},
        # softmax scores, best expert of a group, groups of 20, some experts switched off, bf16 logits
        {"name": "route_softmax_odd", "op": "route", "T": 4001, "E": 160, "K": 6, "groups": 8, "keep": 3, "top": 1,
         "scoring": "softmax", "bias": False, "dtype": "bfloat16", "masked": 9, "scale": 16.0, "norm": False},
        # one sequence decoding, hidden size of qwen3-30b-a3b
        {"name": "norm_t1", "op": "norm", "T": 1, "H": 2048, "pad": 0},
        # the longest prefill batch at the hidden size of qwen3-235b-a22b
        {"name": "norm_prefill", "op": "norm", "T": 16384, "H": 4096, "pad": 0},
        # 64 sequences decoding on the qwen3-30b-a3b layer: every expert's weights for a few rows each
        {"name": "gate_up_t64", "op": "gate_up", "T": 64, "E": 128, "K": 8, "H": 2048, "I": 768, "skew": 0.0,
         "clamp": False},
        # the same layer's longest prefill batch
        {"name": "gate_up_t4096", "op": "gate_up", "T": 4096, "E": 128, "K": 8, "H": 2048, "I": 768, "skew": 0.0,
         "clamp": False},
        # clamped SwiGLU with biases at gpt-oss-20b's sizes (no multiple of the tile sizes), a decode batch
        {"name": "gate_up_bias_t16", "op": "gate_up", "T": 16, "E": 32, "K": 4, "H": 2880, "I": 2880, "skew": 0.0,
         "clamp": True},
        # one token through the down projection of qwen3-30b-a3b
        {"name": "down_t1", "op": "down", "T": 1, "E": 128, "K": 8, "H": 2048, "I": 768, "skew": 0.0},
        # an odd batch with a skewed load: some experts empty, some with many rows
        {"name": "down_skewed", "op": "down", "T": 1000, "E": 128, "K": 8, "H": 4096, "I": 1536, "skew": 1.0},
        # one decoding batch through a normed dense projection
        {"name": "norm_linear_t32", "op": "norm_linear", "T": 32, "H": 2048, "N": 4096, "pad": 0},
        # a prefill batch of odd length through the same kind of projection, compute-bound
        {"name": "norm_linear_t8191", "op": "norm_linear", "T": 8191, "H": 4096, "N": 4096, "pad": 64},
    ]


def _log(rng, lo, hi):
    """An integer between lo and hi, even over its logarithm."""
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(["route", "norm", "gate_up", "down", "norm_linear"])
    if op == "route":
        groups = rng.choice([1, 1, 2, 4, 5, 8, 16])
        size = rng.randint(4, max(4, min(64, 256 // groups)))
        keep = rng.randint(max(1, groups // 2), groups)
        E = groups * size
        return {"op": op, "T": _log(rng, 1, 16384), "E": E, "K": rng.randint(1, min(16, keep * size)),
                "groups": groups, "keep": keep, "top": rng.choice([1, 2]),
                "scoring": rng.choice(["sigmoid", "softmax"]), "bias": rng.random() < 0.6,
                "dtype": rng.choice(["float32", "bfloat16"]), "masked": rng.choice([0, 0, E // 8]),
                "scale": rng.choice([1.0, 2.5]), "norm": rng.random() < 0.7}
    if op == "norm":
        H = 8 * _log(rng, 16, 1024)
        return {"op": op, "T": _log(rng, 1, min(16384, 16384 * 4096 // H)), "H": H,
                "pad": rng.choice([0, 0, 8, 64])}
    if op == "norm_linear":
        H, N = 8 * _log(rng, 16, 512), 8 * _log(rng, 16, 512)
        return {"op": op, "T": _log(rng, 1, 8191), "H": H, "N": N, "pad": rng.choice([0, 0, 8, 64])}
    E = rng.choice([8, 32, 64, 128])
    H, I = 8 * _log(rng, 16, 256), 8 * _log(rng, 8, 96)
    c = {"op": op, "T": _log(rng, 1, 4000), "E": E, "K": rng.randint(1, 8), "H": H, "I": I,
         "skew": rng.choice([0.0, 0.0, 1.0])}
    if op == "gate_up":
        c["clamp"] = rng.random() < 0.3
    return c


def work(case):
    op, T = case["op"], case["T"]
    if op == "route":
        E, K = case["E"], case["K"]
        item = 4 if case["dtype"] == "float32" else 2
        return {"bytes": T * E * item + (4 * E if case["bias"] else 0) + T * K * (8 + 4) + 4 * E,
                "flops": T * E * 4}
    if op == "norm":
        H = case["H"]
        groups = -(-H // 128)
        return {"bytes": T * H * (2 + 2 + 2 + 2 + 1) + 4 * T * groups + 2 * H, "flops": 8 * T * H}
    if op == "norm_linear":
        H, N = case["H"], case["N"]
        return {"bytes": T * H * (2 + 2 + 2) + 2 * H + N * H + 4 * N + 2 * T * N, "flops": 2 * T * H * N}
    E, K, H, I = case["E"], case["K"], case["H"], case["I"]
    rows, used = T * K, E * (1.0 - (1.0 - K / E) ** T)   # experts that a uniform routing reaches
    if op == "gate_up":
        return {"bytes": 2 * T * H + used * (2 * I * H + 8 * I + (4 * I if case["clamp"] else 0)) + 2 * rows * I
                + 4 * rows, "flops": 2 * rows * H * 2 * I}
    return {"bytes": 2 * rows * I + used * (I * H + 4 * H) + 2 * rows * H + 8 * rows, "flops": 2 * rows * H * I}


# --------------------------------------------------------------------------- inputs
def _rows(g, T, H, pad, scale=1.0):
    """bf16 rows [T, H] with a row stride of H + pad."""
    return (torch.randn(T, H + pad, device="cuda", generator=g) * scale).to(torch.bfloat16)[:, :H]


def _int8_weight(g, *shape):
    """int8 weights as rounding a normal weight to its channel's amax gives them, and the channels' scales."""
    q = (torch.randn(*shape, device="cuda", generator=g) * 36).round_().clamp_(-127, 127).to(torch.int8)
    s = (0.5 + torch.rand(*shape[:-1], device="cuda", generator=g)) * (0.02 / 36)
    return q, s


def prepare(case, seed):
    op, T = case["op"], case["T"]
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    st = {"case": case}
    if op == "route":
        E = case["E"]
        logits = torch.randn(T, E, device="cuda", generator=g) * 1.5
        if case["masked"]:   # experts that are switched off, with -inf or with the type's lowest value
            off = torch.randperm(E, device="cuda", generator=g)[:case["masked"]]
            logits[:, off[0::2]] = float("-inf")
            logits[:, off[1::2]] = torch.finfo(getattr(torch, case["dtype"])).min
        st["logits"] = logits.to(getattr(torch, case["dtype"]))
        st["bias"] = torch.randn(E, device="cuda", generator=g) * 0.05 if case["bias"] else None
        return st
    if op in ("norm", "norm_linear"):
        H = case["H"]
        st["x"] = _rows(g, T, H, case["pad"])
        st["residual"] = _rows(g, T, H, case["pad"], 4.0)
        st["residual"][:, :: max(1, H // 5)] *= 30   # the few channels of a residual stream that grow large
        st["weight"] = (1 + 0.1 * torch.randn(H, device="cuda", generator=g)).to(torch.bfloat16)
        if op == "norm_linear":
            st["w"], st["ws"] = _int8_weight(g, case["N"], H)
            if own:
                from moe_serving_profile_b200 import layout
                st["packed"] = layout.int8_linear(st["w"], st["ws"])
        return st
    E, K, H, I = case["E"], case["K"], case["H"], case["I"]
    load = -case["skew"] * torch.log(torch.arange(1, E + 1, device="cuda", dtype=torch.float32))
    score = load - torch.log(-torch.log(torch.rand(T, E, device="cuda", generator=g).clamp_(1e-9, 1 - 1e-7)))
    idx = torch.topk(score, K, dim=1).indices
    slot, tok = torch.arange(K, device="cuda"), torch.arange(T, device="cuda")
    src = torch.argsort(((idx * K + slot) * T + tok[:, None]).reshape(-1))   # expert, then slot, then token
    expert = idx.reshape(-1)[src]
    counts = torch.bincount(expert, minlength=E)
    offsets = torch.cat([counts.new_zeros(1), counts.cumsum(0)])
    inverse = torch.empty_like(src)
    inverse[src] = torch.arange(T * K, device="cuda")
    w1, s1 = _int8_weight(g, E, 2, I, H)
    w2, s2 = _int8_weight(g, E, H, I)
    st.update(counts=counts.int(), offsets=offsets.int(), perm_src=src.int(), inverse=inverse.int(),
              expert=expert, place=torch.arange(T * K, device="cuda") - offsets[expert],
              most=int(counts.max()), w1=w1, s1=s1, w2=w2, s2=s2, b1=None)
    if case.get("clamp"):
        st["b1"] = (torch.randn(E, 2, I, device="cuda", generator=g) * 0.01).to(torch.bfloat16)
    if op == "gate_up":
        st["hidden"] = _rows(g, T, H, 0)
    else:
        st["act"] = (torch.randn(T * K, I, device="cuda", generator=g).square_()
                     * torch.randn(T * K, I, device="cuda", generator=g)).to(torch.bfloat16)
        st["weights"] = torch.softmax(torch.randn(T, K, device="cuda", generator=g), dim=1)
    if own:
        from moe_serving_profile_b200 import _lib, layout
        more = {}
        if case.get("clamp"):
            more = dict(gate_bias=st["b1"][:, 0], up_bias=st["b1"][:, 1],
                        gated_epilogue=_lib.EPI_CLAMP_SWIGLU_F32)
        st["packed"] = layout.int8_experts(w1[:, 0], s1[:, 0], w1[:, 1], s1[:, 1], w2, s2, **more)
    return st


# --------------------------------------------------------------------------- plain forms
def _quant_rows(x):
    """int8 rows (as fp32 whole numbers) and their scales: amax / 127, or 1 for a row of zeros."""
    amax = x.abs().amax(dim=1, keepdim=True)
    s = torch.where(amax > 0, amax / 127.0, torch.ones_like(amax))
    return torch.round(x / s), s


def _route_plain(st):
    c = st["case"]
    T, E, K, G = c["T"], c["E"], c["K"], c["groups"]
    x = st["logits"].double()   # 64 bits: experts whose keys are close are told apart
    if c["scoring"] == "sigmoid":
        score = 1.0 / (1.0 + torch.exp(-x))
    else:
        ex = torch.exp(x - x.amax(dim=1, keepdim=True))
        score = ex / ex.sum(dim=1, keepdim=True)
    key = score if st["bias"] is None else score + st["bias"].double()
    if c["keep"] < G:
        best = torch.topk(key.view(T, G, E // G), min(c["top"], E // G), dim=2).values.sum(dim=2)
        kept = torch.sort(best, dim=1, descending=True, stable=True).indices[:, :c["keep"]]
        mask = torch.zeros(T, G, dtype=torch.bool, device=x.device).scatter_(1, kept, True)
        key = key.view(T, G, E // G).masked_fill(~mask[:, :, None], float("-inf")).view(T, E)
    idx = torch.sort(key, dim=1, descending=True, stable=True).indices[:, :K]
    w = torch.gather(score, 1, idx)
    if c["norm"]:
        w = w / (w.sum(dim=1, keepdim=True) + 1e-20)
    counts = torch.zeros(E, dtype=torch.int32, device=x.device)
    counts.scatter_add_(0, idx.reshape(-1), torch.ones(T * K, dtype=torch.int32, device=x.device))
    return idx, (w * c["scale"]).float(), counts


def _norm_plain(st):
    """(new residual, fp32 normed rows)."""
    h = (st["x"].float() + st["residual"].float()).to(torch.bfloat16)
    f = h.float()
    return h, f * torch.rsqrt(f.square().mean(dim=1, keepdim=True) + EPS) * st["weight"].float()


def _grouped(st, rows, w):
    """rows [R, k] (expert-major) times each row's expert's w [E, n, k], in fp32."""
    E, n, k = w.shape
    buf = rows.new_zeros(E, st["most"], k)
    buf[st["expert"], st["place"]] = rows
    return torch.bmm(buf, w.float().transpose(1, 2))[st["expert"], st["place"]]


def _plain(st):
    c = st["case"]
    op = c["op"]
    if op == "route":
        return _route_plain(st)
    if op == "norm":
        h, y = _norm_plain(st)
        T, H = y.shape
        groups = -(-H // 128)
        p = torch.nn.functional.pad(y, (0, groups * 128 - H)).view(T, groups, 128)
        amax = p.abs().amax(dim=2, keepdim=True)
        s = torch.where(amax > 0, amax / E4M3_MAX, torch.ones_like(amax))
        q = (p / s).clamp(-E4M3_MAX, E4M3_MAX).view(T, groups * 128)[:, :H].to(torch.float8_e4m3fn)
        return h, y.to(torch.bfloat16), q, s.squeeze(2)
    if op == "norm_linear":
        h, y = _norm_plain(st)
        q, s = _quant_rows(y)
        return h, (q @ st["w"].float().t() * s * st["ws"]).to(torch.bfloat16)
    E, K, H, I = c["E"], c["K"], c["H"], c["I"]
    if op == "gate_up":
        q, s = _quant_rows(st["hidden"].float())
        tok = st["perm_src"].long() // K
        d = _grouped(st, q[tok], st["w1"].view(E, 2 * I, H)).view(-1, 2, I) * s[tok, :, None] * st["s1"][st["expert"]]
        if not c["clamp"]:
            g, u = d[:, 0], d[:, 1]
            return (g / (1.0 + torch.exp(-g)) * u).to(torch.bfloat16)
        d = d + st["b1"].float()[st["expert"]]
        g, u = d[:, 0].clamp(max=7.0), d[:, 1].clamp(-7.0, 7.0)
        return (g / (1.0 + torch.exp(-1.702 * g)) * (u + 1.0)).to(torch.bfloat16)
    q, s = _quant_rows(st["act"].float())
    d = _grouped(st, q, st["w2"]) * s * st["s2"][st["expert"]]
    return (d * st["weights"].reshape(-1)[st["perm_src"].long()][:, None]).to(torch.bfloat16)


# --------------------------------------------------------------------------- the package's operators
def _own(st):
    from moe_serving_profile_b200 import experts, ops
    c = st["case"]
    op = c["op"]
    if op == "route":
        r = ops.route_grouped(st["logits"], st["bias"], c["K"], n_group=c["groups"], topk_group=c["keep"],
                              group_top=c["top"], scoring=c["scoring"], normalize=c["norm"], scale=c["scale"])
        return r.indices, r.scores, r.counts
    if op == "norm":
        n = ops.add_rmsnorm(st["x"], st["weight"], EPS, residual=st["residual"], quant="fp8", k_pad=_pad16(c["H"]))
        return n.residual, n.out, n.rows.q[:, :c["H"]], n.rows.scale
    if op == "norm_linear":
        n = ops.add_rmsnorm(st["x"], st["weight"], EPS, residual=st["residual"], quant="int8", normed=False)
        return n.residual, experts.int8_linear(st["packed"], n.rows)
    perm = ops.Permutation(st["counts"], st["offsets"], st["perm_src"], st["inverse"])
    if op == "gate_up":
        act = experts.int8_gate_up(st["packed"], st["hidden"], perm, K=c["K"], num_experts=c["E"], expert_begin=0)
        return act[:, :c["I"]]
    return experts.int8_down(st["packed"], st["act"], perm, st["weights"], K=c["K"], num_experts=c["E"],
                             expert_begin=0)


def _pad16(n):
    return -(-n // 16) * 16


def run(state):
    return _own(state) if own else _plain(state)


# --------------------------------------------------------------------------- definitions in 64 bits
def _q64(x):
    """int8 rows and scales of float64 rows; the scale is held in 32 bits."""
    s = (x.abs().amax(dim=1) / 127.0).float().double()
    s = torch.where(s > 0, s, torch.ones_like(s))
    return torch.round(x / s[:, None]), s


def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    if op == "route":
        x, T, E, K = st["logits"].double(), case["T"], case["E"], case["K"]
        if case["scoring"] == "sigmoid":
            score = torch.sigmoid(x)
        else:
            score = torch.softmax(x, dim=1)
        key = score.clone()
        if st["bias"] is not None:
            key += st["bias"].double()
        size = E // case["groups"]
        if case["keep"] < case["groups"]:
            parts = key.reshape(T, -1, size).sort(dim=2, descending=True).values[:, :, :case["top"]].sum(dim=2)
            order = torch.argsort(-parts, dim=1, stable=True)
            rank = torch.argsort(order, dim=1)
            gone = (rank >= case["keep"]).repeat_interleave(size, dim=1)
            key[gone] = float("-inf")
        idx = torch.argsort(-key, dim=1, stable=True)[:, :K]
        w = score.gather(1, idx)
        if case["norm"]:
            w = w / (w.sum(dim=1, keepdim=True) + 1e-20)
        return None, w * case["scale"], None
    if op in ("norm", "norm_linear"):
        total = st["x"].double() + st["residual"].double()
        h = total.to(torch.bfloat16).double()   # the stored residual is what the norm reads
        y = h / torch.sqrt((h * h).mean(dim=1, keepdim=True) + EPS) * st["weight"].double()
        if op == "norm_linear":
            q, s = _q64(y)
            return total, (q @ st["w"].double().t()) * s[:, None] * st["ws"].double()
        H = case["H"]
        q, scales = torch.empty_like(y), []
        for a in range(0, H, 128):
            part = y[:, a:a + 128]
            s = part.abs().amax(dim=1) / E4M3_MAX
            s = torch.where(s > 0, s, torch.ones_like(s))
            scales.append(s)
            v = part / s[:, None]
            # e4m3: 3 bits after the leading one, the smallest exponent -6, ties to even
            step = torch.exp2(torch.floor(torch.log2(v.abs().clamp_min(2.0 ** -6))) - 3)
            q[:, a:a + 128] = (torch.round(v / step) * step).clamp(-E4M3_MAX, E4M3_MAX)
        return total, y, q, torch.stack(scales, dim=1)
    E, K = case["E"], case["K"]
    rows = st["hidden"].double() if op == "gate_up" else st["act"].double()
    q, s = _q64(rows)
    if op == "gate_up":
        tok = st["perm_src"].long() // K
        q, s = q[tok], s[tok]
    w = st["w1"].view(E, -1, case["H"]) if op == "gate_up" else st["w2"]
    sc = st["s1"].view(E, -1) if op == "gate_up" else st["s2"]
    out = torch.empty(q.shape[0], w.shape[1], dtype=torch.float64, device="cuda")
    at = st["offsets"].tolist()
    for e in range(E):
        if at[e + 1] > at[e]:
            out[at[e]:at[e + 1]] = q[at[e]:at[e + 1]] @ w[e].double().t() * sc[e].double()
    out *= s[:, None]
    if op == "down":
        return out * st["weights"].double().reshape(-1)[st["perm_src"].long()][:, None]
    g, u = out[:, :case["I"]], out[:, case["I"]:]
    if not case["clamp"]:
        return g * torch.sigmoid(g) * u
    b = st["b1"].double()[st["expert"]]
    g, u = torch.clamp(g + b[:, 0], max=7.0), torch.clamp(u + b[:, 1], -7.0, 7.0)
    return g * torch.sigmoid(1.702 * g) * (u + 1)
