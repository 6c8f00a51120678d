"""What the decay-attention, gated-norm and beam-search operators are measured on.

``run`` is one pass through an operator: with ``own`` false in its plain form
(elementary torch operations in 32 bits, 64 where 32 lose what matters, rounded
once at the end), with ``own`` true as the calls a user makes of
``cpu_mamba_b200.ops``.

Operators (``case["op"]``):
  attn     decay_attention: S_t = exp(g_t) S_{t-1} + k_t v_t^T,
           o_t = scale S_t^T q_t over whole prompts, dense or packed
  step     decay_attention_step: the same recurrence for one token, in place
  norm     gated_norm: RMSNorm and SiLU gate after a block, scaled residual
           add, RMSNorm before the next block
  beam     beam_select: the best continuations over beams and vocabulary
  reorder  reorder_states: the beams' recurrent states follow their parents
"""
import math

import torch

own = False

_DT = {"bf16": torch.bfloat16, "fp32": torch.float32}
_BYTES = {"bf16": 2, "fp32": 4}


# ------------------------------------------------------------------- cases
def listed():
    return [
        # a short prompt with odd widths (few tokens, an interactive request)
        {"name": "attn fp32 short odd", "op": "attn", "dtype": "fp32", "batch": 2, "length": 37,
         "heads": 6, "key_heads": 3, "dk": 20, "dv": 36, "decay": "token", "packed": False,
         "state": False},
        # the fp32 block's batch (151 sequences of 180 tokens, d_inner 1536 as 24 heads of 64,
        # d_state 24) with one group of keys and queries
        {"name": "attn fp32 151x180", "op": "attn", "dtype": "fp32", "batch": 151, "length": 180,
         "heads": 24, "key_heads": 1, "dk": 24, "dv": 64, "decay": "token", "packed": False,
         "state": False},
        # long-context prefill (8 sequences of 8192 tokens, d_inner 1536), state 128 wide
        {"name": "attn bf16 8x8192", "op": "attn", "dtype": "bf16", "batch": 8, "length": 8192,
         "heads": 24, "key_heads": 1, "dk": 128, "dv": 64, "decay": "token", "packed": False,
         "state": False},
        # a server's packed prefill: a few ragged requests continued from their states, each
        # head with its own keys and a fixed decay
        {"name": "attn bf16 packed 5", "op": "attn", "dtype": "bf16", "batch": 5,
         "length": 32771, "heads": 8, "key_heads": 8, "dk": 128, "dv": 128, "decay": "head",
         "packed": True, "state": True},
        # interactive decode: few sequences
        {"name": "step bf16 3", "op": "step", "dtype": "bf16", "batch": 3, "heads": 24,
         "key_heads": 1, "dk": 128, "dv": 64, "decay": "token"},
        # throughput decode: many sequences, bound by the states
        {"name": "step fp32 512", "op": "step", "dtype": "fp32", "batch": 512, "heads": 24,
         "key_heads": 1, "dk": 128, "dv": 64, "decay": "token"},
        # a decode step's rows (batch 64, d_model 1024) between two blocks
        {"name": "norm fp32 64x1024", "op": "norm", "dtype": "fp32", "residual": "fp32",
         "rows": 64, "width": 1024, "group": 0, "gate": False, "scale": "number", "next": True,
         "before": True},
        # a prompt's rows (8 x 8192 tokens, d_model 768), all parts, fp32 residual stream
        {"name": "norm bf16 65536x768", "op": "norm", "dtype": "bf16", "residual": "fp32",
         "rows": 65536, "width": 768, "group": 0, "gate": True, "scale": "vector", "next": True,
         "before": True},
        # beam search of a few requests
        {"name": "beam fp32 4x4x32000", "op": "beam", "dtype": "fp32", "batch": 4, "beams": 4,
         "vocab": 32000, "num": 4, "finished": True},
        # a full server batch, twice as many continuations as beams, odd vocabulary
        {"name": "beam bf16 64x8x50257", "op": "beam", "dtype": "bf16", "batch": 64, "beams": 8,
         "vocab": 50257, "num": 16, "finished": False},
        # one request's beams through a 24-layer stack's states (d_inner 1536, d_state 16)
        {"name": "reorder 1x4", "op": "reorder", "dtype": "bf16", "batch": 1, "beams": 4,
         "layers": 24, "inner": 1536, "dstate": 16, "kconv": 4},
        # a batch of them
        {"name": "reorder 16x8", "op": "reorder", "dtype": "bf16", "batch": 16, "beams": 8,
         "layers": 24, "inner": 1536, "dstate": 16, "kconv": 4},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["attn", "attn", "attn", "step", "norm", "beam", "reorder"])
    dtype = rng.choice(["bf16", "fp32"])
    if op in ("attn", "step"):
        heads = rng.choice([1, 2, 4, 6, 8, 12, 16, 24])
        key_heads = rng.choice([d for d in range(1, heads + 1) if heads % d == 0])
        dk = rng.choice([rng.randint(1, 128), 8 * rng.randint(1, 16), 64, 128])
        dv = rng.choice([rng.randint(1, 128), 8 * rng.randint(1, 16), 64, 128])
        decay = rng.choice(["token", "head"])
    if op == "attn":
        packed = rng.random() < 0.5
        room = 8 * 8192 * 24 * 128 * 64 // 6           # token-heads x state kept below the listed
        batch = _log(rng, 1, 64)
        most = max(2, min(8192, room // (batch * heads * max(dk, 16) * max(dv, 16))))
        length = _log(rng, 1, most)
        return {"op": "attn", "dtype": dtype, "batch": batch,
                "length": length * batch if packed else length, "heads": heads,
                "key_heads": key_heads, "dk": dk, "dv": dv, "decay": decay, "packed": packed,
                "state": rng.random() < 0.5}
    if op == "step":
        most = max(2, min(1024, 512 * 24 * 128 * 64 // (heads * dk * dv)))
        return {"op": "step", "dtype": dtype, "batch": _log(rng, 1, most), "heads": heads,
                "key_heads": key_heads, "dk": dk, "dv": dv, "decay": decay}
    if op == "norm":
        width = rng.choice([_log(rng, 16, 8192), 64 * rng.randint(1, 64)])
        group = 64 if width % 64 == 0 and rng.random() < 0.4 else 0
        return {"op": "norm", "dtype": dtype, "residual": rng.choice(["", dtype, "fp32"]),
                "rows": _log(rng, 1, max(2, 65536 * 768 // (2 * width))), "width": width,
                "group": group, "gate": rng.random() < 0.6,
                "scale": rng.choice(["number", "vector"]), "next": rng.random() < 0.6,
                "before": rng.random() < 0.5}
    if op == "beam":
        beams = rng.randint(1, 16)
        vocab = _log(rng, 100, 130000)
        batch = _log(rng, 1, max(2, min(128, 64 * 8 * 50257 // (2 * beams * vocab))))
        return {"op": "beam", "dtype": dtype, "batch": batch, "beams": beams, "vocab": vocab,
                "num": rng.choice([beams, 2 * beams]), "finished": rng.random() < 0.5}
    beams = rng.randint(2, 16)
    return {"op": "reorder", "dtype": dtype, "batch": _log(rng, 1, max(2, 96 // beams)),
            "beams": beams, "layers": rng.randint(1, 24), "inner": 8 * rng.randint(8, 192),
            "dstate": rng.choice([8, 16, 24]), "kconv": rng.randint(2, 4)}


# ----------------------------------------------------------------- prepare
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) % (1 << 62))


def _randn(g, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def _decay(g, case, *lead):
    """Log decays: per token -dt A with dt in (0.001, 0.1) and A in (1, 16), the ranges the
    block starts from, or one fixed decay 1 - 2^-(5 + i) per head."""
    H = case["heads"]
    if case["decay"] == "head":
        return torch.log1p(-torch.exp2(-5.0 - 7.0 * torch.arange(H, device="cuda") / H))
    A = 1 + 15 * torch.rand(H, generator=g, device="cuda")
    dt = torch.exp(torch.rand(*lead, H, generator=g, device="cuda") * math.log(100.0)) * 1e-3
    return -dt * A


def _lengths(total, n, seed):
    """n ragged lengths of sum total, the longest several times the shortest."""
    w = [1.0 + ((seed * 7919 + i * 104729) % 997) / 997 * 3 for i in range(n)]
    got = [int(total * x / sum(w)) for x in w]
    got[0] += total - sum(got)
    return got


def prepare(case, seed):
    g = _gen(seed)
    dt = _DT[case["dtype"]]
    op = case["op"]
    if op == "attn":
        B = 1 if case["packed"] else case["batch"]
        T, H, Hk, dk, dv = (case[k] for k in ("length", "heads", "key_heads", "dk", "dv"))
        st = {"case": case, "scale": dk ** -0.5,
              "q": _randn(g, B, T, Hk, dk, dtype=dt), "k": _randn(g, B, T, Hk, dk, dtype=dt),
              "v": _randn(g, B, T, H, dv, dtype=dt), "g": _decay(g, case, B, T),
              "h0": None, "cu": None, "longest": T}
        if case["packed"]:
            lens = _lengths(T, case["batch"], seed)
            st["longest"] = max(lens)
            st["cu"] = torch.tensor([0] + lens).cumsum(0).to(device="cuda", dtype=torch.int32)
        if case["state"]:
            st["h0"] = _randn(g, case["batch"], H, dk, dv, scale=3.0)
        return st
    if op == "step":
        B, H, Hk, dk, dv = (case[k] for k in ("batch", "heads", "key_heads", "dk", "dv"))
        return {"case": case, "scale": dk ** -0.5, "q": _randn(g, B, Hk, dk, dtype=dt),
                "k": _randn(g, B, Hk, dk, dtype=dt), "v": _randn(g, B, H, dv, dtype=dt),
                "g": _decay(g, case, B), "state": _randn(g, B, H, dk, dv, scale=3.0)}
    if op == "norm":
        R, W = case["rows"], case["width"]
        st = {"case": case, "x": _randn(g, R, W, dtype=dt, scale=2.0), "gate": None,
              "weight": (1 + 0.2 * _randn(g, W)).to(dt), "residual": None, "scale": None,
              "next": None}
        if case["gate"]:
            st["gate"] = _randn(g, R, W, dtype=dt, scale=1.5)
        if case["residual"]:
            st["residual"] = _randn(g, R, W, dtype=_DT[case["residual"]], scale=4.0)
            st["scale"] = 0.5 if case["scale"] == "number" else (0.3 * _randn(g, W)).to(dt)
            if case["next"]:
                st["next"] = (1 + 0.2 * _randn(g, W)).to(dt)
        return st
    if op == "beam":
        B, K, V = case["batch"], case["beams"], case["vocab"]
        z = torch.randn(B, K, V, generator=g, device="cuda")
        logits = (z + 0.4 * z * z.abs()).mul_(2.0).to(dt)      # heavier tails than a normal
        scores = -torch.rand(B, K, generator=g, device="cuda").cumsum(1) * 2 - 10
        fin = torch.rand(B, K, generator=g, device="cuda") < 0.2 if case["finished"] else None
        return {"case": case, "logits": logits, "scores": scores, "finished": fin}
    B, K = case["batch"], case["beams"]
    states = []
    for _ in range(case["layers"]):
        states.append(_randn(g, B * K, case["inner"], case["dstate"]))
        states.append(_randn(g, B * K, case["inner"], case["kconv"] - 1, dtype=dt))
    parents = torch.randint(0, K, (B, K), generator=g, device="cuda")
    return {"case": case, "states": states, "parents": parents}


# --------------------------------------------------------------- plain forms
_CHUNK = 64


def _heads(x, H):
    return x.repeat_interleave(H // x.shape[2], dim=2) if x.shape[2] != H else x


def _plain_attn(q, k, v, g, scale, h0):
    """The chunked form on (N, T, heads, width) in 32 bits, log decays in 64."""
    N, T, H, dv = v.shape
    dk = q.shape[-1]
    C = _CHUNK
    nc = -(-T // C)

    def chunks(x):                                             # (N, H, nc, C, ...)
        x = torch.cat([x, x.new_zeros(N, nc * C - T, *x.shape[2:])], 1)
        return x.unflatten(1, (nc, C)).movedim(3, 1)

    qc, kc, vc = chunks(_heads(q.float(), H)), chunks(_heads(k.float(), H)), chunks(v.float())
    G = chunks(g.double()).cumsum(-1)                          # (N, H, nc, C)
    tri = torch.ones(C, C, dtype=torch.bool, device=q.device).tril()
    D = torch.exp((G.unsqueeze(-1) - G.unsqueeze(-2)).masked_fill(~tri, -math.inf)).float()
    o = ((qc @ kc.transpose(-1, -2)) * D) @ vc
    last = G[..., -1:]
    delta = (kc * torch.exp(last - G).float().unsqueeze(-1)).transpose(-1, -2) @ vc
    Sg = torch.cat([torch.zeros_like(last[:, :, :1, 0]), last[..., 0].cumsum(-1)], -1)
    below = torch.ones(nc + 1, nc, dtype=torch.bool, device=q.device).tril(-1)
    W = (Sg.unsqueeze(-1) - Sg[:, :, 1:].unsqueeze(-2)).masked_fill(~below, -math.inf)
    start = (torch.exp(W).float() @ delta.flatten(-2)).unflatten(-1, (dk, dv))
    if h0 is not None:
        start = start + torch.exp(Sg).float()[..., None, None] * h0.unsqueeze(2)
    o = o + torch.exp(G).float().unsqueeze(-1) * (qc @ start[:, :, :-1])
    o = (o * scale).movedim(1, 3).flatten(1, 2)[:, :T]
    return o.to(v.dtype), start[:, :, -1]


def _plain_packed(st):
    q, k, v, g, cu = st["q"][0], st["k"][0], st["v"][0], st["g"], st["cu"].long()
    T, H = v.shape[:2]
    g = g[0] if g.dim() == 3 else g.expand(T, H)
    pos = torch.arange(st["longest"], device=v.device)
    idx = cu[:-1, None] + pos
    live = idx < cu[1:, None]
    idx = idx.clamp(max=T - 1)

    def rows(x):
        return torch.where(live.reshape(*live.shape, *[1] * (x.dim() - 1)), x[idx],
                           x.new_zeros(()))

    o, h = _plain_attn(rows(q), rows(k), rows(v), rows(g), st["scale"], st["h0"])
    tok = torch.arange(T, device=v.device)
    seq = (tok[:, None] >= cu[1:]).sum(1)
    return o[seq, tok - cu[seq]].unsqueeze(0), h


def _plain_step(st):
    H = st["v"].shape[1]
    q, k = (st[n].float().repeat_interleave(H // st[n].shape[1], 1) for n in ("q", "k"))
    v, s = st["v"].float(), st["state"]
    s.mul_(torch.exp(st["g"])[..., None, None]).add_(k.unsqueeze(-1) * v.unsqueeze(-2))
    o = (q.unsqueeze(-1) * s).sum(-2) * st["scale"]
    return o.to(st["v"].dtype), s


def _plain_norm(st):
    c, x = st["case"], st["x"].float()
    gate = None if st["gate"] is None else st["gate"].float()
    if gate is not None:
        gate = gate / (1 + torch.exp(-gate))
    if gate is not None and not c["before"]:
        x = x * gate
    w = c["group"] or c["width"]
    xg = x.unflatten(-1, (-1, w))
    u = (xg * torch.rsqrt(xg.square().mean(-1, keepdim=True) + 1e-5)).flatten(-2)
    u = u * st["weight"].float()
    if gate is not None and c["before"]:
        u = u * gate
    if st["residual"] is None:
        return u.to(st["x"].dtype)
    s = st["scale"].float() if torch.is_tensor(st["scale"]) else st["scale"]
    r = st["residual"].float() + s * u
    if st["next"] is None:
        return r.to(st["residual"].dtype)
    n = r * torch.rsqrt(r.square().mean(-1, keepdim=True) + 1e-5) * st["next"].float()
    return r.to(st["residual"].dtype), n.to(st["x"].dtype)


def _plain_beam(st):
    """Candidates in 64 bits (neighbours in the order lie next to a border); a tie goes to the
    lowest beam, then the lowest token."""
    B, K, V = st["logits"].shape
    n = st["case"]["num"]
    x = st["logits"].double()
    x = x - x.amax(-1, keepdim=True)
    cand = st["scores"].double().unsqueeze(-1) + (x - torch.log(torch.exp(x).sum(-1, keepdim=True)))
    if st["finished"] is not None:
        only = torch.full_like(cand[:1, :1], -math.inf)
        only[..., 0] = 0.0
        cand = torch.where(st["finished"].unsqueeze(-1), st["scores"].double().unsqueeze(-1) + only,
                           cand)
    cand = cand.flatten(1)
    cand = torch.where(cand == cand, cand, cand.new_full((), -math.inf))
    least = cand.topk(n, -1).values[:, -1:]
    at = torch.arange(K * V, device=x.device)
    key = torch.where(cand > least, 2 * K * V - at, torch.where(cand == least, K * V - at, -1))
    pick = key.topk(n, -1).indices.sort(-1).values
    best, order = cand.gather(1, pick).sort(dim=-1, descending=True, stable=True)
    pick = pick.gather(1, order)
    return best.float(), pick // V, pick % V


def _plain_reorder(st):
    B, K = st["parents"].shape
    rows = (torch.arange(B, device="cuda")[:, None] * K + st["parents"]).flatten()
    return [s.copy_(s[rows]) for s in st["states"]]


# --------------------------------------------------------------------- run
def _ops():
    from cpu_mamba_b200 import ops          # only where `own` is true
    return ops


def run(st):
    op = st["case"]["op"]
    if op == "attn":
        if own:
            return _ops().decay_attention(st["q"], st["k"], st["v"], st["g"], scale=st["scale"],
                                          initial_state=st["h0"], cu_seqlens=st["cu"],
                                          return_final_state=True)
        if st["cu"] is not None:
            return _plain_packed(st)
        g = st["g"] if st["g"].dim() == 3 else st["g"].expand(*st["v"].shape[:2], -1)
        return _plain_attn(st["q"], st["k"], st["v"], g, st["scale"], st["h0"])
    if op == "step":
        if own:
            o = _ops().decay_attention_step(st["q"], st["k"], st["v"], st["g"], st["state"],
                                            scale=st["scale"])
            return o, st["state"]
        return _plain_step(st)
    if op == "norm":
        if own:
            return _ops().gated_norm(st["x"], gate=st["gate"], weight=st["weight"],
                                     residual=st["residual"], residual_scale=st["scale"],
                                     next_weight=st["next"], eps=1e-5,
                                     group_size=st["case"]["group"] or None,
                                     norm_before_gate=st["case"]["before"])
        return _plain_norm(st)
    if op == "beam":
        if own:
            return _ops().beam_select(st["logits"], st["scores"], num=st["case"]["num"],
                                      finished=st["finished"], pad_token=0)
        return _plain_beam(st)
    if own:
        _ops().reorder_states(st["states"], st["parents"])
        return st["states"]
    return _plain_reorder(st)


# -------------------------------------------------------------------- work
def work(case):
    op, e = case["op"], _BYTES[case["dtype"]]
    if op == "attn":
        tok = case["length"] * (1 if case["packed"] else case["batch"])
        H, Hk, dk, dv = (case[k] for k in ("heads", "key_heads", "dk", "dv"))
        b = tok * e * (2 * Hk * dk + 2 * H * dv)
        b += 4 * H * (tok if case["decay"] == "token" else 1)
        b += case["batch"] * H * dk * dv * 4 * (2 if case["state"] else 1)
        return {"bytes": b, "flops": 4 * tok * H * dk * dv}
    if op == "step":
        B, H, Hk, dk, dv = (case[k] for k in ("batch", "heads", "key_heads", "dk", "dv"))
        return {"bytes": B * (2 * H * dk * dv * 4 + e * (2 * Hk * dk + 2 * H * dv)) + 4 * H * (
            B if case["decay"] == "token" else 1), "flops": 5 * B * H * dk * dv}
    if op == "norm":
        n, W = case["rows"] * case["width"], case["width"]
        res = _BYTES[case["residual"]] if case["residual"] else 0
        out = 2 * res + (e if case["next"] else 0) if res else e
        return {"bytes": n * (e * (2 if case["gate"] else 1) + out) + 3 * W * e, "flops": 12 * n}
    if op == "beam":
        n = case["batch"] * case["beams"] * case["vocab"]
        return {"bytes": n * e + case["batch"] * (4 * case["beams"] + 20 * case["num"]),
                "flops": 4 * n}
    rows = case["batch"] * case["beams"]
    per = case["layers"] * case["inner"] * (4 * case["dstate"] + e * (case["kconv"] - 1))
    return {"bytes": 2 * rows * per, "flops": 0}


# ------------------------------------------------------------------- exact
def exact(case, seed):
    """The definitions in 64 bits."""
    st = prepare(case, seed)
    op = case["op"]
    if op == "attn":
        return _exact_attn(st)
    if op == "step":
        H = case["heads"]
        rep = H // case["key_heads"]
        head = torch.arange(H, device="cuda") // rep
        q, k, v = st["q"].double()[:, head], st["k"].double()[:, head], st["v"].double()
        s = torch.exp(st["g"].double()).reshape(-1, H, 1, 1) * st["state"].double()
        s = s + torch.einsum("bhi,bhj->bhij", k, v)
        return torch.einsum("bhi,bhij->bhj", q, s) * st["scale"], s
    if op == "norm":
        return _exact_norm(st)
    if op == "beam":
        B, K, V = st["logits"].shape
        lp = torch.log_softmax(st["logits"].double(), -1) + st["scores"].double()[..., None]
        if st["finished"] is not None:
            b, k = st["finished"].nonzero(as_tuple=True)
            lp[b, k] = -math.inf
            lp[b, k, 0] = st["scores"].double()[b, k]
        best, at = lp.reshape(B, K * V).sort(dim=-1, descending=True, stable=True)
        at = at[:, :case["num"]]
        return best[:, :case["num"]], at // V, at % V
    K = case["beams"]
    return [s.double().reshape(-1, K, *s.shape[1:])[
        torch.arange(case["batch"], device="cuda")[:, None], st["parents"]].flatten(0, 1)
        for s in st["states"]]


def _exact_attn(st):
    case, v = st["case"], st["v"].double()
    H, dk, dv = case["heads"], case["dk"], case["dv"]
    B, T = v.shape[:2]
    head = torch.arange(H, device="cuda") // (H // case["key_heads"])
    q, k = st["q"].double(), st["k"].double()
    a = torch.exp(st["g"].double()).expand(B, T, H)
    o = torch.empty_like(v)
    n = case["batch"]
    h = (st["h0"].double() if st["h0"] is not None
         else torch.zeros(n, H, dk, dv, dtype=torch.float64, device="cuda"))
    # token by token, all sequences that still run side by side
    cu = st["cu"].tolist() if st["cu"] is not None else None
    lens = [T] * n if cu is None else [cu[i + 1] - cu[i] for i in range(n)]
    order = sorted(range(n), key=lambda i: -lens[i])
    h = h[order].clone()
    first = torch.tensor([0 if cu is None else cu[i] for i in order], device="cuda")
    row = torch.tensor([i if cu is None else 0 for i in order], device="cuda")
    for t in range(max(lens)):
        m = sum(1 for i in order if lens[i] > t)
        b, at = row[:m], first[:m] + t
        kt, vt = k[b, at][:, head], v[b, at]
        hm = h[:m]
        hm.mul_(a[b, at][..., None, None]).addcmul_(kt[..., None], vt[..., None, :])
        o[b, at] = (q[b, at][:, head].unsqueeze(-2) @ hm).squeeze(-2)
    back = torch.empty(n, dtype=torch.long, device="cuda")
    back[torch.tensor(order, device="cuda")] = torch.arange(n, device="cuda")
    return o * st["scale"], h[back]


def _exact_norm(st):
    c = st["case"]
    x = st["x"].double()
    act = 1.0 if st["gate"] is None else torch.nn.functional.silu(st["gate"].double())
    w = st["weight"].double()

    def rms(t, width):
        t = t.reshape(t.shape[0], -1, width)
        return (t / (t.pow(2).sum(-1, keepdim=True) / width + 1e-5).sqrt()).reshape(t.shape[0], -1)

    width = c["group"] or c["width"]
    u = rms(x, width) * w * act if c["before"] else rms(x * act, width) * w
    if st["residual"] is None:
        return u
    s = st["scale"].double() if torch.is_tensor(st["scale"]) else st["scale"]
    r = st["residual"].double() + u * s
    if st["next"] is None:
        return r
    return r, rms(r, c["width"]) * st["next"].double()
