"""Measured cases of the decoder block's operators: attention, the gated feed-forward half (swiglu) and
the residual norm (add_norm), each in its plain form and through ``kube_gpu_stats_amd.ops.decoder``.

``run`` computes the plain form (elementary torch operations in 32 bits, rounded once at the end) while
``own`` is false, and calls the framework where it is true.  ``exact`` is the definition in 64 bits.
A case named "... train" is a forward and a backward pass together, as a training step runs them.
"""
import math

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}
LARGEST_FLOPS = 12.0 * 8192 * 4096 * 11008  # the largest listed case: swiglu of the benchmark's step
LARGEST_ROWS = 16384 * 8192                 # elements of the largest listed add_norm


def listed():
    return [
        # A prompt's first tokens through a small decoder: one launch, latency is all there is.
        {"name": "attention short", "op": "attention", "train": False, "batch": 1, "seq": 61, "heads": 4,
         "kv_heads": 4, "dim": 64, "type": "bf16", "causal": True, "padded": False},
        # An encoder's pass over a batch: every key for every query, smaller heads.
        {"name": "attention full", "op": "attention", "train": False, "batch": 8, "seq": 1536, "heads": 12,
         "kv_heads": 12, "dim": 64, "type": "fp16", "causal": False, "padded": False},
        # The benchmark's own training step: --train-dim 4096, --train-batch 4, --train-seq 2048.
        {"name": "attention step train", "op": "attention", "train": True, "batch": 4, "seq": 2048, "heads": 32,
         "kv_heads": 32, "dim": 128, "type": "bf16", "causal": True, "padded": False},
        # A padded batch of sequences of every length, shared key heads, an odd width of the batch.
        {"name": "attention padded train", "op": "attention", "train": True, "batch": 6, "seq": 1021, "heads": 20,
         "kv_heads": 4, "dim": 128, "type": "fp16", "causal": True, "padded": True},
        # One long document.
        {"name": "attention long train", "op": "attention", "train": True, "batch": 1, "seq": 16384, "heads": 8,
         "kv_heads": 2, "dim": 128, "type": "bf16", "causal": True, "padded": False},
        # A handful of tokens through the benchmark's feed-forward width: reading the weights is all there is, and
        # what comes back is small beside them.
        {"name": "swiglu few", "op": "swiglu", "train": False, "tokens": 5, "width": 4096, "inner": 11008,
         "type": "bf16"},
        # A forward pass of the step at --train-dim 2048.
        {"name": "swiglu forward", "op": "swiglu", "train": False, "tokens": 2048, "width": 2048, "inner": 5376,
         "type": "bf16"},
        # A training step on sizes that fill no tile.
        {"name": "swiglu ragged train", "op": "swiglu", "train": True, "tokens": 1777, "width": 1000, "inner": 2680,
         "type": "fp16"},
        # The benchmark's own training step.
        {"name": "swiglu step train", "op": "swiglu", "train": True, "tokens": 8192, "width": 4096, "inner": 11008,
         "type": "bf16"},
        # A few rows of an odd width in full precision: latency.
        {"name": "add_norm few train", "op": "add_norm", "train": True, "tokens": 7, "width": 517, "type": "fp32",
         "post": True, "gate": True, "scale": 0.5},
        # The benchmark's own training step.
        {"name": "add_norm step train", "op": "add_norm", "train": True, "tokens": 8192, "width": 4096, "type": "bf16",
         "post": False, "gate": False, "scale": 1.0},
        # A wide model that normalises its branches too and scales them by a learned gate.
        {"name": "add_norm wide train", "op": "add_norm", "train": True, "tokens": 16384, "width": 8192,
         "type": "bf16", "post": True, "gate": True, "scale": 0.7},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["attention", "swiglu", "add_norm"])
    while True:
        if op == "attention":
            kv = _log(rng, 1, 32)
            c = {"op": op, "train": rng.random() < 0.6, "batch": _log(rng, 1, 16), "seq": _log(rng, 1, 16384),
                 "heads": kv * rng.choice([1, 1, 2, 3, 4, 8]), "kv_heads": kv, "dim": rng.choice([64, 128]),
                 "type": rng.choice(["bf16", "fp16"]), "causal": rng.random() < 0.7, "padded": rng.random() < 0.4}
            if (c["heads"] <= 64 and c["batch"] * c["seq"] * c["heads"] <= 1 << 19
                    and c["batch"] * c["heads"] * c["seq"] ** 2 <= 8 * 16384 ** 2):
                return c
        elif op == "swiglu":
            c = {"op": op, "train": rng.random() < 0.6, "tokens": _log(rng, 1, 16384),
                 "width": 8 * _log(rng, 8, 1024), "inner": 8 * _log(rng, 8, 2048), "type": rng.choice(["bf16", "fp16"])}
            if work(c)["flops"] <= LARGEST_FLOPS:
                return c
        else:
            post = rng.random() < 0.5
            c = {"op": op, "train": rng.random() < 0.7, "tokens": _log(rng, 1, 65536), "width": _log(rng, 16, 12288),
                 "type": rng.choice(["bf16", "bf16", "fp16", "fp32"]), "post": post, "gate": rng.random() < 0.5,
                 "scale": rng.choice([1.0, 0.5, 0.7])}
            if c["tokens"] * c["width"] * SIZE[c["type"]] <= LARGEST_ROWS * 2:
                return c


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    t = TYPES[case["type"]]

    def normal(*shape, std=1.0, mean=0.0):
        return (torch.randn(*shape, generator=g, device="cuda") * std + mean).to(t)

    s = {"case": dict(case)}
    if case["op"] == "attention":
        B, S, H, Hk, D = (case[k] for k in ("batch", "seq", "heads", "kv_heads", "dim"))
        # One projection's output holds queries, keys and values side by side: the operands are views of it.
        packed = normal(B, S, H + 2 * Hk, D)
        s["q"], s["k"], s["v"] = packed[:, :, :H], packed[:, :, H:H + Hk], packed[:, :, H + Hk:]
        s["lengths"] = None
        if case["padded"]:
            n = torch.randint(0, S + 1, (B,), generator=g, device="cuda", dtype=torch.int32)
            n[0] = S
            s["lengths"] = n
        if case["train"]:
            s["dout"] = normal(B, S, H, D)
    elif case["op"] == "swiglu":
        T, K, F = case["tokens"], case["width"], case["inner"]
        s["x"] = normal(T, K)
        s["w"] = normal(2 * F, K, std=K ** -0.5)
        if case["train"]:
            s["dout"] = normal(T, F)
    else:
        T, C = case["tokens"], case["width"]
        s["residual"], s["branch"] = normal(T, C), normal(T, C)
        s["weight"] = normal(C, std=0.2, mean=1.0)
        s["post_weight"] = normal(C, std=0.2, mean=1.0) if case["post"] else None
        s["gate"] = normal(C, std=0.3) if case["gate"] else None
        if case["train"]:
            s["dstream"], s["dout"] = normal(T, C), normal(T, C)
    return s


EPS = 1e-5


def run(state):
    case = state["case"]
    return (_own if own else _plain)[case["op"]](state, case)


# ---------------------------------------------------------------- the framework's calls

def _own_attention(s, c):
    from kube_gpu_stats_amd.ops import decoder

    kw = {"causal": c["causal"], "lengths": s["lengths"]}
    if not c["train"]:
        return {"out": decoder.attention(s["q"], s["k"], s["v"], **kw)}
    out, lse = decoder.attention_fwd(s["q"], s["k"], s["v"], **kw)
    dq, dk, dv = decoder.attention_bwd(s["dout"], s["q"], s["k"], s["v"], out, lse, **kw)
    return {"out": out, "dq": dq, "dk": dk, "dv": dv}


def _own_swiglu(s, c):
    from kube_gpu_stats_amd.ops import decoder

    if not c["train"]:
        return {"out": decoder.swiglu(s["x"], s["w"])}
    out, saved = decoder.swiglu_fwd(s["x"], s["w"])
    dx, dw = decoder.swiglu_bwd(s["dout"], s["x"], s["w"], saved)
    return {"out": out, "dx": dx, "dw": dw}


def _own_add_norm(s, c):
    from kube_gpu_stats_amd.ops import decoder

    kw = {"post_weight": s["post_weight"], "gate": s["gate"], "scale": c["scale"], "eps": EPS}
    if not c["train"]:
        stream, out = decoder.add_norm(s["residual"], s["branch"], s["weight"], **kw)
        return {"stream": stream, "out": out}
    stream, out, saved = decoder.add_norm_fwd(s["residual"], s["branch"], s["weight"], **kw)
    grads = decoder.add_norm_bwd(s["dstream"], s["dout"], stream, s["branch"], s["weight"], saved, **kw)
    return {"stream": stream, "out": out, "dresidual": grads[0], "dbranch": grads[1], "dweight": grads[2],
            "dpost_weight": grads[3], "dgate": grads[4]}


# ---------------------------------------------------------------- the plain forms

def _mask(S, causal, lengths, b0, b1, device):
    """[b, 1, S, S] of the (query, key) pairs that count, or None where all do."""
    i = torch.arange(S, device=device)
    m = None
    if causal:
        m = (i[None, :] <= i[:, None])[None, None]
    if lengths is not None:
        live = i[None, :] < lengths[b0:b1, None]
        m2 = (live[:, :, None] & live[:, None, :])[:, None]
        m = m2 if m is None else m & m2
    return m


def _attention_part(q, k, v, do, mask, scale):
    """Softmax attention of [b, h, S, D] in 32 bits; with do, its gradients too."""
    s = torch.matmul(q, k.transpose(-1, -2).contiguous()) * scale
    if mask is not None:
        s.masked_fill_(~mask, float("-inf"))
    top = s.amax(-1, keepdim=True)
    top = torch.where(top == float("-inf"), torch.zeros_like(top), top)
    p = torch.exp_(s.sub_(top))
    total = p.sum(-1, keepdim=True)
    p.div_(torch.where(total == 0, torch.ones_like(total), total))
    o = torch.matmul(p, v)
    if do is None:
        return o, None, None, None
    dv = torch.matmul(p.transpose(-1, -2).contiguous(), do)
    dp = torch.matmul(do, v.transpose(-1, -2).contiguous())
    ds = dp.sub_((do * o).sum(-1, keepdim=True)).mul_(p).mul_(scale)
    del p
    dq = torch.matmul(ds, k)
    dk = torch.matmul(ds.transpose(-1, -2).contiguous(), q)
    return o, dq, dk, dv


def _plain_attention(s, c):
    B, S, H, Hk, D = (c[k] for k in ("batch", "seq", "heads", "kv_heads", "dim"))
    G, t = H // Hk, TYPES[c["type"]]
    rows = {n: s[n].transpose(1, 2).float().contiguous() for n in ("q", "k", "v")}
    rows["do"] = s["dout"].transpose(1, 2).float().contiguous() if c["train"] else None
    if s["lengths"] is not None:  # what lies behind a sequence's end takes no part
        live = (torch.arange(S, device="cuda")[None, :] < s["lengths"][:, None])[:, None, :, None]
        rows = {n: None if r is None else torch.where(live, r, torch.zeros_like(r)) for n, r in rows.items()}
    k, v = (rows[n].repeat_interleave(G, 1) for n in ("k", "v"))
    q, do = rows["q"], rows["do"]
    per = S * S  # scores of one head: as many heads at once as 2^31 scores allow
    if B * H * per <= 1 << 31:
        parts = [(0, B, 0, H)]
    else:
        step = max(1, (1 << 31) // per)
        parts = [(b, b + 1, h, min(H, h + step)) for b in range(B) for h in range(0, H, step)]
    got = [None] * 4
    for b0, b1, h0, h1 in parts:
        cut = lambda x: None if x is None else x[b0:b1, h0:h1]  # noqa: E731
        r = _attention_part(cut(q), cut(k), cut(v), cut(do), _mask(S, c["causal"], s["lengths"], b0, b1, q.device),
                            D ** -0.5)
        if len(parts) == 1:
            got = list(r)
            break
        for n, x in enumerate(r):
            if x is not None:
                if got[n] is None:
                    got[n] = torch.empty(B, H, S, D, device=q.device)
                got[n][b0:b1, h0:h1] = x
    out = {"out": got[0].transpose(1, 2).to(t).contiguous()}
    if c["train"]:
        dk, dv = (x.view(B, Hk, G, S, D).sum(2) for x in (got[2], got[3]))
        out.update({n: x.transpose(1, 2).to(t).contiguous() for n, x in (("dq", got[1]), ("dk", dk), ("dv", dv))})
    return out


def _plain_swiglu(s, c):
    t, F = TYPES[c["type"]], c["inner"]
    x, w = s["x"].float(), s["w"].float()
    gu = torch.matmul(x, w.t().contiguous())
    g, u = gu[:, :F], gu[:, F:]
    sig = 1.0 / (1.0 + torch.exp(-g))
    act = g * sig
    out = {"out": (act * u).to(t)}
    if c["train"]:
        dh = s["dout"].float()
        dgu = torch.cat([dh * u * (sig + act * (1.0 - sig)), dh * act], dim=1)
        out["dx"] = torch.matmul(dgu, w).to(t)
        out["dw"] = torch.matmul(dgu.t().contiguous(), x).to(t)
    return out


def _plain_add_norm(s, c):
    t = TYPES[c["type"]]
    r, b, w = s["residual"].float(), s["branch"].float(), s["weight"].float()
    pw = s["post_weight"].float() if c["post"] else None
    gate = s["gate"].float() if c["gate"] else None
    if pw is not None:
        rp = torch.rsqrt((b * b).mean(-1, keepdim=True) + EPS)
        bh = b * rp
        n = bh * pw
    else:
        n = b
    stream = r + c["scale"] * (n if gate is None else n * gate)
    rs = torch.rsqrt((stream * stream).mean(-1, keepdim=True) + EPS)
    sh = stream * rs
    out = {"stream": stream.to(t), "out": (sh * w).to(t)}
    if not c["train"]:
        return out
    dy = s["dout"].float()
    dyw = dy * w
    ds = s["dstream"].float() + (dyw - sh * (dyw * sh).mean(-1, keepdim=True)) * rs
    dt = ds * c["scale"]
    dn = dt if gate is None else dt * gate
    if pw is not None:
        dnw = dn * pw
        db = (dnw - bh * (dnw * bh).mean(-1, keepdim=True)) * rp
    else:
        db = dn
    out["dresidual"], out["dbranch"] = ds.to(t), db.to(t)
    out["dweight"] = (dy * sh).sum(0).to(t)
    out["dpost_weight"] = (dn * bh).sum(0).to(t) if pw is not None else None
    out["dgate"] = (dt * n).sum(0).to(t) if gate is not None else None
    return out


_own = {"attention": _own_attention, "swiglu": _own_swiglu, "add_norm": _own_add_norm}
_plain = {"attention": _plain_attention, "swiglu": _plain_swiglu, "add_norm": _plain_add_norm}


# ---------------------------------------------------------------- what a pass cannot do without

def work(case):
    z = SIZE[case["type"]]
    if case["op"] == "attention":
        B, S, H, Hk, D = (case[k] for k in ("batch", "seq", "heads", "kv_heads", "dim"))
        # A padded batch's lengths are drawn evenly from 0 to S (the first is S): S/2 and S^2/3 on average.
        tokens = S * (1 + (B - 1) / 2) if case["padded"] else S * B
        pairs = float(S * S) * (1 + (B - 1) / 3) if case["padded"] else float(S * S) * B
        if case["causal"]:
            pairs = (pairs + tokens) / 2
        flops, bytes_ = 4.0 * pairs * H * D, z * D * (tokens * (H + 2 * Hk) + B * S * H)
        if case["train"]:  # five products for two; reads dout as well, writes dq, dk, dv
            flops, bytes_ = 3.5 * flops, bytes_ + z * D * (tokens * H + B * S * (H + 2 * Hk))
        return {"bytes": float(bytes_), "flops": flops}
    if case["op"] == "swiglu":
        T, K, F = case["tokens"], case["width"], case["inner"]
        flops, bytes_ = 4.0 * T * K * F, z * (T * K + 2 * F * K + T * F)
        if case["train"]:
            flops, bytes_ = 3 * flops, bytes_ + z * (T * F + T * K + 2 * F * K)
        return {"bytes": float(bytes_), "flops": flops}
    T, C = case["tokens"], case["width"]
    return {"bytes": float(z * T * C * (8 if case["train"] else 4)), "flops": float(T * C * (30 if case["train"] else 10))}


# ---------------------------------------------------------------- the definitions in 64 bits

def exact(case, seed):
    s, c = prepare(case, seed), case
    return {"attention": _exact_attention, "swiglu": _exact_swiglu, "add_norm": _exact_add_norm}[c["op"]](s, c)


def _exact_attention(s, c):
    """One sequence's one head at a time, on the rows that the sequence has."""
    B, S, H, Hk, D = (c[k] for k in ("batch", "seq", "heads", "kv_heads", "dim"))
    if 4.0 * B * H * S * S * D * (3.5 if c["train"] else 1) > 2e13 or B * H > 1024:
        return None  # the loop below would take too long
    ends = [S] * B if s["lengths"] is None else s["lengths"].tolist()
    zeros = lambda h: torch.zeros(B, S, h, D, dtype=torch.float64, device="cuda")  # noqa: E731
    out, dq, dk, dv = zeros(H), zeros(H), zeros(Hk), zeros(Hk)
    for b, n in enumerate(ends):
        for h in range(H):
            if n == 0:
                continue
            q, k, v = (s[name][b, :n, head].double().contiguous()
                       for name, head in (("q", h), ("k", h // (H // Hk)), ("v", h // (H // Hk))))
            for lo in range(0, n, 4096):  # rows of queries at a time, for the memory of the scores
                hi = min(n, lo + 4096)
                m = hi if c["causal"] else n
                x = torch.mm(q[lo:hi], k[:m].t().contiguous()) / math.sqrt(D)
                if c["causal"]:
                    x = x.masked_fill(torch.ones(hi - lo, m, dtype=torch.bool, device="cuda").triu(lo + 1),
                                      -math.inf)
                p = torch.softmax(x, dim=1)
                o = torch.mm(p, v[:m])
                out[b, lo:hi, h] = o
                if c["train"]:
                    do = s["dout"][b, lo:hi, h].double().contiguous()
                    dv[b, :m, h // (H // Hk)] += torch.mm(p.t().contiguous(), do)
                    dx = p * (torch.mm(do, v[:m].t().contiguous()) - (do * o).sum(1, keepdim=True)) / math.sqrt(D)
                    dq[b, lo:hi, h] = torch.mm(dx, k[:m])
                    dk[b, :m, h // (H // Hk)] += torch.mm(dx.t().contiguous(), q[lo:hi])
    return {"out": out, "dq": dq, "dk": dk, "dv": dv} if c["train"] else {"out": out}


def _exact_swiglu(s, c):
    x, w = s["x"].double(), s["w"].double()
    gate, up = (torch.mm(x, part.t().contiguous()) for part in w.split(c["inner"]))
    out = {"out": gate * torch.sigmoid(gate) * up}
    if c["train"]:
        dh = s["dout"].double()
        slope = torch.sigmoid(gate) * (1 + gate * torch.sigmoid(-gate))
        dgate, dup = dh * up * slope, dh * gate * torch.sigmoid(gate)
        wg, wu = w.split(c["inner"])
        out["dx"] = torch.mm(dgate, wg) + torch.mm(dup, wu)
        out["dw"] = torch.cat([torch.mm(dgate.t().contiguous(), x), torch.mm(dup.t().contiguous(), x)])
    return out


def _exact_add_norm(s, c):
    r, b, w = s["residual"].double(), s["branch"].double(), s["weight"].double()
    C = c["width"]
    ones = torch.ones(C, dtype=torch.float64, device="cuda")
    pw = s["post_weight"].double() if c["post"] else ones
    gate = s["gate"].double() if c["gate"] else ones
    inv_b = ((b.square().sum(1, keepdim=True) / C + EPS) ** -0.5) if c["post"] else 1.0
    stream = r + c["scale"] * gate * pw * b * inv_b
    inv_s = (stream.square().sum(1, keepdim=True) / C + EPS) ** -0.5
    out = {"stream": stream, "out": w * stream * inv_s}
    if not c["train"]:
        return out
    dy = s["dout"].double()
    # d/ds of s_i inv(s): inv (delta_ij - s_i s_j inv^2 / C)
    a = w * dy
    ds = s["dstream"].double() + inv_s * a - stream * inv_s ** 3 * (a * stream).sum(1, keepdim=True) / C
    a = c["scale"] * gate * pw * ds
    if c["post"]:
        db = inv_b * a - b * inv_b ** 3 * (a * b).sum(1, keepdim=True) / C
    else:
        db = a
    out["dresidual"], out["dbranch"] = ds, db
    out["dweight"] = (dy * stream * inv_s).sum(0)
    out["dpost_weight"] = (c["scale"] * gate * ds * b * inv_b).sum(0) if c["post"] else None
    out["dgate"] = (c["scale"] * ds * pw * b * inv_b).sum(0) if c["gate"] else None
    return out
