"""The decoder block's operators (ops/decoder.py) against their definitions in 64 bits, and their refusals.

Tolerances are bounds per element, worked out from what the kernels round: with u half a
step of the tensors' type, every rounded operand of a sum adds u times that term's
magnitude, every 32-bit sum of n terms at most n 2^-24 times the sum of magnitudes, the
rounded result u times itself.  The bounds are computed in 64 bits beside the reference.
"""
import gc
import math

import pytest
import torch

from kube_gpu_stats_amd.ops import decoder

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
E32 = 2.0 ** -24


def half_step(t):
    return torch.finfo(t).eps / 2


def close(got, want, tol, what):
    """|got - want| <= tol everywhere (and got finite)."""
    got = got.double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert torch.isfinite(got).all(), what
    over = ((got - want).abs() - tol).max().item() if got.numel() else 0.0
    assert over <= 0, (what, over, (got - want).abs().max().item(), tol.max().item())


def mm(a, b):
    return torch.matmul(a.contiguous(), b.contiguous())


# --------------------------------------------------------------------- attention's oracle

def attention_oracle(q, k, v, do, causal, scale, ends):
    """Outputs, gradients and their tolerances, in 64 bits, a sequence at a time."""
    B, S, H, D = q.shape
    Hk, t, u = k.shape[2], q.dtype, half_step(q.dtype)
    z = lambda n: torch.zeros(B, S, n, D, dtype=torch.float64, device=q.device)  # noqa: E731
    r = {"out": z(H), "dq": z(H), "dk": z(Hk), "dv": z(Hk)}
    tol = {n: torch.zeros_like(x) for n, x in r.items()}
    lse = torch.full((B, H, S), -math.inf, dtype=torch.float64, device=q.device)
    for b, n in enumerate(ends):
        if n == 0:
            continue
        for h in range(H):
            g = h // (H // Hk)
            Q, K, V, G = (x[b, :n, i].double().contiguous() for x, i in ((q, h), (k, g), (v, g), (do, h)))
            s = mm(Q, K.t()) * scale
            if causal:
                s = s.masked_fill(torch.ones(n, n, dtype=torch.bool, device=q.device).triu(1), -math.inf)
            lse[b, h, :n] = torch.logsumexp(s, 1) / math.log(2)
            p = torch.softmax(s, 1)
            o = mm(p, V)
            dp = mm(G, V.t())
            ds = p * (dp - (G * o).sum(1, keepdim=True))
            r["out"][b, :n, h] = o
            r["dq"][b, :n, h] = scale * mm(ds, K)
            r["dk"][b, :n, g] += scale * mm(ds.t(), Q)
            r["dv"][b, :n, g] += mm(p.t(), G)
            # relative error of a probability: its score (D products and the sum), the power, the sum of the row
            size = mm(Q.abs(), K.abs().t()).max() * scale
            e = 2 * (E32 * (D + 8) * size + E32 * (n + 16))
            tiny = 2.0 ** -25 * n if t == F16 else 0.0  # fp16 probabilities below its normal range
            # A probability below 2^-126 leaves the range of 32 bits and becomes 0: of a sum over at most n of
            # them, each times a factor f, 2^-126 n max f is lost; and a result below 2^-126 is lost itself.
            # (Here scores lie hundreds apart: the 64-bit reference holds values like 1e-93.)
            gone = 2.0 ** -126 * (1 + n * (H // Hk))
            top_dp = (mm(G.abs(), V.abs().t()).max() + (G * o).abs().sum(1).max()) * scale
            av = mm(p, V.abs())
            t_o = u * o.abs() + (u * (1 + u) + e + E32 * n) * av + tiny * V.abs().max() + gone * (1 + V.abs().max())
            tol["out"][b, :n, h] = t_o
            ag = mm(p.t(), G.abs())
            tol["dv"][b, :n, g] += (u * (1 + u) + e + E32 * n * (H // Hk)) * ag + tiny * G.abs().max() + gone * (1 + G.abs().max())
            # ds: p's error, the products dp, delta (from the rounded output); then rounded itself
            adp = mm(G.abs(), V.abs().t())
            # delta comes from out and its low bits: out's error without its rounding, and 2^-9 of that
            t_low = t_o - u * o.abs() * (1 - 2.0 ** -8)
            e_ds = ds.abs() * (u + e) + p * (E32 * 2 * D * adp + (G.abs() * t_low).sum(1, keepdim=True)
                                             + E32 * 2 * D * (G * o).abs().sum(1, keepdim=True))
            e_ds = e_ds * (1 + u) + (2.0 ** -25 if t == F16 else 0.0)
            tol["dq"][b, :n, h] = scale * (mm(e_ds, K.abs()) + E32 * n * mm(ds.abs(), K.abs()))
            tol["dq"][b, :n, h] += gone * (1 + top_dp * K.abs().max())
            tol["dk"][b, :n, g] += scale * (mm(e_ds.t(), Q.abs()) + E32 * n * (H // Hk) * mm(ds.t().abs(), Q.abs()))
            tol["dk"][b, :n, g] += gone * (1 + top_dp * Q.abs().max())
    for n in ("dq", "dk", "dv"):
        tol[n] += u * r[n].abs()
    if t == F16:  # results below the normal range
        for n in tol:
            tol[n] += 2.0 ** -25
    return r, tol, lse


def attention_inputs(B, S, H, Hk, D, t, dev, seed=0, std=1.0):
    g = torch.Generator(device=dev).manual_seed(seed)
    mk = lambda n, s=1.0: (torch.randn(B, S, n, D, generator=g, device=dev) * s).to(t)  # noqa: E731
    return mk(H, std), mk(Hk), mk(Hk), mk(H)


def attention_check(q, k, v, do, causal, lengths=None, scale=None):
    B, S, H, D = q.shape
    ends = [S] * B if lengths is None else [min(max(n, 0), S) for n in lengths]
    dl = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device=q.device)
    kw = {"causal": causal, "scale": scale, "lengths": dl}
    out, saved = decoder.attention_fwd(q, k, v, **kw)
    dq, dk, dv = decoder.attention_bwd(do, q, k, v, out, saved, **kw)
    lse = saved[0]
    ref, tol, ref_lse = attention_oracle(q, k, v, do, causal, D ** -0.5 if scale is None else scale, ends)
    for n, x in (("out", out), ("dq", dq), ("dk", dk), ("dv", dv)):
        close(x, ref[n], tol[n], n)
    for b, n in enumerate(ends):  # behind the end: exactly zero
        for x in (out, dq, dk, dv):
            assert (x[b, n:] == 0).all()
        assert (lse[b, :, n:] == -math.inf).all()
        if n:
            assert (lse[b, :, :n].double() - ref_lse[b, :, :n]).abs().max() < 1e-3
    assert torch.equal(decoder.attention(q, k, v, **kw), out)
    return out, saved, dq, dk, dv


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "GPU tests need a GPU"
    yield torch.device("cuda", 0)
    gc.collect()
    torch.cuda.empty_cache()  # other modules measure the GPU's memory


gpu = pytest.mark.gpu


@gpu
@pytest.mark.parametrize("t", [BF16, F16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("B,S,H,Hk", [(1, 1, 1, 1), (2, 2, 3, 3), (1, 31, 2, 1), (2, 64, 2, 2), (1, 65, 3, 1),
                                      (1, 127, 2, 2), (2, 128, 1, 1), (1, 129, 4, 2), (3, 200, 2, 2), (1, 513, 5, 1)])
def test_attention_sizes(dev, B, S, H, Hk, D, causal, t):
    attention_check(*attention_inputs(B, S, H, Hk, D, t, dev, seed=S), causal)


@gpu
@pytest.mark.parametrize("D,t", [(64, F16), (128, BF16)])
@pytest.mark.parametrize("causal", [True, False])
def test_attention_split_walk(dev, D, t, causal):
    """One key head and long rows: dk and dv are summed in parts and joined."""
    assert decoder._dkv_splits(1, 1100, 8, 1, causal) > 8
    assert decoder._dkv_splits(2, 700, 3, 1, causal) > 1
    attention_check(*attention_inputs(1, 1100, 8, 1, D, t, dev, seed=5), causal)
    attention_check(*attention_inputs(2, 700, 3, 1, D, t, dev, seed=6), causal, lengths=[33, 699])


@gpu
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("t", [BF16, F16])
def test_attention_padded(dev, causal, t):
    """Lengths of zero, one, all, out of range; what lies behind them is NaN and infinite."""
    lengths = [0, 1, 63, 64, 65, 150, 129, 1000, -3]
    for D in (64, 128):
        q, k, v, do = attention_inputs(len(lengths), 150, 4, 2, D, t, dev, seed=11)
        out, saved, *grads = attention_check(q, k, v, do, causal, lengths)
        clean = out, *saved, *grads
        for b, n in enumerate(lengths):
            n = min(max(n, 0), 150)
            for i, x in enumerate((q, k, v, do)):
                x[b, n:] = math.nan if (b + i) % 2 else math.inf
        dl = torch.tensor(lengths, dtype=torch.int32, device=dev)
        out, saved = decoder.attention_fwd(q, k, v, causal=causal, lengths=dl)
        again = (out, *saved, *decoder.attention_bwd(do, q, k, v, out, saved, causal=causal, lengths=dl))
        for a, b in zip(clean, again):
            assert torch.equal(a, b)


@gpu
def test_attention_large_scores(dev):
    """Scores over hundreds, in rising order (the running maximum moves at every step) and falling."""
    for flip in (False, True):
        q, k, v, do = attention_inputs(1, 300, 2, 2, 128, BF16, dev, seed=3)
        ramp = torch.linspace(-40, 40, 300, device=dev)
        ramp = ramp.flip(0) if flip else ramp
        k = (k.float() * 0.1 + ramp[None, :, None, None] * (torch.arange(128, device=dev) % 2)).to(BF16)
        q = (q.float() * 0.1 + 0.5 * (torch.arange(128, device=dev) % 2)).to(BF16)
        for causal in (True, False):
            attention_check(q, k, v, do, causal)
            attention_check(q, k, v, do, causal, scale=0.31)


@gpu
@pytest.mark.parametrize("four", [0, 4])
def test_attention_scores_rising_in_turn(dev, four):
    """Keys whose scores rise lie in every other group of four, which half of a wave's lanes see."""
    q, k, v, do = attention_inputs(1, 333, 2, 1, 64, F16, dev, seed=4)
    j = torch.arange(333, device=dev)
    ramp = torch.where((j & 4) == four, j / 333.0 * 30, torch.zeros_like(j, dtype=torch.float32))
    k = (k.float() * 0.1 + ramp[None, :, None, None] * (torch.arange(64, device=dev) % 2)).to(F16)
    q = (q.float() * 0.1 + 0.3 * (torch.arange(64, device=dev) % 2)).to(F16)
    for causal in (True, False):
        attention_check(q, k, v, do, causal)


@gpu
def test_attention_layouts(dev):
    """Views of a packed projection, heads before positions, expanded heads, odd strides, loose pointers."""
    B, S, H, Hk, D = 2, 77, 4, 2, 64
    q, k, v, do = attention_inputs(B, S, H, Hk, D, F16, dev, seed=4)
    want = attention_check(q, k, v, do, True)
    packed = torch.cat([q, k, v], dim=2)
    views = packed[:, :, :H], packed[:, :, H:H + Hk], packed[:, :, H + Hk:]
    across = tuple(x.transpose(1, 2).contiguous().transpose(1, 2) for x in (q, k, v))
    wide = []
    for x in (q, k, v):
        y = torch.full((B, S, x.shape[2], D + 5), math.nan, dtype=F16, device=dev)
        y[..., 3:3 + D] = x
        wide.append(y[..., 3:3 + D])
    last = tuple(x.transpose(1, 3).contiguous().transpose(1, 3) for x in (q, k, v))
    loose = []
    for x in (q, k, v):
        y = torch.empty(x.numel() + 1, dtype=F16, device=dev)
        y[1:] = x.reshape(-1)
        loose.append(y[1:].view(x.shape))
    for a in (views, across, wide, last, loose):
        out, lse = decoder.attention_fwd(*a)
        assert torch.equal(out, want[0])
        for x, y in zip(decoder.attention_bwd(do, *a, out, lse), want[2:]):
            assert torch.equal(x, y)
    # gradient and output tensors of other layouts
    out, lse = want[:2]
    tr = lambda x: x.transpose(1, 2).contiguous().transpose(1, 2)  # noqa: E731
    for x, y in zip(decoder.attention_bwd(tr(do), q, k, v, tr(out), lse), want[2:]):
        assert torch.equal(x, y)
    one = do[:, :1, :1].expand(B, S, H, D)
    for x, y in zip(decoder.attention_bwd(one, q, k, v, out, lse), decoder.attention_bwd(one.contiguous(), q, k, v, out, lse)):
        assert torch.equal(x, y)
    ek = k[:, :, :1].expand(B, S, Hk, D)
    assert torch.equal(decoder.attention(q, ek, v), decoder.attention(q, ek.contiguous(), v))


@gpu
def test_attention_autograd(dev):
    """The differentiable forms return the pairs' gradients; a packed projection gets one."""
    B, S, H, Hk, D = 2, 130, 6, 2, 64
    q, k, v, do = attention_inputs(B, S, H, Hk, D, BF16, dev, seed=8)
    lengths = torch.tensor([130, 40], dtype=torch.int32, device=dev)
    out, lse = decoder.attention_fwd(q, k, v, lengths=lengths)
    want = decoder.attention_bwd(do, q, k, v, out, lse, lengths=lengths)
    a = [x.clone().requires_grad_() for x in (q, k, v)]
    got = decoder.attention(*a, lengths=lengths)
    assert torch.equal(got, out)
    got.backward(do)
    for x, y in zip(a, want):
        assert torch.equal(x.grad, y)
    packed = torch.cat([q, k, v], 2).requires_grad_()
    got = decoder.attention_qkv(packed, H, lengths=lengths)
    got.backward(do)
    assert torch.equal(got, out) and torch.equal(packed.grad, torch.cat(want, 2))
    k2 = k.clone().requires_grad_()
    decoder.attention(q, k2, v, lengths=lengths).backward(do)
    assert torch.equal(k2.grad, want[1])
    with torch.no_grad():
        assert not decoder.attention(*a, lengths=lengths).requires_grad


@gpu
def test_attention_gradient_by_differences(dev):
    """The gradient's product with a direction against a difference of the 64-bit definition."""
    q, k, v, do = attention_inputs(1, 90, 2, 1, 64, F16, dev, seed=9)
    out, lse = decoder.attention_fwd(q, k, v)
    grads = decoder.attention_bwd(do, q, k, v, out, lse)
    ref, tol, _ = attention_oracle(q, k, v, do, True, 64 ** -0.5, [90])

    def value(q, k, v):
        s = torch.matmul(q.transpose(1, 2).contiguous(), k.expand(1, 90, 2, 64).permute(0, 2, 3, 1).contiguous()) / 8
        s = s.masked_fill(torch.ones(90, 90, dtype=torch.bool, device=dev).triu(1), -math.inf)
        o = torch.matmul(torch.softmax(s, -1), v.expand(1, 90, 2, 64).transpose(1, 2).contiguous())
        return (o.transpose(1, 2) * do.double()).sum()

    x = [t.double() for t in (q, k, v)]
    for i, n in enumerate(("dq", "dk", "dv")):
        way = torch.randn(x[i].shape, dtype=torch.float64, device=dev, generator=torch.Generator(device=dev).manual_seed(i))
        h = 1e-4
        lo, hi = list(x), list(x)
        lo[i], hi[i] = x[i] - h * way, x[i] + h * way
        slope = (value(*hi) - value(*lo)) / (2 * h)
        # the difference's own error is O(h^2) of third derivatives: 1e-6 relative to the terms' sum
        bound = (tol[n] * way.abs()).sum() + 1e-6 * (ref[n] * way).abs().sum()
        assert abs((grads[i].double() * way).sum() - slope) <= bound, n


@gpu
def test_attention_empty(dev):
    for shape in ((0, 5, 2, 64), (3, 0, 2, 64)):
        q = torch.zeros(shape, dtype=BF16, device=dev)
        out, lse = decoder.attention_fwd(q, q, q)
        assert out.shape == shape and lse[0].shape == (shape[0], 2, shape[1])
        assert all(x.shape == shape for x in decoder.attention_bwd(q, q, q, q, out, lse))


@gpu
def test_attention_far_apart(dev):
    """Positions 8 MiB apart: a sequence spans more than 2^31 bytes."""
    S, D = 300, 128
    base = torch.empty(S, 1 << 22, dtype=BF16, device=dev)
    views = []
    for i, x in enumerate(attention_inputs(1, S, 2, 1, D, BF16, dev, seed=9)):
        to = base[:, i * 1000 * 8:][:, :x.shape[2] * D].view(1, S, x.shape[2], D)
        views.append(to.copy_(x))
    assert views[0].stride(1) * S * 2 > 2 ** 31 and not views[0].is_contiguous()
    for causal in (True, False):
        attention_check(*views, causal)
        attention_check(*views, causal, lengths=[271])


@gpu
def test_attention_long_padded(dev):
    """Over 2^31 elements of mostly padding, which is NaN: not read, and zero in the results."""
    B, S, H, D, ends = 2, (1 << 20) + 64, 16, 128, [70, 200]
    full = lambda h: torch.full((B, S, h, D), math.nan, dtype=BF16, device=dev)  # noqa: E731
    q, k, v, do = full(H), full(1), full(1), full(H)
    small = attention_inputs(B, 200, H, 1, D, BF16, dev, seed=10)
    for x, y in zip((q, k, v, do), small):
        x[:, :200] = y
        for b, n in enumerate(ends):
            x[b, n:200] = math.nan
            y[b, n:] = 0
    kw = {"lengths": torch.tensor(ends, dtype=torch.int32, device=dev)}
    out, saved = decoder.attention_fwd(q, k, v, **kw)
    got = (out, *decoder.attention_bwd(do, q, k, v, out, saved, **kw))
    ref, tol, _ = attention_oracle(*small, True, D ** -0.5, ends)
    for name, x in zip(("out", "dq", "dk", "dv"), got):
        close(x[:, :200], ref[name], tol[name], name)
        for b in range(B):
            assert not x[b, 200:].any()


# ------------------------------------------------------------------------ swiglu's oracle

def swiglu_oracle(x, w, dh):
    """Results, gradients and tolerances in 64 bits: x [T, K], w [2F, K], dh [T, F]."""
    u, (F, K), T = half_step(x.dtype), (w.shape[0] // 2, w.shape[1]), x.shape[0]
    sub = 2.0 ** -25 if x.dtype == F16 else 0.0
    X, W, G = x.double(), w.double(), dh.double()
    gu = mm(X, W.t())
    e = E32 * (K + 4) * mm(X.abs(), W.abs().t())
    g, up, eg, eu = gu[:, :F], gu[:, F:], e[:, :F], e[:, F:]
    s = torch.sigmoid(g)
    act, slope = g * s, s * (1 + g * (1 - s))
    h = act * up
    # |silu'| <= 1.1, |silu''| <= 0.5
    r = {"h": h, "saved": gu}
    tol = {"h": u * h.abs() + 1.01 * (1.1 * up.abs() * eg + act.abs() * eu) + 16 * E32 * h.abs() + sub,
           "saved": e + 2.0 ** -16 * gu.abs()}  # 24 of 32 bits: 23 - 8 = 15 of the fraction, half a step is 2^-16
    dg, du = G * up * slope, G * act
    # the backward sees g and u as saved, rounds dg and du
    rg, ru = tol["saved"][:, :F], tol["saved"][:, F:]
    e_dg = 1.02 * G.abs() * (up.abs() * 0.5 * rg + 1.1 * ru) + (u + 16 * E32) * dg.abs() + sub
    e_du = 1.02 * G.abs() * 1.1 * rg + (u + 16 * E32) * du.abs() + sub
    d, e_d = torch.cat([dg, du], 1), 1.02 * torch.cat([e_dg, e_du], 1)
    r["dx"], r["dw"] = mm(d, W), mm(d.t(), X)
    tol["dx"] = u * r["dx"].abs() + mm(e_d + E32 * (2 * F + 20) * d.abs(), W.abs()) + sub
    tol["dw"] = u * r["dw"].abs() + mm((e_d + E32 * (T + 20) * d.abs()).t(), X.abs()) + sub
    return r, tol


def swiglu_inputs(T, K, F, t, dev, seed=0):
    g = torch.Generator(device=dev).manual_seed(seed)
    mk = lambda *s, std=1.0: (torch.randn(*s, generator=g, device=dev) * std).to(t)  # noqa: E731
    return mk(T, K), mk(2 * F, K, std=K ** -0.5), mk(T, F)


def projections(saved):
    """The 32-bit values of a ``saved`` of swiglu_fwd, [..., 2 inner]."""
    n = saved.shape[-1] // 3
    high = saved[..., :2 * n].contiguous().view(torch.int16).int() << 16
    return (high | (saved[..., 2 * n:].int() << 8)).view(F32)


def swiglu_check(x, w, dh):
    h, saved = decoder.swiglu_fwd(x, w)
    dx, dw = decoder.swiglu_bwd(dh, x, w, saved)
    ref, tol = swiglu_oracle(x.reshape(-1, x.shape[-1]), w, dh.reshape(-1, dh.shape[-1]))
    for n, got in (("h", h), ("saved", projections(saved)), ("dx", dx), ("dw", dw)):
        close(got.reshape(ref[n].shape), ref[n], tol[n], n)
    assert torch.equal(decoder.swiglu(x, w), h)
    return h, saved, dx, dw


@gpu
@pytest.mark.parametrize("t", [BF16, F16])
@pytest.mark.parametrize("T,K,F", [(1, 8, 8), (1, 64, 40), (3, 72, 8), (5, 4096, 264), (17, 520, 1032), (31, 128, 64),
                                   (64, 64, 64), (65, 200, 136), (129, 1000, 520), (257, 264, 264), (1000, 8, 2000),
                                   (700, 2000, 8)])
def test_swiglu_sizes(dev, T, K, F, t):
    swiglu_check(*swiglu_inputs(T, K, F, t, dev, seed=T))


@gpu
@pytest.mark.parametrize("t,T,K,F", [(BF16, 4001, 200, 2056), (F16, 4095, 4104, 2048)])
def test_swiglu_large(dev, t, T, K, F):
    swiglu_check(*swiglu_inputs(T, K, F, t, dev, seed=T))


@gpu
@pytest.mark.parametrize("splits", [1, 3])
@pytest.mark.parametrize("tile", decoder.PRODUCT_TILES)
def test_swiglu_every_tile(dev, monkeypatch, tile, splits):
    """Each tile, whole and with the sum in parts, on sizes that fill none and are not what it is chosen for."""
    monkeypatch.setattr(decoder, "_product_plan", lambda M, N, K, forward=False: (tile if forward or tile != 2 else 0, min(splits, -(-K // 64))))
    for t, T, K, F in ((BF16, 300, 328, 200), (F16, 9, 200, 520), (BF16, 530, 8, 8)):
        swiglu_check(*swiglu_inputs(T, K, F, t, dev, seed=T))


@gpu
def test_swiglu_layouts(dev):
    """Leading dimensions, row strides, loose pointers, transposed weights, an expanded gradient."""
    x, w, dh = swiglu_inputs(6 * 7, 72, 40, BF16, dev)
    want = swiglu_check(x, w, dh)
    h, saved = decoder.swiglu_fwd(x.view(6, 7, 72), w)
    assert h.shape == (6, 7, 40) and torch.equal(h.view(42, 40), want[0])
    dx, dw = decoder.swiglu_bwd(dh.view(6, 7, 40), x.view(6, 7, 72), w, saved)
    assert dx.shape == (6, 7, 72) and torch.equal(dx.view(42, 72), want[2]) and torch.equal(dw, want[3])
    big = torch.full((42, 88), math.nan, dtype=BF16, device=dev)
    for at in (0, 8, 3):  # aligned in place, aligned in place, copied
        big[:, at:at + 72] = x
        a = big[:, at:at + 72]
        wt = w.t().contiguous().t()
        h, saved = decoder.swiglu_fwd(a, wt)
        dx, dw = decoder.swiglu_bwd(dh.t().contiguous().t(), a, wt, saved)
        for p, q in zip((h, saved, dx, dw), want):
            assert torch.equal(p, q)
    one = dh[:1].expand(42, 40)
    for p, q in zip(decoder.swiglu_bwd(one, x, w, want[1]), decoder.swiglu_bwd(one.contiguous(), x, w, want[1])):
        assert torch.equal(p, q)


@gpu
def test_swiglu_garbage_beside_the_rows(dev):
    """What lies between strided rows is not part of the sums, whatever it holds."""
    T, K, F = 70, 72, 40
    x, w, dh = swiglu_inputs(T, K, F, F16, dev, seed=2)
    want = swiglu_check(x, w, dh)
    hold = [torch.full((n + 40, m + 128), math.nan, dtype=F16, device=dev) for n, m in ((T, K), (2 * F, K), (T, F))]
    for b, t in zip(hold, (x, w, dh)):
        b[16:16 + t.shape[0], 64:64 + t.shape[1]] = t
    x, w, dh = (b[16:16 + t.shape[0], 64:64 + t.shape[1]] for b, t in zip(hold, (x, w, dh)))
    h, saved = decoder.swiglu_fwd(x, w)
    for p, q in zip((h, saved, *decoder.swiglu_bwd(dh, x, w, saved)), want):
        assert torch.equal(p, q)


@gpu
def test_swiglu_extremes(dev):
    """Gates far out on both sides: silu is 0 or the gate itself, its slope 0 or 1, nothing overflows."""
    x = torch.eye(8, dtype=BF16, device=dev)
    g = torch.tensor([-3e4, -200.0, -89.0, -1e-30, 0.0, 1e-30, 89.0, 3e4], device=dev)
    w = torch.cat([torch.diag(g), 2 * torch.eye(8, device=dev)]).to(BF16)
    h, saved = decoder.swiglu_fwd(x, w)
    dx, dw = decoder.swiglu_bwd(torch.ones(8, 8, dtype=BF16, device=dev), x, w, saved)
    assert torch.isfinite(h).all() and torch.isfinite(dx).all() and torch.isfinite(dw).all()
    gd = w[:8].double().diagonal()
    assert torch.allclose(h.double().diagonal(), 2 * gd * torch.sigmoid(gd), rtol=2 ** -7, atol=1e-30)


@gpu
def test_swiglu_offsets(dev):
    """Over 2^31 elements of h ; gradients of the last rows."""
    T, K, F, n = 262147, 64, 8200, 5
    g = torch.Generator(device=dev).manual_seed(11)
    x = torch.randn(T, K, generator=g, device=dev).to(BF16)
    w = (torch.randn(2 * F, K, generator=g, device=dev) * K ** -0.5).to(BF16)
    dh = torch.zeros(T, F, dtype=BF16, device=dev)
    dh[-n:] = torch.randn(n, F, generator=g, device=dev).to(BF16)
    h, saved = decoder.swiglu_fwd(x, w)
    dx, dw = decoder.swiglu_bwd(dh, x, w, saved)
    rows = torch.cat([torch.arange(0, T - n, 26003), torch.arange(T - n, T)]).to(dev)
    ref, tol = swiglu_oracle(x[rows], w, dh[rows])
    for name, got in (("h", h[rows]), ("saved", projections(saved[rows])), ("dx", dx[rows]), ("dw", dw)):
        close(got, ref[name], tol[name], name)


@gpu
def test_swiglu_far_apart(dev):
    """Rows 4 MiB apart, over 2^31 bytes in all, of x and w."""
    T, K, F = 600, 72, 296
    x, w, dh = swiglu_inputs(T, K, F, BF16, dev, seed=12)
    base = torch.empty(600, 1 << 21, dtype=BF16, device=dev)
    far = [base[:len(t), i * 8000:][:, :t.shape[1]].copy_(t) for i, t in enumerate((x, w, dh))]
    assert far[0].stride(0) * T * 2 > 2 ** 31
    swiglu_check(*far)


@gpu
def test_swiglu_autograd(dev):
    x, w, dh = swiglu_inputs(50, 64, 48, BF16, dev)
    want = swiglu_check(x, w, dh)
    a, b = x.view(5, 10, 64).clone().requires_grad_(), w.clone().requires_grad_()
    h = decoder.swiglu(a, b)
    h.backward(dh.view(5, 10, 48))
    assert torch.equal(h.view(50, 48), want[0]) and torch.equal(a.grad.view(50, 64), want[2]) and torch.equal(b.grad, want[3])
    b2 = w.clone().requires_grad_()
    decoder.swiglu(x, b2).backward(dh)
    assert torch.equal(b2.grad, want[3])
    a2 = x.clone().requires_grad_()
    decoder.swiglu(a2, w).backward(dh)
    assert torch.equal(a2.grad, want[2])
    # one gradient wanted where both products' sums are cut into parts
    x, w, dh = swiglu_inputs(1100, 72, 1032, BF16, dev)
    assert decoder._product_plan(1100, 72, 2064)[1] > 1 and decoder._product_plan(2064, 72, 1100)[1] > 1
    want = swiglu_check(x, w, dh)
    a2, b2 = x.clone().requires_grad_(), w.clone().requires_grad_()
    decoder.swiglu(a2, w).backward(dh)
    decoder.swiglu(x, b2).backward(dh)
    assert torch.equal(a2.grad, want[2]) and torch.equal(b2.grad, want[3])


@gpu
def test_swiglu_empty(dev):
    x = torch.zeros(0, 64, dtype=BF16, device=dev)
    w = torch.ones(16, 64, dtype=BF16, device=dev)
    h, saved = decoder.swiglu_fwd(x, w)
    dx, dw = decoder.swiglu_bwd(h, x, w, saved)
    assert h.shape == (0, 8) and dx.shape == (0, 64) and (dw == 0).all() and dw.shape == w.shape


# ----------------------------------------------------------------------- add_norm's oracle

def norm_oracle(r, b, w, pw, gate, scale, eps, dS, dy):
    t = r.dtype
    u, C, T = half_step(t), r.shape[1], r.shape[0]
    sub = 2.0 ** -25 if t == F16 else 0.0
    # a 32-bit sum over a row: 16 products a thread, 6 exchanges, 16 waves; quotient, root, products
    e = 64 * E32
    ones = torch.ones(C, dtype=torch.float64, device=r.device)
    R, B, W, PW, G = (x.double() if x is not None else ones for x in (r, b, w, pw, gate))
    rb = (B.square().mean(1, keepdim=True) + eps).rsqrt() if pw is not None else torch.ones(T, 1, dtype=torch.float64, device=r.device)
    bh = B * rb
    add = scale * G * PW * bh
    s = R + add
    rs = (s.square().mean(1, keepdim=True) + eps).rsqrt()
    sh = s * rs
    out = {"stream": s, "out": W * sh}
    e_s = e * (R.abs() + add.abs())
    tol = {"stream": u * s.abs() + e_s + sub}
    # a relative error of the mean of squares from e_s: at most 2 |s| e_s / mean s^2
    e_rs = e + (s.abs() * e_s).mean(1, keepdim=True) * rs ** 2
    e_sh = sh.abs() * e_rs + e_s * rs
    tol["out"] = u * out["out"].abs() + W.abs() * (e_sh + e * sh.abs()) + sub
    DS = torch.zeros_like(s) if dS is None else dS.double()
    DY = torch.zeros_like(s) if dy is None else dy.double()
    a = W * DY
    m = (a * sh).mean(1, keepdim=True)
    ds = DS + rs * (a - sh * m)
    # the stream is added up again, rs is the forward's
    e_sh = rs * e_s + sh.abs() * (e_rs + e)
    e_m = (a.abs() * e_sh + 2 * e * a.abs() * sh.abs()).mean(1, keepdim=True)
    e_ds = 1.02 * (rs * (e_sh * m.abs() + sh.abs() * e_m) + (e + e_rs) * (DS.abs() + rs * (a.abs() + sh.abs() * m.abs())))
    tm = scale * ds
    dn = G * tm
    x = PW * dn
    m2 = (x * bh).mean(1, keepdim=True) if pw is not None else 0.0 * rb
    db = rb * (x - bh * m2)
    e_t = abs(scale) * (e_ds + e * ds.abs())
    e_x = PW.abs() * G.abs() * e_t + e * x.abs()
    e_m2 = (bh.abs() * e_x + 2 * e * x.abs() * bh.abs()).mean(1, keepdim=True) if pw is not None else 0.0 * rb
    e_db = 1.02 * rb * (e_x + bh.abs() * e_m2 + e * (x.abs() + 3 * bh.abs() * m2.abs()))
    out.update(dresidual=ds, dbranch=db, dweight=(DY * sh).sum(0))
    tol.update(dresidual=e_ds + u * ds.abs() + sub, dbranch=e_db + u * db.abs() + sub)
    far = E32 * (T + 64)  # the order of a column's sum
    tol["dweight"] = u * out["dweight"].abs() + (DY.abs() * (e_sh + (far + e) * sh.abs())).sum(0) + sub
    if pw is not None:
        out["dpost_weight"] = (dn * bh).sum(0)
        tol["dpost_weight"] = u * out["dpost_weight"].abs() + (bh.abs() * (G.abs() * e_t + (far + e) * dn.abs())).sum(0) + sub
    if gate is not None:
        n = PW * bh
        out["dgate"] = (tm * n).sum(0)
        tol["dgate"] = u * out["dgate"].abs() + (n.abs() * (e_t + (far + e) * tm.abs())).sum(0) + sub
    return out, tol


NORM_GRADS = ("dresidual", "dbranch", "dweight", "dpost_weight", "dgate")


def norm_inputs(T, C, t, dev, post, gate, seed=0):
    g = torch.Generator(device=dev).manual_seed(seed)
    mk = lambda *s, std=1.0, mean=0.0: (torch.randn(*s, generator=g, device=dev) * std + mean).to(t)  # noqa: E731
    return (mk(T, C), mk(T, C, std=2.0), mk(C, std=0.3, mean=1.0), mk(C, std=0.3, mean=1.0) if post else None,
            mk(C, std=0.5) if gate else None, mk(T, C), mk(T, C))


def norm_check(r, b, w, pw, gate, dS, dy, scale=1.0, eps=1e-5):
    kw = {"post_weight": pw, "gate": gate, "scale": scale, "eps": eps}
    s, y, saved = decoder.add_norm_fwd(r, b, w, **kw)
    grads = decoder.add_norm_bwd(dS, dy, r, b, w, saved, **kw)
    flat = lambda x: None if x is None else x.reshape(-1, x.shape[-1])  # noqa: E731
    ref, tol = norm_oracle(flat(r), flat(b), w, pw, gate, scale, eps, flat(dS), flat(dy))
    for n, got in (("stream", s), ("out", y), *zip(NORM_GRADS, grads)):
        if n not in ref:
            assert got is None
            continue
        close(got.reshape(ref[n].shape), ref[n], tol[n], n)
    one, two = decoder.add_norm(r, b, w, **kw)
    assert torch.equal(one, s) and torch.equal(two, y)
    return s, y, saved, grads


@gpu
@pytest.mark.parametrize("t", [BF16, F16, F32])
@pytest.mark.parametrize("C", [1, 7, 8, 64, 300, 512, 513, 2047, 2048, 2056, 4096, 4101, 8192, 8200, 16384])
@pytest.mark.parametrize("post,gate,scale", [(False, False, 1.0), (True, True, 0.7), (True, False, 1.0), (False, True, 1.0),
                                             (False, False, -0.5)])
def test_add_norm_sizes(dev, C, t, post, gate, scale):
    for T in (1, 5, 37):
        norm_check(*norm_inputs(T, C, t, dev, post, gate, seed=C + T), scale=scale)


@gpu
@pytest.mark.parametrize("t,T,C", [(BF16, 3000, 2048), (F16, 2100, 72), (F32, 9000, 16), (BF16, 1500, 8192), (F16, 700, 10000)])
def test_add_norm_many_rows(dev, t, T, C):
    """More rows than parts: a workgroup adds several rows to its column sums."""
    norm_check(*norm_inputs(T, C, t, dev, True, True, seed=T), scale=0.3)
    norm_check(*norm_inputs(T, C, t, dev, False, False, seed=T))


@gpu
def test_add_norm_missing_gradients(dev):
    for full in (False, True):
        a = norm_inputs(20, 130, BF16, dev, full, full)
        norm_check(*a[:5], None, a[6])
        norm_check(*a[:5], a[5], None)
    dr, db = decoder.add_norm_bwd(a[5], a[6], a[0], a[1], a[2], torch.ones(2, 20, device=dev))[:2]
    assert dr is db


@gpu
def test_add_norm_zero_rows_and_layouts(dev):
    """Rows of zeros (eps alone under the root), leading dimensions, row strides, expanded rows."""
    r, b, w, pw, gate, dS, dy = norm_inputs(12, 200, BF16, dev, True, True)
    r[3] = 0
    b[3] = 0
    want = norm_check(r, b, w, pw, gate, dS, dy)
    assert (want[1][3] == 0).all()
    shaped = lambda x: x.view(3, 4, 200)  # noqa: E731
    got = norm_check(shaped(r), shaped(b), w, pw, gate, shaped(dS), shaped(dy))
    assert got[1].shape == (3, 4, 200)
    for x, y in zip(got[3], want[3]):
        assert torch.equal(x.reshape(y.shape), y)
    def wide(x):
        y = torch.full((12, 207), math.nan, dtype=BF16, device=dev)
        y[:, 3:203] = x
        return y[:, 3:203]
    def tall(x):
        return x.t().contiguous().t()
    for f in (wide, tall):
        kw = {"post_weight": pw, "gate": gate, "eps": 1e-5}
        s, y, saved = decoder.add_norm_fwd(f(r), f(b), w, **kw)
        assert torch.equal(s, want[0]) and torch.equal(y, want[1])
        for x, z in zip(decoder.add_norm_bwd(f(dS), f(dy), f(r), f(b), w, saved, **kw), want[3]):
            assert torch.equal(x, z)
    row = dy[:1].expand(12, 200)
    norm_check(r, b[:1].expand(12, 200), w, pw, gate, row, row)


@gpu
@pytest.mark.parametrize("C", [300, 1000])
def test_add_norm_far_apart(dev, C):
    """Rows 2 GiB apart."""
    r, b, w, pw, gate, dS, dy = norm_inputs(3, C, BF16, dev, True, True, seed=13)
    base = torch.empty(2 * (1 << 30) + 8192, dtype=BF16, device=dev)
    far = [base[i * 1024 + 1:].as_strided((3, C), (1 << 30, 1)).copy_(t) for i, t in enumerate((r, b, dS, dy))]
    norm_check(far[0], far[1], w, pw, gate, far[2], far[3])


@gpu
@pytest.mark.parametrize("T,C", [((1 << 21) + 3, 1024), ((1 << 26) + 3, 33)])
def test_add_norm_offsets(dev, T, C):
    """Over 2^31 elements; gradients of the last rows."""
    n = 5
    last = norm_inputs(n, C, BF16, dev, False, False, seed=14)
    r, b, dS, dy = (torch.zeros(T, C, dtype=BF16, device=dev) for _ in range(4))
    for to, x in zip((r, b, dS, dy), (last[0], last[1], last[5], last[6])):
        to[-n:] = x
    s, y, saved = decoder.add_norm_fwd(r, b, last[2], eps=1e-5)
    grads = decoder.add_norm_bwd(dS, dy, r, b, last[2], saved, eps=1e-5)
    ref, tol = norm_oracle(*last[:5], 1.0, 1e-5, *last[5:])
    for name, x in (("stream", s), ("out", y), *zip(NORM_GRADS[:2], grads)):
        close(x[-n:], ref[name], tol[name], name)
        assert not x[:-n].any()
    close(grads[2], ref["dweight"], tol["dweight"], "dweight")


@gpu
def test_add_norm_autograd(dev):
    a = norm_inputs(30, 96, F32, dev, True, True)
    want = norm_check(*a, scale=0.4)
    leaves = [x.clone().requires_grad_() for x in a[:5]]
    s, y = decoder.add_norm(leaves[0], leaves[1], leaves[2], post_weight=leaves[3], gate=leaves[4], scale=0.4, eps=1e-5)
    torch.autograd.backward([s, y], [a[5], a[6]])
    for x, z in zip(leaves, want[3]):
        assert torch.equal(x.grad, z)
    # one result used, one tensor wanted; residual and branch one tensor: both gradients arrive
    x = a[0].clone().requires_grad_()
    decoder.add_norm(x, x, a[2])[1].backward(a[6])
    s, y, saved = decoder.add_norm_fwd(a[0], a[0], a[2])
    g = decoder.add_norm_bwd(None, a[6], a[0], a[0], a[2], saved)
    assert torch.equal(x.grad, g[0] + g[1])
    r, b = a[0].clone().requires_grad_(), a[1].clone().requires_grad_()
    decoder.add_norm(r, b, a[2])[0].backward(a[5])
    assert torch.equal(r.grad, a[5]) and torch.equal(b.grad, a[5]) and r.grad.data_ptr() != b.grad.data_ptr()


@gpu
def test_add_norm_empty(dev):
    x, w = torch.zeros(0, 64, dtype=BF16, device=dev), torch.ones(64, dtype=BF16, device=dev)
    s, y, saved = decoder.add_norm_fwd(x, x, w, gate=w)
    g = decoder.add_norm_bwd(s, y, x, x, w, saved, gate=w)
    assert s.shape == y.shape == g[0].shape == (0, 64) and (g[2] == 0).all() and (g[4] == 0).all() and g[3] is None


# ------------------------------------------------------- streams, graphs, equal bits, a run of them

def block_step(x, ws, lengths, grads):
    """norm - attention - norm - gate and back, on explicit pairs: every gradient."""
    w0, wq, w1, wgu, wd = ws
    B, S, C = x.shape
    H, Hk, D = 4, 2, 64
    s0, y0, k0 = decoder.add_norm_fwd(x, x, w0, scale=0.5)
    qkv = torch.matmul(y0, wq).view(B, S, H + 2 * Hk, D)
    q, k, v = qkv[:, :, :H], qkv[:, :, H:H + Hk], qkv[:, :, H + Hk:]
    o, lse = decoder.attention_fwd(q, k, v, lengths=lengths)
    s1, y1, k1 = decoder.add_norm_fwd(s0, o.view(B, S, H * D), w1)
    h, kept = decoder.swiglu_fwd(y1, wgu)
    z = torch.matmul(h, wd)
    dh = torch.matmul(grads, wd.t().contiguous())
    dy1, dwgu = decoder.swiglu_bwd(dh, y1, wgu, kept)
    ds0, do, dw1, _, _ = decoder.add_norm_bwd(grads, dy1, s0, o.view(B, S, H * D), w1, k1)
    dq, dk, dv = decoder.attention_bwd(do.view(B, S, H, D), q, k, v, o, lse, lengths=lengths)
    dqkv = torch.cat([dq, dk, dv], 2).view(B, S, -1)
    dy0 = torch.matmul(dqkv, wq.t().contiguous())
    dx, dx2, dw0, _, _ = decoder.add_norm_bwd(ds0, dy0, x, x, w0, k0, scale=0.5)
    return z, dx, dx2, dw0, dw1, dwgu, dq, dk, dv


def block_inputs(dev, t=BF16, B=2, S=70, seed=21):
    g = torch.Generator(device=dev).manual_seed(seed)
    mk = lambda *s, std=1.0, mean=0.0: (torch.randn(*s, generator=g, device=dev) * std + mean).to(t)  # noqa: E731
    C = 256
    ws = mk(C, std=0.2, mean=1), mk(C, 8 * 64, std=C ** -0.5), mk(C, std=0.2, mean=1), mk(2 * 320, C, std=C ** -0.5), mk(320, C, std=0.05)
    return mk(B, S, C), ws, torch.tensor([S, 33], dtype=torch.int32, device=dev), mk(B, S, C)


@gpu
def test_block_runs_together(dev):
    """The operators one after the other, as a decoder block uses them, against the same block in 64 bits."""
    x, ws, lengths, gr = block_inputs(dev, F16)
    leaf = x.clone().requires_grad_()
    w = [t.clone().requires_grad_() for t in ws]
    s0, y0 = decoder.add_norm(leaf, leaf, w[0], scale=0.5)
    o = decoder.attention_qkv(torch.matmul(y0, w[1]).view(2, 70, 8, 64), 4, lengths=lengths)
    s1, y1 = decoder.add_norm(s0, o.reshape(2, 70, 256), w[2])
    z = s1 + torch.matmul(decoder.swiglu(y1, w[3]), w[4])
    z.backward(gr)

    leaf64 = x.double().requires_grad_()
    w64 = [t.double().requires_grad_() for t in ws]

    def norm(v, weight):
        return v * (v.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * weight
    s = leaf64 + 0.5 * leaf64
    qkv = torch.matmul(norm(s, w64[0]), w64[1]).view(2, 70, 8, 64)
    q, k, v = (a.transpose(1, 2) for a in (qkv[:, :, :4], qkv[:, :, 4:6].repeat_interleave(2, 2), qkv[:, :, 6:].repeat_interleave(2, 2)))
    sc = torch.matmul(q, k.transpose(-1, -2)) / 8
    i = torch.arange(70, device=dev)
    live = (i[None, :] <= i[:, None])[None] & (i[None, None, :] < lengths[:, None, None])
    p = torch.softmax(sc.masked_fill(~live[:, None], -math.inf), -1)
    oo = torch.matmul(p, v) * (i[None, :] < lengths[:, None])[:, None, :, None]
    s = s + oo.transpose(1, 2).reshape(2, 70, 256)
    gu = torch.matmul(norm(s, w64[2]), w64[3].t())
    z64 = s + torch.matmul(torch.nn.functional.silu(gu[..., :320]) * gu[..., 320:], w64[4])
    z64.backward(gr.double())
    # A chain of about a dozen rounded tensors: each adds at most half a step in the mean square, and the
    # chain's gains here are about one; 12 half steps of the whole.
    for a, b, n in [(z, z64, "z"), (leaf.grad, leaf64.grad, "x")] + [(p1.grad, p2.grad, f"w{j}") for j, (p1, p2) in enumerate(zip(w, w64))]:
        err = (a.double() - b).norm() / b.norm()
        assert err < 12 * half_step(F16), (n, err.item())


@gpu
def test_equal_bits(dev):
    x, ws, lengths, gr = block_inputs(dev)
    a, b = block_step(x, ws, lengths, gr), block_step(x, ws, lengths, gr)
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    q, k, v, do = attention_inputs(1, 1100, 8, 1, 64, BF16, dev)
    out, lse = decoder.attention_fwd(q, k, v)
    one, two = (decoder.attention_bwd(do, q, k, v, out, lse) for _ in range(2))
    assert all(torch.equal(p, r) for p, r in zip(one, two))


@gpu
def test_graph_replays(dev):
    """Captured and replayed with new values in the inputs, eager work between; two graphs side by side."""
    x, ws, lengths, gr = block_inputs(dev)
    x2 = block_inputs(dev, seed=77)[0]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        block_step(x, ws, lengths, gr)
    torch.cuda.current_stream().wait_stream(s)
    graphs = []
    for inp in (x.clone(), x2.clone()):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            res = block_step(inp, ws, lengths, gr)
        graphs.append((g, inp, res))
    for k in range(4):
        fresh = [block_inputs(dev, seed=100 + 2 * k + i)[0] for i in range(2)]
        want = [block_step(f, ws, lengths, gr) for f in fresh]
        for (g, inp, _), f in zip(graphs, fresh):
            inp.copy_(f)
        for g, _, _ in graphs:
            g.replay()
        torch.cuda.synchronize()
        for (_, _, res), w in zip(graphs, want):
            assert all(torch.equal(p, q) for p, q in zip(res, w)), k


@gpu
@pytest.mark.parametrize("tile,T", [(0, 300), (1, 300), (2, 9)])
def test_graph_of_every_tile(dev, monkeypatch, tile, T):
    """Products whose workgroups take more LDS than a launch has by default, captured before they ever ran."""
    monkeypatch.setattr(decoder, "_product_plan", lambda M, N, K, forward=False: (tile if forward or tile != 2 else 0, 2))
    x, w, dh = swiglu_inputs(T, 328, 264, F16, dev, seed=6)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        h, saved = decoder.swiglu_fwd(x, w)
        got = (h, *decoder.swiglu_bwd(dh, x, w, saved))
    for seed in (6, 7, 8):
        y = swiglu_inputs(T, 328, 264, F16, dev, seed=seed)
        for a, b in zip((x, w, dh), y):
            a.copy_(b)
        g.replay()
        torch.cuda.synchronize()
        h, saved = decoder.swiglu_fwd(*y[:2])
        assert all(torch.equal(p, q) for p, q in zip(got, (h, *decoder.swiglu_bwd(y[2], *y[:2], saved))))


@gpu
def test_strided_lengths_and_stream(dev):
    """lengths of any stride, with a given stream: its copy belongs to that stream too."""
    q, k, v, do = attention_inputs(3, 70, 2, 2, 64, BF16, dev)
    both = torch.tensor([[70, 1], [13, 2], [0, 3]], dtype=torch.int32, device=dev)
    want = decoder.attention(q, k, v, lengths=both[:, 0].contiguous())
    assert torch.equal(decoder.attention(q, k, v, lengths=both[:, 0]), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    out, saved = decoder.attention_fwd(q, k, v, lengths=both[:, 0], stream=side)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(out, want)


@gpu
def test_autograd_step_captured(dev):
    """A forward and backward pass of the differentiable forms in a graph, no eager graph of the leaves alive."""
    x, w, dh = swiglu_inputs(40, 64, 48, BF16, dev)
    want = decoder.swiglu_bwd(dh, x, w, decoder.swiglu_fwd(x, w)[1])
    a, b = x.clone().requires_grad_(), w.clone().requires_grad_()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        torch.autograd.grad(decoder.swiglu(a, b), (a, b), dh)
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = torch.autograd.grad(decoder.swiglu(a, b), (a, b), dh)
    for _ in range(3):
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(got, want))


@gpu
def test_streams(dev):
    """On a side stream, current or given, with work of the default stream in between."""
    x, ws, lengths, gr = block_inputs(dev)
    want = block_step(x, ws, lengths, gr)
    q, k, v, do = attention_inputs(2, 100, 4, 2, 64, BF16, dev)
    o, lse = decoder.attention_fwd(q, k, v)
    grads = decoder.attention_bwd(do, q, k, v, o, lse)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = block_step(x, ws, lengths, gr)
    o2, lse2 = decoder.attention_fwd(q, k, v, stream=side)
    grads2 = decoder.attention_bwd(do, q, k, v, o2, lse2, stream=side)
    s2 = decoder.add_norm_fwd(x, x, ws[0], stream=side)
    h2, kept = decoder.swiglu_fwd(x, ws[3], stream=side)
    d2 = decoder.swiglu_bwd(h2, x, ws[3], kept, stream=side)
    n2 = decoder.add_norm_bwd(x, x, x, x, ws[0], s2[2], stream=side)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(p, r) for p, r in zip(got, want))
    assert torch.equal(o, o2) and all(torch.equal(p, r) for p, r in zip(lse, lse2)) and all(torch.equal(p, r) for p, r in zip(grads, grads2))
    s3 = decoder.add_norm_fwd(x, x, ws[0])
    h3, kept3 = decoder.swiglu_fwd(x, ws[3])
    assert all(torch.equal(p, r) for p, r in zip(s2, s3)) and torch.equal(h2, h3)
    assert all(torch.equal(p, r) for p, r in zip(d2, decoder.swiglu_bwd(h3, x, ws[3], kept3)))
    assert all(torch.equal(p, r) for p, r in zip(n2, decoder.add_norm_bwd(x, x, x, x, ws[0], s3[2])) if p is not None)


@gpu
def test_train_load_on_own_operators(dev):
    """bench.py --load train --train-ops hip: the step runs, and its gradients are the torch model's."""
    import bench

    loads = []
    for ops in ("torch", "hip"):
        a = bench.parse_args(["--load", "train", "--train-ops", ops, "--train-dim", "256", "--train-layers", "2",
                              "--train-batch", "2", "--train-seq", "96", "--train-vocab", "512"])
        loads.append(bench.TrainLoad(a, 0, None))
    grads = []
    for ld in loads:
        logits = ld.model(ld.tok[:, :-1])
        ld.F.cross_entropy(logits.float().view(-1, ld.vocab), ld.tok[:, 1:].reshape(-1)).backward()
        grads.append({n: p.grad.double() for n, p in ld.model.named_parameters()})
    # The two differ by what either rounds: about 30 tensors on the longest way (two layers, there and
    # back), each half a step of bfloat16 in the mean square at most, on both sides.
    for n, g in grads[0].items():
        assert (grads[1][n] - g).norm() <= 2 * math.sqrt(30) * half_step(BF16) * g.norm(), n
    ld = loads[1]
    ld.opt.zero_grad(set_to_none=True)
    ld.step()
    assert all(torch.isfinite(p).all() for p in ld.model.parameters())
    assert ld.calibrate()["train_ops"] == "hip" and ld.op_flops > 0


# ----------------------------------------------------------------------------- refusals (CPU)

def z(*shape, t=BF16):
    return torch.zeros(*shape, dtype=t)


def kept(*shape, t=F32, low=torch.uint8):
    return z(*(shape or (1, 2, 4)), t=t), z(1, 4, 2, 64, t=low)


ATTENTION_REFUSED = [
    ("rank", lambda: decoder.attention(z(4, 2, 64), z(4, 2, 64), z(4, 2, 64)), ValueError),
    ("type", lambda: decoder.attention(*[z(1, 4, 2, 64, t=F32)] * 3), TypeError),
    ("mixed types", lambda: decoder.attention(z(1, 4, 2, 64), z(1, 4, 2, 64, t=F16), z(1, 4, 2, 64)), TypeError),
    ("head dimension", lambda: decoder.attention(*[z(1, 4, 2, 96)] * 3), ValueError),
    ("shared heads", lambda: decoder.attention(z(1, 4, 3, 64), z(1, 4, 2, 64), z(1, 4, 2, 64)), ValueError),
    ("no key heads", lambda: decoder.attention(z(1, 4, 3, 64), z(1, 4, 0, 64), z(1, 4, 0, 64)), ValueError),
    ("positions", lambda: decoder.attention(z(1, 4, 2, 64), z(1, 5, 2, 64), z(1, 5, 2, 64)), ValueError),
    ("v's heads", lambda: decoder.attention(z(1, 4, 2, 64), z(1, 4, 2, 64), z(1, 4, 1, 64)), ValueError),
    ("scale", lambda: decoder.attention(*[z(1, 4, 2, 64)] * 3, scale=0.0), ValueError),
    ("scale", lambda: decoder.attention(*[z(1, 4, 2, 64)] * 3, scale=math.nan), ValueError),
    ("scale", lambda: decoder.attention(*[z(1, 4, 2, 64)] * 3, scale=1e39), ValueError),
    ("scale", lambda: decoder.attention(*[z(1, 4, 2, 64)] * 3, scale=1e-46), ValueError),
    ("nothing kept", lambda: decoder.attention_bwd(*[z(1, 4, 2, 64)] * 5, (None, None)), TypeError),
    ("lengths type", lambda: decoder.attention(*[z(1, 4, 2, 64)] * 3, lengths=torch.tensor([4])), TypeError),
    ("lengths shape", lambda: decoder.attention(*[z(1, 4, 2, 64)] * 3, lengths=torch.tensor([4, 4], dtype=torch.int32)), ValueError),
    ("device", lambda: decoder.attention(*[z(1, 4, 2, 64)] * 3), ValueError),
    ("qkv rank", lambda: decoder.attention_qkv(z(1, 4, 6 * 64), 2), ValueError),
    ("qkv heads", lambda: decoder.attention_qkv(z(1, 4, 5, 64), 2), ValueError),
    ("qkv no heads", lambda: decoder.attention_qkv(z(1, 4, 4, 64), 0), ValueError),
    ("dout shape", lambda: decoder.attention_bwd(z(1, 4, 1, 64), *[z(1, 4, 2, 64)] * 4, kept()), ValueError),
    ("dout type", lambda: decoder.attention_bwd(z(1, 4, 2, 64, t=F16), *[z(1, 4, 2, 64)] * 4, kept()), TypeError),
    ("lse type", lambda: decoder.attention_bwd(*[z(1, 4, 2, 64)] * 5, kept(t=BF16)), ValueError),
    ("lse shape", lambda: decoder.attention_bwd(*[z(1, 4, 2, 64)] * 5, kept(1, 4, 2)), ValueError),
    ("low type", lambda: decoder.attention_bwd(*[z(1, 4, 2, 64)] * 5, kept(low=F16)), ValueError),
]
SWIGLU_REFUSED = [
    ("type", lambda: decoder.swiglu(z(4, 64, t=F32), z(16, 64, t=F32)), TypeError),
    ("mixed types", lambda: decoder.swiglu(z(4, 64), z(16, 64, t=F16)), TypeError),
    ("width", lambda: decoder.swiglu(z(4, 60), z(16, 60)), ValueError),
    ("inner", lambda: decoder.swiglu(z(4, 64), z(20, 64)), ValueError),
    ("odd rows of w", lambda: decoder.swiglu(z(4, 64), z(17, 64)), ValueError),
    ("w's width", lambda: decoder.swiglu(z(4, 64), z(16, 72)), ValueError),
    ("w's rank", lambda: decoder.swiglu(z(4, 64), z(2, 8, 64)), ValueError),
    ("no inner", lambda: decoder.swiglu(z(4, 64), z(0, 64)), ValueError),
    ("device", lambda: decoder.swiglu(z(4, 64), z(16, 64)), ValueError),
    ("dh shape", lambda: decoder.swiglu_bwd(z(4, 16), z(4, 64), z(16, 64), z(4, 16)), ValueError),
    ("saved shape", lambda: decoder.swiglu_bwd(z(4, 8), z(4, 64), z(16, 64), z(4, 24, t=torch.uint8)), ValueError),
    ("saved type", lambda: decoder.swiglu_bwd(z(4, 8), z(4, 64), z(16, 64), z(4, 48)), ValueError),
]
NORM_REFUSED = [
    ("type", lambda: decoder.add_norm(*[z(4, 64, t=torch.float64)] * 2, z(64, t=torch.float64)), TypeError),
    ("mixed types", lambda: decoder.add_norm(z(4, 64), z(4, 64), z(64, t=F32)), TypeError),
    ("shape", lambda: decoder.add_norm(z(4, 64), z(3, 64), z(64)), ValueError),
    ("weight", lambda: decoder.add_norm(z(4, 64), z(4, 64), z(4, 64)), ValueError),
    ("gate", lambda: decoder.add_norm(z(4, 64), z(4, 64), z(64), gate=z(4, 64)), ValueError),
    ("post_weight", lambda: decoder.add_norm(z(4, 64), z(4, 64), z(64), post_weight=z(1)), ValueError),
    ("width", lambda: decoder.add_norm(z(1, 16385), z(1, 16385), z(16385)), ValueError),
    ("no width", lambda: decoder.add_norm(z(1, 0), z(1, 0), z(0)), ValueError),
    ("eps", lambda: decoder.add_norm(z(4, 64), z(4, 64), z(64), eps=-1.0), ValueError),
    ("scale", lambda: decoder.add_norm(z(4, 64), z(4, 64), z(64), scale=math.inf), ValueError),
    ("scale", lambda: decoder.add_norm(z(4, 64), z(4, 64), z(64), scale=-1e39), ValueError),
    ("eps", lambda: decoder.add_norm(z(4, 64), z(4, 64), z(64), eps=1e39), ValueError),
    ("nothing kept", lambda: decoder.add_norm_bwd(z(4, 64), None, z(4, 64), z(4, 64), z(64), None), TypeError),
    ("device", lambda: decoder.add_norm(z(4, 64), z(4, 64), z(64)), ValueError),
    ("no gradient", lambda: decoder.add_norm_bwd(None, None, z(4, 64), z(4, 64), z(64), z(2, 4, t=F32)), ValueError),
    ("saved", lambda: decoder.add_norm_bwd(z(4, 64), None, z(4, 64), z(4, 64), z(64), z(4, 2, t=F32)), ValueError),
]


@pytest.mark.parametrize("name,call,error", [pytest.param(n, c, e, id=f"{op} {n}") for op, cases in
                                        (("attention", ATTENTION_REFUSED), ("swiglu", SWIGLU_REFUSED), ("add_norm", NORM_REFUSED))
                                        for n, c, e in cases])
def test_refusals(name, call, error):
    with pytest.raises(error) as raised:
        call()
    # (where the tensors are is looked at last)
    assert ("must be on a GPU" in str(raised.value)) == (name == "device")


def test_plans_cover_their_ranges():
    """Splits leave every part work; the column sums come in a sensible number of parts."""
    for M in (1, 5, 128, 1000, 9000):
        for N in (8, 256, 5000, 30000):
            for K in (8, 512, 4096, 30000):
                for forward in (False, True):
                    tile, splits = decoder._product_plan(M, N, K, forward)
                    assert tile in decoder.PRODUCT_TILES[:3 if forward and M <= 32 else 2]
                    assert 1 <= splits <= max(1, K // 128)
    for T in (1, 3, 5, 100, 5000, 1 << 20):
        for C in (1, 512, 513, 4096, 4097, 16384):
            assert 1 <= decoder._norm_parts(T, C) <= 65536
    for S in (1, 128, 5000, 100000):
        assert 1 <= decoder._dkv_splits(1, S, 8, 1, True) <= 16


def test_structures_match_the_header():
    """The packed argument blocks have the C structures' sizes."""
    import os
    import shutil
    import subprocess
    import tempfile

    if not shutil.which("g++"):
        pytest.skip("no host compiler")
    here = os.path.dirname(os.path.abspath(decoder.__file__))
    with tempfile.TemporaryDirectory() as d:
        src = os.path.join(d, "s.cpp")
        with open(src, "w") as f:
            f.write('#include <cstddef>\n#include <cstdio>\n#include "decoder.h"\nint main() { std::printf("%zu %zu %zu %zu %zu %zu", '
                    "offsetof(KgsAttention, scale) + 4, offsetof(KgsSwiglu, splits) + 12, offsetof(KgsAddNorm, eps) + 4, "
                    "offsetof(KgsAttention, B), offsetof(KgsSwiglu, T), offsetof(KgsAddNorm, rows)); }\n")
        subprocess.run(["g++", "-I", os.path.join(here, "hip"), src, "-o", os.path.join(d, "s")], check=True)
        got = [int(x) for x in subprocess.run([os.path.join(d, "s")], check=True, capture_output=True, text=True).stdout.split()]
    assert got[:3] == [decoder._ATTENTION.size, decoder._SWIGLU.size, decoder._ADD_NORM.size]
    assert got[3:] == [(13 + 24) * 8, (9 + 3) * 8, (16 + 5) * 8]
