"""Calls of the decoder block's operators (ops/decoder.py) at the edges of what they document: values that
change when they are rounded to 32 bits, ranges of the 16-bit types, limits of a launch, streams.

Oracles and tolerances as in test_decoder_ops.py, whose bounds are per element and worked out beforehand.
"""
import gc
import math

import pytest
import test_decoder_ops
import torch

from kube_gpu_stats_amd.ops import decoder
from test_decoder_ops import (BF16, F16, F32, NORM_GRADS, attention_inputs, close, half_step, mm, norm_check, norm_inputs,
                              norm_oracle, z)

gpu = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "GPU tests need a GPU"
    yield torch.device("cuda", 0)
    gc.collect()
    torch.cuda.empty_cache()  # other modules measure the GPU's memory


@pytest.fixture
def launches(monkeypatch):
    """The entries that calls on CPU tensors would launch, with their argument blocks."""
    seen = []
    monkeypatch.setattr(decoder, "_on_gpu", lambda t, name: None)
    monkeypatch.setattr(decoder, "_here", lambda t, stream: True)
    monkeypatch.setattr(decoder, "_call", lambda entry, args, index: seen.append((entry, args)))
    return seen


# ------------------------------------------------------- add_norm: scales that are one in 32 bits

NEAR_ONE = [0.7 + 0.2 + 0.1, 1 + 1e-9, 1 - 2.0 ** -25, 1 + 2.0 ** -24]  # the last two: ties, rounded to even
NEXT_TO_ONE = [1 - 2.0 ** -24, 1 + 2.0 ** -23]


@pytest.mark.parametrize("scale", NEAR_ONE + NEXT_TO_ONE)
def test_scale_is_rounded_before_it_decides(launches, scale):
    """dbranch is a tensor of its own exactly where the kernels, which get 32 bits, write one."""
    x, w = z(4, 64), z(64)
    _, _, saved = decoder.add_norm_fwd(x, x, w, scale=scale)
    dr, db, *_ = decoder.add_norm_bwd(x, x, x, x, w, saved, scale=scale)
    entry, args = launches[-1]
    packed = decoder._ADD_NORM.unpack(args)
    assert entry == "kgs_add_norm_bwd"
    assert (packed[-2] == 1.0) == (scale in NEAR_ONE)
    assert (dr is db) == (packed[-2] == 1.0)


@gpu
@pytest.mark.parametrize("t", [BF16, F32])
@pytest.mark.parametrize("scale", NEAR_ONE + NEXT_TO_ONE)
def test_gradients_of_scales_next_to_one(dev, scale, t):
    a = norm_inputs(9, 200, t, dev, False, False, seed=3)
    want = norm_check(*a, scale=scale)[3]
    r, b = a[0].clone().requires_grad_(), a[1].clone().requires_grad_()
    torch.autograd.backward(decoder.add_norm(r, b, a[2], scale=scale, eps=1e-5), [a[5], a[6]])
    assert torch.equal(r.grad, want[0]) and torch.equal(b.grad, want[1])


# ------------------------------------------------- add_norm: a backward that starts from the stream

def stream_tolerance(ref, tol, a, scale, eps):
    """tol, and what the stream's own error adds to the gradients: half of a 256th of its last place, twice (cut
    and middle), where 16 bits and 8 are kept; below fp16's normal range what 16 bits leave."""
    r, b, w, pw, gate, dS, dy = (None if x is None else x.double() for x in a)
    t, u, C = a[0].dtype, torch.finfo(a[0].dtype).eps / 2, a[0].shape[1]
    if t == F32:
        return tol  # the stream as it was computed
    tol = dict(tol)
    s = ref["stream"]
    e_s = 2.0 ** -7 * u * s.abs() + (2.0 ** -25 if t == F16 else 0.0)
    rs = (s.square().mean(1, keepdim=True) + eps).rsqrt()
    sh, e_sh = s * rs, e_s * rs
    d = w * dy
    m = (d * sh).mean(1, keepdim=True)
    e_ds = 1.02 * rs * (e_sh * m.abs() + sh.abs() * (d.abs() * e_sh).mean(1, keepdim=True))
    tol["dresidual"] = tol["dresidual"] + e_ds
    tol["dweight"] = tol["dweight"] + (dy.abs() * e_sh).sum(0)
    rb = (b.square().mean(1, keepdim=True) + eps).rsqrt() if pw is not None else torch.ones_like(rs)
    one = torch.ones(C, dtype=torch.float64, device=s.device)
    p, g = one if pw is None else pw, one if gate is None else gate
    e_x = abs(scale) * (p * g).abs() * e_ds
    tol["dbranch"] = tol["dbranch"] + 1.02 * rb * e_x
    if pw is not None:
        tol["dbranch"] = tol["dbranch"] + 1.02 * rb * (b * rb).abs() * ((b * rb).abs() * e_x).mean(1, keepdim=True)
        tol["dpost_weight"] = tol["dpost_weight"] + abs(scale) * ((b * rb * g).abs() * e_ds).sum(0)
    if gate is not None:
        tol["dgate"] = tol["dgate"] + abs(scale) * ((b * rb * p).abs() * e_ds).sum(0)
    return tol


def stream_check(a, scale=1.0, eps=1e-5):
    r, b, w, pw, gate, dS, dy = a
    kw = {"post_weight": pw, "gate": gate, "scale": scale, "eps": eps}
    s, y, saved = decoder.add_norm_fwd(r, b, w, **kw)
    grads = decoder.add_norm_bwd(dS, dy, s, b, w, saved, **kw)
    flat = lambda x: None if x is None else x.reshape(-1, x.shape[-1])  # noqa: E731
    f = [flat(x) if x is not None and x.dim() > 1 else x for x in a]
    ref, tol = norm_oracle(*f[:5], scale, eps, *f[5:])
    tol = stream_tolerance(ref, tol, f, scale, eps)
    for n, got in (("stream", s), ("out", y), *zip(NORM_GRADS, grads)):
        if n not in ref:
            assert got is None
            continue
        close(got.reshape(ref[n].shape), ref[n], tol[n], n)
    assert (grads[0] is grads[1]) == (pw is None and gate is None and scale == 1.0)
    return kw, s, y, saved, grads


@gpu
@pytest.mark.parametrize("t", [BF16, F16, F32])
@pytest.mark.parametrize("C", [1, 7, 8, 300, 512, 513, 2056, 8192, 8200, 12296, 16384])
@pytest.mark.parametrize("post,gate,scale", [(False, False, 1.0), (True, True, 0.7), (False, False, -0.5), (False, True, 1.0)])
def test_add_norm_gradients_from_the_stream(dev, C, t, post, gate, scale):
    """The residual's place taken by the stream that the forward pass returned: the same gradients."""
    for T in (1, 37):
        stream_check(norm_inputs(T, C, t, dev, post, gate, seed=C + T), scale)


@gpu
@pytest.mark.parametrize("t,T,C", [(BF16, 3000, 2048), (F16, 2100, 72), (F32, 9000, 16), (BF16, 1501, 8193)])
def test_add_norm_many_rows_from_the_stream(dev, t, T, C):
    stream_check(norm_inputs(T, C, t, dev, True, True, seed=T), 0.3)
    stream_check(norm_inputs(T, C, t, dev, False, False, seed=T))


@gpu
@pytest.mark.parametrize("t", [BF16, F32])
def test_stream_and_residual_are_told_apart(dev, t):
    """By their memory: views of the stream count, a program's own buffer with everything in it does not."""
    a = norm_inputs(12, 200, t, dev, True, False, seed=5)
    r, b, w, pw, _, dS, dy = a
    kw, s, y, saved, want = stream_check(a, 0.5)
    shaped = [x.view(3, 4, 200) for x in (dS, dy, s, b)]
    for x, q in zip(decoder.add_norm_bwd(*shaped, w, saved, **kw), want):
        assert x is q is None or torch.equal(x.reshape(q.shape), q)
    with pytest.raises(ValueError):
        decoder.add_norm_bwd(*(x.view(3, 4, 200).transpose(0, 1) for x in (dS, dy, s, b)), w, saved, **kw)
    plain = decoder.add_norm_bwd(dS, dy, r, b, w, saved, **kw)
    room = torch.zeros(1 << 16, dtype=torch.uint8, device=dev)
    size = r.numel() * r.element_size()
    r2 = room[:size].view(t).view(r.shape).copy_(r)
    at = -(-size // 16) * 16
    k2 = room[at:at + 96].view(F32).view(2, 12).copy_(saved)
    for x, q in zip(decoder.add_norm_bwd(dS, dy, r2, b, w, k2, **kw), plain):
        assert x is q is None or torch.equal(x, q)
    # a stream changed in place does not count as a change of saved, nor a pass's results as views
    v = saved._version
    s.add_(1)
    assert saved._version == v and s._base is None and saved._base is None


@gpu
def test_add_norm_pair_from_the_stream_captured(dev):
    """In a graph, replayed with other inputs between eager calls; on another stream."""
    a = norm_inputs(33, 520, BF16, dev, True, True, seed=1)

    def step(r, b, w, pw, gate, dS, dy, **on):
        kw = {"post_weight": pw, "gate": gate, "scale": 0.5}
        s, y, saved = decoder.add_norm_fwd(r, b, w, **kw, **on)
        return (s, y, *decoder.add_norm_bwd(dS, dy, s, b, w, saved, **kw, **on))

    step(*a)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = step(*a)
    for seed in (2, 3, 4):
        fresh = norm_inputs(33, 520, BF16, dev, True, True, seed=seed)
        want = step(*fresh)
        for x, q in zip(a, fresh):
            x.copy_(q)
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, q) for x, q in zip(got, want)), seed
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    other = step(*a, stream=side)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(x, q) for x, q in zip(other, want))


@gpu
def test_a_stream_that_overflowed_stays_infinite(dev):
    """fp16 rows whose sum leaves the type's range: the gradients of those rows are not finite, the others are right."""
    a = norm_inputs(4, 64, F16, dev, False, False, seed=7)
    r, b, w, _, _, dS, dy = a
    want = norm_check(*a)[3]
    r[2, 5] = b[2, 5] = 60000.0
    s, y, saved = decoder.add_norm_fwd(r, b, w, eps=1e-5)
    dr = decoder.add_norm_bwd(dS, dy, s, b, w, saved, eps=1e-5)[0]
    assert math.isinf(s[2, 5]) and not torch.isfinite(dr[2]).all()
    for i in (0, 1, 3):
        assert (dr[i].double() - want[0][i].double()).abs().max() <= 2 * torch.finfo(F16).eps * want[0][i].abs().max()


# ----------------------------------------------------------- the training step's two models are one

def train_loads(device, *more):
    import bench

    loads = []
    for ops in ("torch", "hip"):
        a = bench.parse_args(["--load", "train", "--train-ops", ops, "--train-dim", "256", "--train-layers", "2",
                              "--train-batch", "2", "--train-seq", "96", "--train-vocab", "512", *more])
        loads.append(bench.TrainLoad(a, device, None))
    for ld in loads:  # small activations, at which the norms' eps counts
        with torch.no_grad():
            ld.model.emb.weight.mul_(0.01)
    return loads


def same_gradients(loads):
    grads = []
    for ld in loads:
        logits = ld.model(ld.tok[:, :-1])
        ld.F.cross_entropy(logits.float().view(-1, ld.vocab), ld.tok[:, 1:].reshape(-1)).backward()
        grads.append({n: p.grad.double() for n, p in ld.model.named_parameters()})
    # as many roundings, and as large ones, as in test_decoder_ops.py's test of the same models
    for n, g in grads[0].items():
        assert (grads[1][n] - g).norm() <= 2 * math.sqrt(30) * half_step(BF16) * g.norm(), n


def test_train_models_agree_on_small_activations(monkeypatch):
    """With the operators in torch's own words, on the CPU: what the two models pass to them is the same."""
    import torch.nn.functional as TF

    def attention_qkv(qkv, heads):
        q, k, v = (x.transpose(1, 2) for x in qkv.split(heads, dim=2))
        return TF.scaled_dot_product_attention(q, k, v, is_causal=True).transpose(1, 2)

    def add_norm(r, b, w, *, eps):
        return r + b, TF.rms_norm(r + b, w.shape, w, eps)

    def swiglu(x, w):
        g, u = TF.linear(x, w).chunk(2, -1)
        return TF.silu(g) * u

    for f in (attention_qkv, add_norm, swiglu):
        monkeypatch.setattr(decoder, f.__name__, f)
    same_gradients(train_loads(-1))


@gpu
def test_train_models_agree_on_small_activations_on_gpu(dev):
    same_gradients(train_loads(0))


# -------------------------------------------------------- attention in fp16: ranges of ds

def fp16_oracle(monkeypatch, q, k, v, do, causal, scale):
    """attention_oracle without what it allows for fp16's lack of range, and in its place: results round to
    multiples of 2^-24 at the least; ds is rounded times a power of two that brings a bound of |do.v - delta|,
    2.02 |do| |v| of the largest norms, over 2^14, so to multiples of 2^-38 of that bound at the least;
    probabilities times 2^6 forward (over a sum of at least as much) and 2^12 backward."""
    with monkeypatch.context() as m:
        m.setattr(test_decoder_ops, "F16", None)
        ref, tol, _ = test_decoder_ops.attention_oracle(q, k, v, do, causal, scale, [q.shape[1]] * q.shape[0])
    n, G = q.shape[1], q.shape[2] // k.shape[2]
    size = [x.double().abs().max() for x in (q, k, v, do)]
    most = 2.02 * q.shape[3] * size[3] * size[2]  # a norm is at most the largest element by the root of D
    tol["out"] += 2.0 ** -31 * n * size[2]
    tol["dv"] += 2.0 ** -37 * n * G * size[3]
    tol["dq"] += 2.0 ** -39 * scale * n * most * size[1]
    tol["dk"] += 2.0 ** -39 * scale * n * G * most * size[0]
    for x in tol.values():
        x += 2.0 ** -25
    return ref, tol


def fp16_check(monkeypatch, q, k, v, do, causal, names=("out", "dq", "dk", "dv")):
    scale = q.shape[3] ** -0.5
    out, saved = decoder.attention_fwd(q, k, v, causal=causal)
    got = dict(zip(("out", "dq", "dk", "dv"), (out, *decoder.attention_bwd(do, q, k, v, out, saved, causal=causal))))
    ref, tol = fp16_oracle(monkeypatch, q, k, v, do, causal, scale)
    for n in names:
        # a result from 65520 on, half a step past fp16's largest, rounds to infinity
        over = ref[n].abs() - tol[n] >= 65520
        assert torch.isinf(got[n][over]).all(), n
        near = ref[n].abs() + tol[n] >= 65520
        close(torch.where(near, torch.zeros_like(got[n]), got[n]), torch.where(near, torch.zeros_like(ref[n]), ref[n]), tol[n], n)


@gpu
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("B,S,H,Hk,D", [(1, 200, 2, 2, 128), (2, 61, 2, 1, 64), (1, 33, 1, 1, 64), (1, 1100, 4, 1, 128)])
@pytest.mark.parametrize("e,a", [(-20, 10), (-20, -10), (-14, 5), (-8, 0), (0, 0), (8, 0)])
def test_fp16_gradients_of_small_and_large_dout(dev, monkeypatch, e, a, B, S, H, Hk, D, causal):
    """dout of 2^e, keys of 2^a and queries of 2^-a: dq (or dk) lies well inside fp16's range, ds far below it."""
    q, k, v, do = (x.float() for x in attention_inputs(B, S, H, Hk, D, F32, dev, seed=S))
    fp16_check(monkeypatch, *(x.to(F16) for x in (q * 2.0 ** -a, k * 2.0 ** a, v, do * 2.0 ** e)), causal)


@gpu
@pytest.mark.parametrize("D", [64, 128])
def test_fp16_gradients_of_large_products(dev, monkeypatch, D):
    """do.v of over 2^20, ds of over fp16's largest, gradients of a few hundreds; rows that grow, and that shrink."""
    q, k, v, do = attention_inputs(1, 300, 2, 1, D, F32, dev, seed=D)
    q, k, v, do = q * 2.0 ** -8, k * 2.0 ** -8, v * 2.0 ** 6, do * 2.0 ** 12
    for causal in (True, False):
        fp16_check(monkeypatch, *(x.to(F16) for x in (q, k, v, do)), causal, ("out", "dq", "dk"))
        for way in (1, -1):  # rows and keys of very different sizes, in rising and falling order
            grow = 2.0 ** (torch.linspace(-12, 0, 300, device=dev) * way + min(0, way) * 12).view(1, 300, 1, 1)
            fp16_check(monkeypatch, *(x.to(F16) for x in (q, k, v * grow, do * grow)), causal, ("out", "dq", "dk"))


@gpu
def test_fp16_gradients_of_zero_rows(dev, monkeypatch):
    """Rows whose dout is zero, at the start, between others and all of them."""
    q, k, v, do = attention_inputs(1, 150, 2, 2, 64, F32, dev, seed=2)
    do = do * 2.0 ** -16
    do[:, :40] = 0
    do[:, 70] = 0
    for causal in (True, False):
        fp16_check(monkeypatch, *(x.to(F16) for x in (q, k * 64, v, do)), causal)
        h = [x.to(F16) for x in (q, k, v)]
        out, saved = decoder.attention_fwd(*h, causal=causal)
        assert not any(x.any() for x in decoder.attention_bwd(torch.zeros_like(out), *h, out, saved, causal=causal))


# -------------------------------------------- attention in fp16: probabilities far below one

@gpu
@pytest.mark.parametrize("gap", [16, 22, 26, 30])
@pytest.mark.parametrize("D", [64, 128])
def test_fp16_probabilities_far_below_one(dev, monkeypatch, gap, D):
    """One key has all but 2^-gap of every row's probability, and nothing in v: what the others add is the result,
    and their dv is a sum of such probabilities times large gradients."""
    S, H = 260, 2
    q, k, v, do = attention_inputs(1, S, H, 1, D, F32, dev, seed=gap)
    q, k = q * 0.01, k * 0.01
    q[..., 0], k[..., 0] = 8.0, 0.0
    k[:, 0, :, 0] = gap * math.log(2) * D ** 0.5 / 8
    v = v.abs() * 512
    v[:, 0] = 0
    fp16_check(monkeypatch, *(x.to(F16) for x in (q, k, v, do * 1024)), True, ("out", "dv"))
    fp16_check(monkeypatch, *(x.to(F16) for x in (q, k, v, do * 1024)), False, ("out", "dv"))


# ----------------------------------------------------------------- argument blocks (CPU)

def test_argument_blocks_are_whole_structures(tmp_path):
    """The library copies each structure whole, with what pads it: so much has to be there to be read."""
    import os
    import shutil
    import subprocess

    if not shutil.which("g++"):
        pytest.skip("no host compiler")
    here = os.path.join(os.path.dirname(os.path.abspath(decoder.__file__)), "hip")
    (tmp_path / "s.cpp").write_text('#include <cstdio>\n#include "decoder.h"\nint main() { std::printf("%zu %zu %zu", '
                                    "sizeof(KgsAttention), sizeof(KgsSwiglu), sizeof(KgsAddNorm)); }\n")
    subprocess.run(["g++", "-I", here, str(tmp_path / "s.cpp"), "-o", str(tmp_path / "s")], check=True)
    got = subprocess.run([str(tmp_path / "s")], check=True, capture_output=True, text=True).stdout.split()
    assert [int(x) for x in got] == [decoder._ATTENTION.size, decoder._SWIGLU.size, decoder._ADD_NORM.size]


# ----------------------------------------------------------------- limits of a launch

def big(*shape, t=BF16):
    return torch.zeros(1, dtype=t).expand(*shape)


TOO_LARGE = [
    ("attention pieces", lambda: decoder.attention(*[big(1 << 20, 1, 16, 64)] * 3)),
    ("attention pieces of long rows", lambda: decoder.attention(*[big(1, (1 << 30) - 1, 3, 128)] * 3)),
    ("attention pieces back", lambda: decoder.attention_bwd(*[big(1 << 20, 1, 16, 64)] * 5,
                                                            (big(1 << 20, 16, 1, t=F32), big(1 << 20, 1, 16, 64, t=torch.uint8)))),
    ("attention heads", lambda: decoder.attention(*[big(1, 4, (1 << 16) + 1, 64)] * 3)),
    ("attention heads on few", lambda: decoder.attention(big(1, 4, 1 << 16, 128), *[big(1, 4, 1, 128)] * 2)),
    ("qkv heads", lambda: decoder.attention_qkv(big(1, 4, 3 << 15, 64), 1 << 15)),
    ("swiglu rows and inner", lambda: decoder.swiglu(big((1 << 30) - 1, 8), big(1 << 10, 8))),
    ("swiglu weights", lambda: decoder.swiglu(big(4, 1 << 20), big(1 << 21, 1 << 20))),
]


@pytest.mark.parametrize("call", [pytest.param(c, id=n) for n, c in TOO_LARGE])
def test_what_no_launch_holds_is_refused(call, monkeypatch):
    """With a ValueError, before anything is launched."""
    monkeypatch.setattr(decoder, "_kept", lambda *a: None)  # (expanded tensors are not contiguous)
    with pytest.raises(ValueError) as raised:
        call()
    assert "must be on a GPU" not in str(raised.value)


def test_every_product_that_is_not_refused_has_a_plan():
    # (the most: 2^23 - 8 tiles of 256 x 256)
    for M, N, K in ((1 << 20, 1 << 18, 8), (1 << 30, 128, 8), (1 << 19, 1 << 19, 1 << 20), (1 << 21, 8, 1 << 30), (1 << 29, 512, 64)):
        for forward in (False, True):
            tile, splits = decoder._product_plan(M, N, K, forward)
            rows, columns, threads = ((128, 128, 256), (256, 256, 512))[tile]
            assert (-(-M // rows) * -(-N // columns) * splits + 7) * threads < 1 << 32


@gpu
@pytest.mark.parametrize("B,S,H", [(65536, 1, 16), (40000, 3, 32), (1 << 19, 1, 16)])
def test_attention_of_many_short_sequences(dev, B, S, H):
    """Over a million heads of one piece each."""
    g = torch.Generator(device=dev).manual_seed(B)
    q, k, v, do = (torch.randn(B, S, H, 64, generator=g, device=dev).to(BF16) for _ in range(4))
    out, saved = decoder.attention_fwd(q, k, v)
    grads = decoder.attention_bwd(do, q, k, v, out, saved)
    assert torch.equal(out[:, 0], v[:, 0])  # the first position sees itself
    for b in (0, 1, B // 2 + 1, B - 1):
        one = [x[b:b + 1].contiguous() for x in (q, k, v, do)]
        o, keep = decoder.attention_fwd(*one[:3])
        for x, y in zip((out, *grads), (o, *decoder.attention_bwd(one[3], *one[:3], o, keep))):
            assert torch.equal(x[b:b + 1], y)
    lengths = torch.arange(B, device=dev, dtype=torch.int32) % (S + 1)
    padded = decoder.attention(q, k, v, lengths=lengths)
    for s in range(S):
        live = (lengths > s)[:, None, None]
        assert torch.equal(padded[:, s], torch.where(live, out[:, s], torch.zeros_like(out[:, s])))


# ----------------------------------------------------------------- forward-mode derivatives (CPU)

@pytest.mark.parametrize("call", [
    pytest.param(lambda dual: decoder.attention(z(1, 4, 2, 64), dual(1, 4, 2, 64), z(1, 4, 2, 64)), id="attention"),
    pytest.param(lambda dual: decoder.attention_qkv(dual(1, 4, 4, 64), 2), id="attention_qkv"),
    pytest.param(lambda dual: decoder.attention_fwd(dual(1, 4, 2, 64), z(1, 4, 2, 64), z(1, 4, 2, 64)), id="attention_fwd"),
    pytest.param(lambda dual: decoder.attention_bwd(dual(1, 4, 2, 64), *[z(1, 4, 2, 64)] * 4, test_decoder_ops.kept()), id="attention_bwd"),
    pytest.param(lambda dual: decoder.swiglu(z(4, 64), dual(16, 64)), id="swiglu"),
    pytest.param(lambda dual: decoder.swiglu_bwd(dual(4, 8), z(4, 64), z(16, 64), z(4, 48, t=torch.uint8)), id="swiglu_bwd"),
    pytest.param(lambda dual: decoder.add_norm_bwd(None, dual(4, 64), z(4, 64), z(4, 64), z(64), z(2, 4, t=F32)), id="add_norm_bwd"),
    pytest.param(lambda dual: decoder.swiglu_fwd(dual(4, 64), z(16, 64)), id="swiglu_fwd"),
    pytest.param(lambda dual: decoder.add_norm(z(4, 64), z(4, 64), z(64), gate=dual(64)), id="add_norm"),
    pytest.param(lambda dual: decoder.add_norm_fwd(z(4, 64), dual(4, 64), z(64)), id="add_norm_fwd"),
])
@pytest.mark.parametrize("grad", [True, False])
def test_forward_mode_tangents_are_refused(call, grad):
    """They were dropped without a word."""
    import torch.autograd.forward_ad as fw

    with torch.set_grad_enabled(grad), fw.dual_level():
        with pytest.raises(TypeError, match="forward-mode"):
            call(lambda *shape: fw.make_dual(z(*shape), z(*shape)))
        with pytest.raises(ValueError, match="must be on a GPU"):  # no tangent among the arguments: as ever
            decoder.swiglu(z(4, 64), z(16, 64))


# ----------------------------------------------------------------- scores of minus infinity

@gpu
@pytest.mark.parametrize("t", [BF16, F16])
@pytest.mark.parametrize("first", [1, 32, 64, 130, 200])
@pytest.mark.parametrize("causal", [True, False])
def test_keys_of_minus_infinity(dev, causal, first, t):
    """Keys whose scores are -inf take no part, also where a row sees no others at first, or none at all."""
    S, H, D = 200, 2, 64
    q, k, v, _ = attention_inputs(1, S, H, 1, D, t, dev, seed=first)
    q = q.abs()
    k[:, :first] = -math.inf
    out = decoder.attention(q, k, v, causal=causal)
    assert torch.equal(decoder.attention_fwd(q, k, v, causal=causal)[0], out)
    u = half_step(t)
    for h in range(H):
        s = mm(q[0, :, h].double(), k[0, first:, 0].double().t()) * D ** -0.5
        if causal:
            s = s.masked_fill(torch.arange(first, S, device=dev)[None] > torch.arange(S, device=dev)[:, None], -math.inf)
        p = torch.softmax(s, 1).nan_to_num(0.0)
        V = v[0, first:, 0].double()
        # roundings of p and of the result; 32-bit scores, sums and powers: 2^-14 of p covers 200 terms of 2^-24
        close(out[0, :, h], mm(p, V), u * mm(p, V).abs() + (1.01 * u + 2.0 ** -14) * mm(p, V.abs()), "out")


# ----------------------------------------------------------------- results of a given stream

@gpu
def test_results_of_a_given_stream_outlive_their_use_on_the_current_one(dev):
    """Memory of a result that is dropped while the current stream still reads it is not handed out again."""
    q = torch.randn(1, 512, 8, 64, device=dev).to(BF16)
    x, w = torch.randn(512, 520, device=dev).to(BF16), torch.randn(520, device=dev).to(BF16)
    wg = torch.randn(1024, 520, device=dev).to(BF16)
    out, saved = decoder.attention_fwd(q, q, q)
    _, kept = decoder.swiglu_fwd(x, wg)
    s, _, rstd = decoder.add_norm_fwd(x, x, w)
    h = torch.randn(512, 512, device=dev).to(BF16)
    side = torch.cuda.Stream()
    for call in (lambda: decoder.attention_fwd(q, q, q, stream=side), lambda: decoder.attention_bwd(out, q, q, q, out, saved, stream=side),
                 lambda: decoder.swiglu_fwd(x, wg, stream=side), lambda: decoder.swiglu_bwd(h, x, wg, kept, stream=side),
                 lambda: decoder.add_norm_fwd(x, x, w, stream=side), lambda: decoder.add_norm_bwd(x, x, s, x, w, rstd, gate=w, stream=side)):
        torch.cuda.synchronize()
        torch.cuda.empty_cache()
        side.wait_stream(torch.cuda.current_stream())
        flat = []
        for r in call():
            flat.extend(r if isinstance(r, tuple) else [r])
        flat = [r for r in flat if r is not None]
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda._sleep(100_000_000)  # the current stream is about to read them
        used = [r.clone() for r in flat]
        was = {r.untyped_storage().data_ptr(): r.untyped_storage().nbytes() for r in flat}
        side.synchronize()
        del flat, r
        with torch.cuda.stream(side):
            again = {torch.empty(n, dtype=torch.uint8, device=dev).data_ptr(): n for n in list(was.values()) * 2}
        assert not torch.cuda.current_stream().query(), "the use is over: nothing was shown"
        assert not was.keys() & again.keys()
        torch.cuda.synchronize()
        del used


# ----------------------------------------------------------------- what the matrix units are given (CPU)

def attention_products(S, D):
    """Products of 32 x 32 x D of one head's causal forward and backward, by walking as the kernels do."""
    forward = back = 0
    for q0 in range(0, S, 128):
        for qw in range(q0, q0 + 128, 32):
            last = min(qw + 32, S)
            for s0 in range(0, min(S, q0 + 128), 64):
                if s0 >= last:
                    continue
                forward += 4  # scores and values of two halves of 32 keys
                back += 4 if last <= 64 else 0  # the exact delta of a row's only step
                back += 3 * (1 + (s0 + 32 < last))
        for kw in range(q0, q0 + 128, 32):
            for s0 in range(q0, S, 32):
                back += 4 * (s0 + 32 > kw)
    return forward * 2 * 32 * 32 * D, back * 2 * 32 * 32 * D


@pytest.mark.parametrize("S", [1, 31, 64, 65, 100, 128, 200, 640, 1021])
def test_attention_matrix_flops(S):
    for D in (64, 128):
        forward, back = attention_products(S, D)
        assert decoder.attention_matrix_flops(3, S, 4, D) == (12 * forward, 12 * back)
    assert decoder.attention_matrix_flops(1, 0, 4, 64) == (0, 0)


def test_swiglu_matrix_flops():
    for T, K, F in ((8192, 4096, 11008), (5, 4096, 11008), (1777, 1000, 2680), (1, 8, 8)):
        up = lambda x, n: -(-x // n) * n  # noqa: E731
        want = []
        for M, N, sum_, forward in ((T, 2 * F, K, True), (T, K, 2 * F, False), (2 * F, K, T, False)):
            rows, columns = ((128, 128), (256, 256), (32, 256))[decoder._product_plan(M, N, sum_, forward)[0]]
            n = 2 * up(F, columns // 2) if forward else up(N, columns)
            want.append(2 * up(M, rows) * n * up(sum_, 64))
        assert decoder.swiglu_matrix_flops(T, K, F) == (want[0], want[1] + want[2])
    assert decoder.swiglu_matrix_flops(0, 64, 64) == (0, 0)


def test_train_load_reports_both_counts():
    import bench

    a = bench.parse_args(["--load", "train", "--train-ops", "hip", "--train-dim", "256", "--train-layers", "3",
                          "--train-batch", "2", "--train-seq", "96", "--train-vocab", "512"])
    ld = bench.TrainLoad(a, -1, None)
    tokens, ff = 2 * 96, 768
    assert ld.op_flops == 3 * (14.0 * 2 * 96 * 97 / 2 * 256 + 12.0 * tokens * 256 * ff)
    assert ld.matrix_flops == 3 * (sum(decoder.attention_matrix_flops(2, 96, 2, 128)) + sum(decoder.swiglu_matrix_flops(tokens, 256, ff)))
    assert ld.matrix_flops > ld.op_flops


@gpu
def test_fp16_attention_captured(dev):
    """Forward and backward in a graph, with all launches that fp16 takes, a split walk among them."""
    def inputs(seed):
        return attention_inputs(1, 900, 8, 1, 64, F16, dev, seed=seed)

    def step(q, k, v, do):
        out, saved = decoder.attention_fwd(q, k, v)
        return (out, *decoder.attention_bwd(do, q, k, v, out, saved))

    a = inputs(1)
    step(*a)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            got = step(*a)
        graphs.append((g, got))
    for seed in (2, 3, 4):
        for x, y in zip(a, inputs(seed)):
            x.copy_(y * 2.0 ** -seed)
        want = step(*a)
        for g, _ in graphs:
            g.replay()
        torch.cuda.synchronize()
        for _, got in graphs:
            assert all(torch.equal(x, y) for x, y in zip(got, want)), seed
