"""The many-tensor optimizer on the GPU: grad_norm, clip_grad_norm_ and AdamW
with 32-bit and 8-bit states, each step against the formulas in 64 bits from
the state it began with (tests/adamw_oracle.py counts the roundings)."""
import math

import numpy as np
import pytest
import torch

import adamw_oracle as AO
from diffrast import optim

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
PAIRS = [(F32, F32), (F32, BF16), (F32, F16), (BF16, BF16), (BF16, F32), (F16, F16), (F16, F32)]
HALF = {F32: 0.0, BF16: 2.0 ** -9, F16: 2.0 ** -11}  # half a step of the type, relative to the value
HALF[BF16] = torch.finfo(BF16).eps / 2
LEAST = {F32: 0.0, BF16: 0.0, F16: 2.0 ** -25}  # half of float16's smallest step


def f64(t):
    return t.detach().double().cpu().numpy().reshape(-1)


def grads_like(rng, shape, dtype, zeros=0.3):
    """Gradients of a render: some exactly zero, the others over four decades."""
    x = rng.normal(size=shape) * 10.0 ** rng.uniform(-4, 0, size=shape) * (rng.random(shape) >= zeros)
    return torch.from_numpy(x).to("cuda", dtype)


def check_step(opt, before, grads, norm, lr, wd=1e-2, eps=1e-8):
    """One step of `opt` against 64 bits.  before: [(p or master, m, sqrt(v), t, p16)] of each parameter."""
    top = opt.max_grad_norm
    if top:
        ref = math.sqrt(sum(float((f64(g) ** 2).sum()) for g in grads if g is not None))
        assert abs(float(norm) - ref) <= 2 * AO.U * ref  # 64 bits inside, one rounding to float32
        coef = AO.clip_factor(ref, top)
    else:
        assert norm is None
        coef = 1.0
    for i, (p, g) in enumerate(zip(opt.params, grads)):
        p0, m0, r0, t0 = before[i]
        m1, r1 = (f64(x) for x in opt.moments(i))
        t1, b1t, b2t, _ = opt.state["clocks"][i].tolist()
        if g is None or p.numel() == 0:
            assert t1 == t0 and np.array_equal(m1, m0) and np.array_equal(r1, r0)
            continue
        t = int(t0) + 1
        assert t1 == t and abs(b1t / 0.9 ** t - 1) < 1e-13 and abs(b2t / 0.999 ** t - 1) < 1e-13
        (p2, m2, v2), (dp, dm, dv) = AO.step(p0, f64(g.contiguous()), m0, r0, t, lr, wd=wd, eps=eps, coef=coef,
                                             clipped=bool(top), bits=opt.state_bits)
        held = "master" in opt.state and opt._half[i]
        weights = f64(opt._flat("master", i)) if held else f64(p)
        if held:
            assert np.all(np.abs(weights - p2) <= dp)
            # the parameter is the master's rounding
            assert torch.equal(p.reshape(-1), opt._flat("master", i).to(p.dtype))
        else:
            assert np.all(np.abs(weights - p2) <= dp + HALF[p.dtype] * (np.abs(p2) + dp) + LEAST[p.dtype])
        if opt.state_bits == 32:
            assert np.all(np.abs(m1 - m2) <= dm)
            assert np.all(np.abs(f64(opt._flat("v", i)) - v2) <= dv)
            continue
        r2 = np.sqrt(v2)
        for name, x, dx in (("m", m2, dm), ("r", r2, np.where(v2 > 0, dv / np.maximum(2 * r2, 1e-300), 0) + 2 * AO.U * r2)):
            scale = f64(opt._flat(name + "_scale", i))
            ref = AO.scales(x)
            np.testing.assert_allclose(scale, ref, rtol=2 * AO.U + float(np.max(dx / np.maximum(np.abs(x), 1e-300),
                                                                               where=np.abs(x) == AO.blocks(np.abs(x)).max(1).repeat(256)[:x.size], initial=0)))
            code = f64(opt._flat(name, i).float())
            per = np.maximum(scale, 1e-300).repeat(256)[:x.size]
            y = np.where(scale.repeat(256)[:x.size] > 0, x / per, 0.0)
            dy = np.where(scale.repeat(256)[:x.size] > 0, dx / per, 0.0) + 4 * AO.U * np.abs(y)
            if name == "m":
                lo, hi = AO.neighbours(np.minimum(np.abs(y), 448))
                near = np.where(np.abs(y) - lo <= hi - np.abs(y), lo, hi) * np.sign(y)
                # equal, or y lies within its error of the middle between two codes
                middle = np.abs(np.abs(y) - (lo + hi) / 2) <= dy + 1e-12
                assert np.all((code == near) | (middle & ((np.abs(code) == lo) | (np.abs(code) == hi))))
            else:
                bits = AO.random16(x.size, int(opt._tab["seed"][i]), t)
                want, gap = AO.stochastic(y, bits)
                lo, hi = AO.neighbours(np.maximum(y, 2.0 ** -9))
                width = np.where(hi > lo, hi - lo, 1.0)
                # a step of the grid is 2^20 float steps wide at its least: the low bits' cut is one of them
                close = gap <= dy / width + 2.0 ** -19
                assert np.all((code == want) | close)
                assert np.all((code == 0) == (x == 0))
                assert np.mean(close & (code != want)) < 1e-2


def snapshot(opt):
    out = []
    for i, p in enumerate(opt.params):
        w = opt._flat("master", i) if "master" in opt.state and opt._half[i] else opt._memory_order(p.detach())
        m, r = opt.moments(i)
        out.append((f64(w), f64(opt._memory_order(m)), f64(opt._memory_order(r)), opt.state["clocks"][i, 0].item()))
    return out


def run_steps(opt, grads_of, steps=3, lr=1e-2, wd=1e-2, eps=1e-8):
    for _ in range(steps):
        before, grads = snapshot(opt), grads_of()
        norm = opt.step(grads)
        check_step(opt, before, grads, norm, lr, wd, eps)


# -------------------------------------------------------------------- norm

@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("sizes", [[1], [3, 9], [255], [2048], [2049, 1, 0, 7], [100003], [1 << 20, 5]])
def test_norm(dtype, sizes):
    rng = np.random.default_rng(len(sizes) + sizes[0])
    gs = [grads_like(rng, n, dtype) + 0 for n in sizes]
    ref = math.sqrt(sum(float((f64(g) ** 2).sum()) for g in gs))
    got = optim.grad_norm(gs)
    assert got.dtype == F32 and got.shape == ()
    assert abs(float(got) - ref) <= 1.01 * AO.U * ref
    assert torch.equal(got, optim.grad_norm(gs))


def test_norm_of_many_and_mixed_tensors():
    # more tensors than one launch carries, of all types, at odd addresses
    rng = np.random.default_rng(1)
    gs = []
    for i in range(1500):
        base = grads_like(rng, int(rng.integers(2, 300)), (F32, BF16, F16)[i % 3])
        gs.append(base[1:] if i % 2 else base)
    ref = math.sqrt(sum(float((f64(g) ** 2).sum()) for g in gs))
    assert abs(float(optim.grad_norm(gs)) - ref) <= 1.01 * AO.U * ref


def test_norm_of_strided_empty_and_extreme():
    x = torch.arange(24.0, device="cuda").view(4, 6)
    for t in (x.t(), x[:, ::2], x[:, 1:3], x[0].expand(5, 6), x[2, 3]):
        ref = math.sqrt(float((f64(t.contiguous()) ** 2).sum()))
        assert abs(float(optim.grad_norm(t)) - ref) <= 1.01 * AO.U * ref
    assert float(optim.grad_norm(torch.zeros(0, device="cuda"))) == 0.0
    assert float(optim.grad_norm([torch.zeros(0, device="cuda"), torch.zeros(5, device="cuda")])) == 0.0
    for big in (1e30, 1e-30, 3e38, 1e-42):  # squares outside float32
        t = torch.full((3,), big, device="cuda")
        ref = float(t[0].double()) * math.sqrt(3)
        got = float(optim.grad_norm(t))
        assert got == math.inf if ref > 3.4028235677973366e38 else abs(got - ref) <= 1.01 * AO.U * ref + 2.0 ** -149
    assert math.isnan(float(optim.grad_norm(torch.tensor([1.0, math.nan], device="cuda"))))
    assert float(optim.grad_norm(torch.tensor([1.0, -math.inf], device="cuda"))) == math.inf


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("max_norm", [1e-3, 0.7, 1e6])
def test_clip(dtype, max_norm):
    rng = np.random.default_rng(7)
    gs = [grads_like(rng, n, dtype) for n in (1, 300, 2049, 0, 70001)] + [grads_like(rng, 1001, dtype)[1:]]
    old = [f64(g) for g in gs]
    ref = math.sqrt(sum(float((x ** 2).sum()) for x in old))
    version = gs[1]._version
    got = optim.clip_grad_norm_(gs, max_norm)
    assert abs(float(got) - ref) <= 1.01 * AO.U * ref
    assert gs[1]._version > version
    c = AO.clip_factor(ref, max_norm)
    for g, x in zip(gs, old):
        if c == 1.0:
            assert np.array_equal(f64(g), x)
        else:
            y = x * c
            assert np.all(np.abs(f64(g) - y) <= 2 * AO.U * np.abs(y) + HALF[dtype] * np.abs(y) * (1 + 3 * AO.U) +
                          LEAST[dtype] + 2.0 ** -149 + (2.0 ** -134 if dtype == BF16 else 0))


def test_clip_of_permuted_memory_and_what_is_refused():
    x = torch.randn(4, 6, 8, device="cuda")
    y = x.clone()
    n = float(optim.clip_grad_norm_(x.permute(2, 0, 1), 1.0))
    np.testing.assert_allclose(f64(x), f64(y) * (1 / (n + 1e-6)), rtol=4 * AO.U)
    for bad, text in (([x[:, :3]], "fill"), ([x, x], "share"), ([x, x[1:2]], "share")):
        with pytest.raises(ValueError, match=text):
            optim.clip_grad_norm_(bad, 1.0)
    for top in (0.0, -1.0, math.nan, math.inf):
        with pytest.raises(ValueError, match="max_norm"):
            optim.clip_grad_norm_(x, top)


def test_clip_by_a_norm_that_is_not_finite():
    x = torch.tensor([1.0, math.nan, 2.0], device="cuda")
    optim.clip_grad_norm_(x, 1.0)
    assert torch.isnan(x).all()
    x = torch.tensor([1.0, math.inf, 2.0], device="cuda")
    optim.clip_grad_norm_(x, 1.0)
    assert x[0] == 0 and torch.isnan(x[1]) and x[2] == 0


# ------------------------------------------------------------------- AdamW

SIZES = [(1,), (3, 3), (255,), (256,), (257,), (2048,), (5, 2049), (0,), (7, 11, 13)]


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("clip", [None, 0.05, 1e5])
@pytest.mark.parametrize("p,g", PAIRS)
def test_adamw(p, g, clip, bits):
    rng = np.random.default_rng(11)
    params = [torch.from_numpy(rng.normal(size=s)).to("cuda", p) for s in SIZES]
    opt = optim.AdamW(params, learning_rate=1e-2, state_bits=bits, max_grad_norm=clip, seed=5)
    run_steps(opt, lambda: [grads_like(rng, s, g) for s in SIZES])


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("p,g", [x for x in PAIRS if x[0] != F32])
def test_adamw_master_weights(p, g, bits):
    rng = np.random.default_rng(12)
    params = [torch.from_numpy(rng.normal(size=s)).to("cuda", p) for s in SIZES]
    opt = optim.AdamW(params, learning_rate=1e-2, state_bits=bits, master_weights=True, max_grad_norm=1.0)
    run_steps(opt, lambda: [grads_like(rng, s, g) for s in SIZES])


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_mixed_types_odd_addresses_and_many(bits):
    # 700 tensors of every combination, more than one launch carries; half of them begin one element off
    rng = np.random.default_rng(13)
    kinds = PAIRS + [(BF16, BF16)]
    params, types = [], []
    for i in range(700):
        p, g = kinds[i % 8] if i < 100 else kinds[0 if i < 500 else 3]
        base = torch.from_numpy(rng.normal(size=int(rng.integers(2, 700)))).to("cuda", p)
        params.append(base[1:] if i % 2 else base)
        types.append(g)
    opt = optim.AdamW(params, learning_rate=1e-2, state_bits=bits, master_weights=True, max_grad_norm=2.0)

    def grads():
        out = []
        for i, (x, g) in enumerate(zip(params, types)):
            y = grads_like(rng, x.numel() + 1, g)
            out.append(y[1:] if i % 3 == 1 else y[:-1])
        return out

    run_steps(opt, grads, steps=2)


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_strides_and_missing_gradients(bits):
    rng = np.random.default_rng(14)
    params = [torch.randn(2, 3, 8, 10, device="cuda").to(memory_format=torch.channels_last),
              torch.randn(40, 30, device="cuda").t(), torch.randn(17, device="cuda"), torch.randn((), device="cuda"),
              torch.randn(9, 5, device="cuda")]
    opt = optim.AdamW(params, learning_rate=1e-2, state_bits=bits)
    ref = optim.AdamW([p.contiguous().clone() for p in params], learning_rate=1e-2)
    for k in range(3):
        gs = [torch.randn(p.shape, device="cuda") for p in params]
        gs[4] = torch.randn(9, 1, device="cuda").expand(9, 5)  # a broadcast input's gradient
        if k == 1:
            gs[2] = None
        given = [gs[0].to(memory_format=torch.channels_last), gs[1], gs[2], gs[3], gs[4]]
        opt.step(given)
        ref.step(gs)
    for i, (a, b) in enumerate(zip(opt.params, ref.params)):
        assert opt.state["clocks"][i, 0] == (2 if i == 2 else 3)
        if bits == 32:
            assert torch.equal(a, b)
            assert torch.equal(opt.moments(i)[0], ref.moments(i)[0]) and torch.equal(opt.moments(i)[1], ref.moments(i)[1])
    opt.step([None] * 5)  # nothing to do
    assert opt.state["clocks"][0, 0] == 3


def test_adamw_takes_the_parameters_gradients():
    w = torch.randn(50, 3, device="cuda", requires_grad=True)
    u = torch.randn(4, device="cuda", requires_grad=True)
    opt = optim.AdamW([w, u], learning_rate=0.1, max_grad_norm=1.0)
    y = (w * w).sum()
    y.backward()
    p0, version = w.detach().clone(), w._version
    norm = opt.step()
    assert float(norm) == pytest.approx(2 * float(p0.norm()), rel=1e-5)
    assert w._version > version and not torch.equal(w.detach(), p0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        z = (w * w).sum()
        opt.step()
        z.backward()


def test_adamw_refusals():
    w = torch.randn(6, 4, device="cuda")
    h = torch.randn(6, device="cuda").half()
    with pytest.raises(ValueError, match="fill"):
        optim.AdamW([w[:, :2]])
    with pytest.raises(ValueError, match="share"):
        optim.AdamW([w, w[2:]])
    with pytest.raises(ValueError, match="float32, bfloat16 or float16"):
        optim.AdamW([w.double()])
    for kw in (dict(weight_decay=[0.1]), dict(lr_ratios=[1.0, 2.0, 3.0]), dict(weight_decay=-1.0),
               dict(lr_ratios=[1.0, math.nan])):
        with pytest.raises(ValueError, match="weight_decay|lr_ratios"):
            optim.AdamW([w, h], **kw)
    opt = optim.AdamW([w, h])
    before = snapshot(opt)
    g, k = torch.zeros_like(w), torch.zeros_like(h)
    for bad in ([g], [g, k, k], [g.t(), k], [g.cpu(), k], [g.double(), k], [g, k.bfloat16()], [3.0, k],
                [g.to_sparse(), k], [g[:, :3], k]):
        with pytest.raises(ValueError, match="AdamW"):
            opt.step(bad)
    opt.learning_rate = -1.0
    with pytest.raises(ValueError, match="learning_rate"):
        opt.step([g, k])
    opt.learning_rate = 0.1
    h.data = torch.randn(6, device="cuda")
    with pytest.raises(ValueError, match="another"):
        opt.step([g, k])
    for a, b in zip(before[:1], snapshot(opt)[:1]):
        assert all(np.array_equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_adamw_skips_a_step_whose_norm_is_not_finite(bits, bad):
    rng = np.random.default_rng(15)
    params = [torch.randn(300, device="cuda"), torch.randn(9, device="cuda").half()]
    opt = optim.AdamW(params, state_bits=bits, max_grad_norm=1.0)
    opt.step([grads_like(rng, 300, F32), grads_like(rng, 9, F16)])
    before = snapshot(opt)
    gs = [grads_like(rng, 300, F32), grads_like(rng, 9, F16)]
    gs[1][4] = bad
    assert not math.isfinite(float(opt.step(gs)))
    for a, b in zip(before, snapshot(opt)):
        assert all(np.array_equal(x, y) for x, y in zip(a, b))
    run_steps(opt, lambda: [grads_like(rng, 300, F32), grads_like(rng, 9, F16)], lr=1e-3)


def test_adamw8_blocks_with_extremes():
    # (a) a NaN or an infinity makes its block NaN, and no other; (b) a block of zeros stays zero; (c) gradients whose
    # squares vanish in float32 leave v at 0; (d) first moments below 2^-100 are dropped
    w = torch.randn(256 * 6 + 10, device="cuda")
    opt = optim.AdamW([w], state_bits=8, learning_rate=1e-3)
    g = torch.randn_like(w)
    g[5], g[256 + 3], g[512:768], g[768:1024], g[1024:1280] = math.nan, math.inf, 0, 1e-30, 1e-36
    old = w.clone()
    opt.step([g])
    m, r = opt.moments(0)
    assert torch.isnan(m[:512]).all() and torch.isnan(r[:512]).all() and torch.isfinite(m[512:]).all()
    assert torch.isnan(w[5]) and torch.isfinite(w[:5]).all() and torch.isfinite(w[512:]).all()
    assert (m[512:768] == 0).all() and (r[512:768] == 0).all()
    np.testing.assert_allclose(f64(w[512:768]), f64(old[512:768]) * (1 - 1e-5), rtol=3 * AO.U)
    # 0.1 * 1e-30 = 1e-31 < 2^-100 = 7.9e-31: both small blocks' first moments are dropped
    assert (r[768:1280] == 0).all() and (m[768:1280] == 0).all()
    assert torch.isfinite(r[1280:]).all() and (r[1280:] > 0).all()


def test_adamw8_root_of_a_vanishing_square():
    # 0.1 * 1e-25 > 2^-100 is kept as a first moment; 0.001 * 1e-50 is 0 in float32, and so is its root
    w = torch.zeros(300, device="cuda")
    opt = optim.AdamW([w], state_bits=8, learning_rate=1e-3)
    opt.step([torch.full((300,), 1e-25, device="cuda")])
    m, r = opt.moments(0)
    np.testing.assert_allclose(f64(m), 1e-26, rtol=2.0 ** -4)
    assert (r == 0).all() and torch.isfinite(w).all()


def test_adamw8_second_moment_is_unbiased():
    # Constant gradients: v's mean over many elements follows 1 - beta2^t.  Nearest rounding would stop it after some
    # tens of steps.  r's noise is below 0.3 of itself (a step of the grid is at most 1/8), so the mean of 65,536
    # elements is within 6 * 0.3 / 256 of the mean.
    n = 1 << 16
    w = torch.zeros(n, device="cuda")
    scale = torch.rand(n, device="cuda") * 0.9 + 0.1
    scale[::256] = 1.0  # each block's largest
    opt = optim.AdamW([w], state_bits=8, learning_rate=0.0, seed=3)
    for t in range(1, 401):
        opt.step([scale])
        if t in (20, 100, 400):
            r = opt.moments(0)[1]
            ratio = f64((r / scale).square()).mean() / (1 - 0.999 ** t)
            # E[r^2] exceeds E[r]^2 by the noise
            assert 1 - 0.01 < ratio < 1 + 0.3 ** 2 + 0.01, (t, ratio)


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_ratios_decays_and_a_device_learning_rate(bits):
    rng = np.random.default_rng(16)
    shapes, ratios, decays = [(300,), (20, 9), (5,)], [1.0, 0.1, 0.0], [0.0, 0.5, 0.02]
    params = [torch.randn(s, device="cuda") for s in shapes]
    lr = torch.tensor([0.03125], device="cuda")
    opt = optim.AdamW(params, learning_rate=lr, lr_ratios=ratios, weight_decay=decays, state_bits=bits)
    for k in range(3):
        before, gs = snapshot(opt), [grads_like(rng, s, F32) for s in shapes]
        lr.mul_(0.5)
        opt.step(gs)
        for i in range(3):
            p0, m0, r0, t0 = before[i]
            (p2, _, _), (dp, _, _) = AO.step(p0, f64(gs[i]), m0, r0, int(t0) + 1, 0.03125 * 0.5 ** (k + 1) * ratios[i],
                                             wd=decays[i], bits=bits)
            assert np.all(np.abs(f64(params[i]) - p2) <= dp)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("clip", [None, 0.5])
def test_adamw_captured_steps_are_the_eager_ones(bits, clip):
    shapes = [(1000,), (77, 3), (5,)]
    torch.manual_seed(0)
    init = [torch.randn(s, device="cuda") for s in shapes]
    grads = [[torch.randn(s, device="cuda") for s in shapes] for _ in range(4)]
    eager = optim.AdamW([x.clone() for x in init], state_bits=bits, max_grad_norm=clip, seed=9)
    norms = [eager.step(g) for g in grads]
    opt = optim.AdamW([x.clone() for x in init], state_bits=bits, max_grad_norm=clip, seed=9)
    held = [g.clone() for g in grads[0]]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = opt.step(held)
    for k, g in enumerate(grads):
        for a, b in zip(held, g):
            a.copy_(b)
        graph.replay()
        if clip:
            assert torch.equal(norm, norms[k])
    torch.cuda.synchronize()
    for a, b in zip(opt.params, eager.params):
        assert torch.equal(a, b)
    for k in opt.state:
        assert torch.equal(opt.state[k].view(torch.uint8), eager.state[k].view(torch.uint8))
    assert int(opt._ticket) == 0


def test_adamw_on_other_streams_two_optimizers_and_two_graphs():
    # Two optimizers' captured clipped steps replay side by side on two streams: nothing of the one is in the other.
    torch.manual_seed(1)
    n = 300_001
    sides = []
    for k in range(2):
        w = torch.randn(n, device="cuda")
        g = torch.randn(n, device="cuda") * (k + 1)
        ref = optim.AdamW([w.clone()], state_bits=8, max_grad_norm=0.1 + k, seed=k)
        opt = optim.AdamW([w], state_bits=8, max_grad_norm=0.1 + k, seed=k)
        for _ in range(20):
            ref.step([g])
        torch.cuda.synchronize()
        s = torch.cuda.Stream()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            norm = opt.step([g])
        sides.append((w, g, ref, opt, s, graph, norm))
    torch.cuda.synchronize()
    for _ in range(20):
        for w, g, ref, opt, s, graph, norm in sides:
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    for w, g, ref, opt, s, graph, norm in sides:
        assert torch.equal(w, ref.params[0])
        assert abs(float(norm) - float(f64(g).dot(f64(g))) ** 0.5) <= 1.01 * AO.U * float(norm)


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_goes_on_from_a_saved_state(bits, tmp_path):
    rng = np.random.default_rng(17)
    shapes = [(500,), (3, 100)]
    types = [F32, BF16]
    kw = dict(state_bits=bits, master_weights=True, seed=2, learning_rate=1e-2)
    params = [torch.randn(s, device="cuda").to(t) for s, t in zip(shapes, types)]
    opt = optim.AdamW(params, **kw)
    grads = [[grads_like(rng, s, t) for s, t in zip(shapes, types)] for _ in range(5)]
    for g in grads[:2]:
        opt.step(g)
    torch.save({"opt": opt.state_dict(), "params": [p.clone() for p in params]}, tmp_path / "x.pt")
    for g in grads[2:]:
        opt.step(g)
    saved = torch.load(tmp_path / "x.pt")
    again = optim.AdamW(saved["params"], **kw)
    again.load_state_dict(saved["opt"])
    for g in grads[2:]:
        again.step(g)
    for a, b in zip(opt.params, again.params):
        assert torch.equal(a, b)
    with pytest.raises(ValueError, match="seed"):
        optim.AdamW(saved["params"], **{**kw, "seed": 3}).load_state_dict(saved["opt"])
    with pytest.raises(ValueError, match="state_bits"):
        optim.AdamW(saved["params"], **{**kw, "state_bits": 40 - bits}).load_state_dict(saved["opt"])
    with pytest.raises(ValueError, match="other parameters"):
        optim.AdamW(saved["params"][:1], **kw).load_state_dict(saved["opt"])


def test_adamw_offsets_beyond_32_bits():
    # One tensor of 2^32 + 300 elements (26 GB with its gradient and state): its last block against a small tensor's
    # same step; the random bits differ with the block's place, the rest must not.
    n = (1 << 32) + 300
    if torch.cuda.get_device_properties(0).total_memory < 60e9:
        pytest.skip("needs 30 GB")
    w = torch.zeros(n, device="cuda", dtype=BF16)
    g = torch.zeros(n, device="cuda", dtype=BF16)
    tail = torch.randn(300, device="cuda").to(BF16)
    w[-300:], g[-300:] = tail, tail.flip(0)
    g[:4] = 1.0
    opt = optim.AdamW([w], state_bits=8, max_grad_norm=1.0, learning_rate=0.1)
    small_w, small_g = tail.clone(), tail.flip(0).clone()
    small = optim.AdamW([small_w, torch.zeros(4, device="cuda", dtype=BF16)], state_bits=8, max_grad_norm=1.0,
                        learning_rate=0.1)
    norm = opt.step([g])
    ref = small.step([small_g, torch.ones(4, device="cuda", dtype=BF16)])
    assert abs(float(norm) - float(ref)) <= 3 * AO.U * float(ref)
    assert torch.equal(w[-300:], small_w)
    assert torch.equal(opt.state["m"][-512:][:300].view(torch.uint8), small.state["m"][:300].view(torch.uint8))
    assert torch.equal(opt.state["m_scale"][-2:], small.state["m_scale"][:2])
    assert bool((w[4:1 << 20] == 0).all()) and bool((w[(1 << 32) - 4096:-300] == 0).all()) and bool((w[:4] < 0).all())
    del w, g, opt
    torch.cuda.empty_cache()


def test_a_training_step_from_render_to_update():
    # The colour fit's chain, its gradients' norm, the clipped step: each update is the formula's of the gradients that
    # the chain gave, in fp32 and with 8-bit states, and the same gradients clipped by themselves give the same step.
    from diffrast import chains
    for bits in (32, 8):
        c = chains.Cfg1(torch.device("cuda"))
        params = c.params()
        opt = optim.AdamW(params, learning_rate=1e-2, state_bits=bits, max_grad_norm=1e-3)
        by_hand = optim.AdamW([p.detach().clone() for p in params], learning_rate=1e-2, state_bits=bits)
        for _ in range(4):
            c.zero_grad()
            c.step()
            before, grads = snapshot(opt), [p.grad.clone() for p in params]
            assert float(optim.grad_norm(grads)) > 1e-3
            norm = opt.step()
            check_step(opt, before, grads, norm, 1e-2)
            clipped = [g.clone() for g in grads]
            assert torch.equal(optim.clip_grad_norm_(clipped, 1e-3), norm)
            by_hand.step(clipped)
        for a, b in zip(params, by_hand.params):
            assert torch.equal(a.detach(), b)


# ---------------------------------------------------------- calls in the wild

def unfused8(state, g, coef, seeds, begins, counts, t):
    """8-bit states after a step, each operation a torch one in float32: (m, r, scales) of each tensor."""
    out = []
    for b, n, seed in zip(begins, counts, seeds):
        pad = -(-n // 256) * 256
        gi = torch.zeros(pad, device="cuda")
        gi[:n] = g[b:b + n].float()
        if coef is not None:
            gi = gi * coef
        m, r = (state[k][b:b + pad].float().view(-1, 256) * state[k + "_scale"][b // 256:(b + pad) // 256, None]
                for k in ("m", "r"))
        m = (m * 0.9).view(-1) + gi * (1 - 0.9)
        r = ((r * r * 0.999).view(-1) + gi * gi * (1 - 0.999)).sqrt()
        res = []
        for x in (m, r):
            x = x.view(-1, 256)
            top = x.abs().amax(1)
            inv = torch.where(top > 0, torch.full_like(top, 448.0) / top, 0.0)
            res += [(x * inv[:, None]).view(-1), top * (1 / 448)]
        bits = torch.from_numpy(AO.random16(pad, seed, t)).to("cuda", torch.int32)
        y = torch.where(res[2] > 0, res[2].clamp_min(2.0 ** -9), 0.0)
        low = torch.where(y < 2.0 ** -6, 2.0 ** -6, 0.0)
        y = (((y + low).view(torch.int32) + bits * 16 + 8) & ~0xFFFFF).view(torch.float32) - low
        out.append((res[0].clamp(-448, 448).to(torch.float8_e4m3fn).float()[:n], y.clamp(max=448.0)[:n], res[1], res[3]))
    return out


@pytest.mark.parametrize("g_type", [F32, F16])
def test_adamw8_codes_are_the_unfused_evaluations(g_type):
    # Codes and scales bit for bit, over several steps: no rounding is left out and none is added.
    rng = np.random.default_rng(19)
    counts = [100_000, 777, 3]
    params = [torch.randn(n, device="cuda").to(g_type) for n in counts]
    opt = optim.AdamW(params, state_bits=8, max_grad_norm=0.5, seed=11)
    begins = [int(b) for b in opt._begins]
    flat = torch.zeros(opt.state["m"].numel(), device="cuda", dtype=g_type)
    for t in range(1, 6):
        gs = [grads_like(rng, n, g_type) for n in counts]
        for b, g in zip(begins, gs):
            flat[b:b + g.numel()] = g
        norm = torch.stack([g.double().square().sum() for g in gs]).sum().sqrt()
        coef = (0.5 / (norm + 1e-6)).clamp(max=1.0).float()
        want = unfused8(opt.state, flat, coef, [int(x) for x in opt._tab["seed"]], begins, counts, t)
        opt.step(gs)
        for i, (m, r, ms, rs) in enumerate(want):
            assert torch.equal(opt._flat("m", i).float(), m) and torch.equal(opt._flat("r", i).float(), r)
            assert torch.equal(opt._flat("m_scale", i), ms) and torch.equal(opt._flat("r_scale", i), rs)


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_queued_steps_are_the_waited_ones(bits):
    # 60 clipped steps queued without a wait, their gradients made by kernels between them, against the same steps
    # with a wait after each launch: the step that begins while the norm still runs reads nothing too early.
    def run(wait):
        torch.manual_seed(4)
        params = [torch.randn(n, device="cuda") for n in (400_000, 31, 70_003)]
        opt = optim.AdamW(params, state_bits=bits, max_grad_norm=1.0, learning_rate=1e-2)
        norms = []
        for _ in range(60):
            gs = [torch.sin(p * 3) * 0.1 for p in params]
            if wait:
                torch.cuda.synchronize()
            norms.append(opt.step(gs))
            if wait:
                torch.cuda.synchronize()
            optim.clip_grad_norm_(gs, 0.01)
            norms.append(optim.grad_norm(gs))
        torch.cuda.synchronize()
        return params, norms
    (p1, n1), (p2, n2) = run(False), run(True)
    assert all(torch.equal(a, b) for a, b in zip(p1, p2)) and torch.equal(torch.stack(n1), torch.stack(n2))


def test_clip_of_more_tensors_than_a_launch_carries():
    rng = np.random.default_rng(21)
    gs = [grads_like(rng, int(rng.integers(1, 400)), (F32, BF16, F16)[i % 3]) for i in range(2300)]
    old = [f64(g) for g in gs]
    ref = math.sqrt(sum(float((x ** 2).sum()) for x in old))
    got = optim.clip_grad_norm_(gs, 0.25 * ref)
    assert abs(float(got) - ref) <= 1.01 * AO.U * ref
    c = AO.clip_factor(ref, 0.25 * ref)
    for g, x in zip(gs, old):
        y = x * c
        assert np.all(np.abs(f64(g) - y) <= (2 * AO.U + HALF[g.dtype]) * np.abs(y) * (1 + 4 * AO.U) + 2.0 ** -25)


def test_modules_parameters_inference_tensors_and_generators():
    lin = torch.nn.Linear(17, 5).cuda()
    opt = optim.AdamW(lin.parameters(), learning_rate=0.01, max_grad_norm=1.0)
    lin(torch.randn(3, 17, device="cuda")).sum().backward()
    before = [p.detach().clone() for p in lin.parameters()]
    run_steps(opt, lambda: [p.grad for p in lin.parameters()], steps=1)
    assert all(not torch.equal(a, b) for a, b in zip(before, lin.parameters()))
    with torch.inference_mode():
        x = torch.ones(9, device="cuda")
        y = torch.zeros(9, device="cuda")
        inner = optim.AdamW([y], learning_rate=0.1)
        inner.step([x])
        assert float(optim.clip_grad_norm_((t for t in [x]), 1.5)) == 3.0
    torch.testing.assert_close(x.cpu(), torch.full((9,), 0.5), rtol=1e-6, atol=0)
    assert (y < -0.09).all()


def test_state_stays_where_it_is_while_a_graph_lives():
    # A captured step, an eager one between its replays, a state loaded between them: one sequence of steps.
    torch.manual_seed(8)
    w0, g = torch.randn(1000, device="cuda"), torch.randn(1000, device="cuda")
    ref = optim.AdamW([w0.clone()], state_bits=8, max_grad_norm=1.0)
    opt = optim.AdamW([w0.clone()], state_bits=8, max_grad_norm=1.0)
    fresh = {k: v.clone() if isinstance(v, torch.Tensor) else v for k, v in opt.state_dict().items()}
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step([g])
    for _ in range(2):
        graph.replay()
        opt.step([g])
    for _ in range(4):
        ref.step([g])
    assert torch.equal(opt.params[0], ref.params[0]) and opt.state["clocks"][0, 0] == 4
    opt.load_state_dict(fresh)
    opt.params[0].copy_(w0)
    for _ in range(4):
        graph.replay()
    assert torch.equal(opt.params[0], ref.params[0])


def test_c_entries_refuse_bad_rows():
    import ctypes

    from diffrast import _lib
    L, c = _lib.lib(), _lib.ctx_for(0)
    x = torch.zeros(600, device="cuda")
    k = torch.zeros(4, dtype=torch.float64, device="cuda")
    ticket = torch.zeros(1, dtype=torch.int32, device="cuda")
    work = torch.zeros(4096, dtype=torch.float64, device="cuda")
    p = x.data_ptr()
    good = dict(param=p, grad=p + 1024, master=0, m=p + 1600, v=p + 1800, m_scale=p + 2000, v_scale=p + 2100,
                clock=k.data_ptr(), n=8, lr_ratio=1.0, weight_decay=0.0, seed=0, param_type=0, grad_type=0)

    def step(bits=8, lr=0.0, b1=0.9, eps=1e-8, top=0.0, norm=p + 2200, wk=work.data_ptr(), tick=ticket.data_ptr(), **kw):
        row = np.zeros(1, optim._ADAMW_ROW)
        for name, v in {**good, **kw}.items():
            row[name] = v
        return L.dr_adamw_step(c, row.ctypes.data, 1, lr, None, b1, 0.999, eps, bits, top, norm, wk, tick)

    assert step() == _lib.DR_OK
    for kw in (dict(bits=16), dict(lr=-1.0), dict(lr=math.nan), dict(b1=1.0), dict(eps=0.0), dict(eps=1e-40),
               dict(top=-1.0), dict(top=math.nan), dict(top=1.0, norm=None), dict(top=1.0, wk=None), dict(tick=None),
               dict(n=-1), dict(n=1 << 62), dict(param=0), dict(grad=0), dict(m=0), dict(clock=0), dict(m_scale=0),
               dict(param_type=3), dict(grad_type=-1), dict(param_type=1, grad_type=2), dict(master=p),
               dict(param=p + 2), dict(clock=k.data_ptr() + 4), dict(lr_ratio=-1.0), dict(weight_decay=math.inf)):
        assert step(**kw) == _lib.DR_EINVAL, kw
        assert b"adamw" in L.dr_last_error(c)

    def norm(fn, *extra, **kw):
        row = np.zeros(1, optim._GRAD_ROW)
        for name, v in {**dict(data=p, n=8, type=0), **kw}.items():
            row[name] = v
        return fn(c, row.ctypes.data, 1, *extra, p + 2200, work.data_ptr())

    for fn, extra in ((L.dr_grad_norm, ()), (L.dr_clip_grad_norm, (1.0,))):
        assert norm(fn, *extra) == _lib.DR_OK
        for kw in (dict(data=0), dict(n=-1), dict(n=1 << 62), dict(type=5), dict(data=p + 1)):
            assert norm(fn, *extra, **kw) == _lib.DR_EINVAL, kw
    for top in (0.0, -1.0, math.nan, math.inf):
        assert norm(L.dr_clip_grad_norm, top) == _lib.DR_EINVAL
    assert L.dr_grad_norm(c, None, 1, p, work.data_ptr()) == _lib.DR_EINVAL
    assert L.dr_grad_norm(c, None, 0, None, work.data_ptr()) == _lib.DR_EINVAL
    assert L.dr_grad_norm(c, None, -1, p, work.data_ptr()) == _lib.DR_EINVAL
    torch.cuda.synchronize()
    assert ctypes.sizeof(ctypes.c_void_p) == 8 and bool((x[:256] == 0).all())


def test_small_norms_need_no_work_and_large_ones_do():
    # The bounds that the header names: 64 tensors, 16,384 elements in steps of 2048.
    from diffrast import _lib
    L, c = _lib.lib(), _lib.ctx_for(0)
    x = torch.randn(40_000, device="cuda")
    norm = torch.zeros((), device="cuda")

    def call(sizes):
        rows = np.zeros(len(sizes), optim._GRAD_ROW)
        rows["data"], rows["n"] = x.data_ptr(), sizes
        return L.dr_grad_norm(c, rows.ctypes.data, len(sizes), norm.data_ptr(), None)

    for sizes in ([16384], [2048] * 8, [1] * 8, [0] * 64 + [], [5] * 7 + [0] * 50, [14336, 1]):
        assert call(sizes) == _lib.DR_OK
        ref = math.sqrt(sum(float((f64(x[:n]) ** 2).sum()) for n in sizes))
        assert abs(float(norm) - ref) <= 1.01 * AO.U * ref, sizes
    for sizes in ([16385], [2048] * 8 + [1], [1] * 9, [0] * 65, [14337, 1, 1]):
        assert call(sizes) == _lib.DR_EINVAL
    for n in (16384, 16385):
        ref = math.sqrt(float((f64(x[:n]) ** 2).sum()))
        assert abs(float(optim.grad_norm([x[:n]])) - ref) <= 1.01 * AO.U * ref


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("sizes", [[5], [2048] * 8, [16384], [1, 0, 300, 7] * 2, [16385], [2048] * 8 + [1]])
def test_clip_in_one_block_and_in_more(dtype, sizes):
    rng = np.random.default_rng(sum(sizes))
    gs = [(grads_like(rng, n + 1, dtype) + 0)[i % 2:][:n] for i, n in enumerate(sizes)]
    old = [f64(g) for g in gs]
    ref = math.sqrt(sum(float((x ** 2).sum()) for x in old))
    for top in (2 * ref + 1, 0.3 * ref + 1e-4):
        got = optim.clip_grad_norm_(gs, top)
        assert abs(float(got) - ref) <= 1.01 * AO.U * ref
    c = AO.clip_factor(ref, top)
    for g, x in zip(gs, old):
        y = x * c
        assert np.all(np.abs(f64(g) - y) <= (2 * AO.U + HALF[dtype]) * np.abs(y) * (1 + 4 * AO.U) + 2.0 ** -25)
