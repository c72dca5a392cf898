"""Calls of grad_norm, clip_grad_norm_ and AdamW that their documentation allows and that are easy to get wrong:
threads, streams, lazily negated tensors, norms beyond float32, lists with gaps, betas and eps of every kind."""
import math
import os
import subprocess
import sys
import textwrap
import threading

import numpy as np
import pytest
import torch

import adamw_oracle as AO
from conftest import ROOT
from diffrast import optim

pytestmark = pytest.mark.gpu


def f64(t):
    return t.detach().double().cpu().numpy().reshape(-1)


def fresh_python(code):
    """Runs `code` in a process of its own."""
    paths = os.pathsep.join([ROOT, os.path.join(ROOT, "mlx-swift-diffrast_b200"), os.path.join(ROOT, "tests")])
    r = subprocess.run([sys.executable, "-c", textwrap.dedent(code)], capture_output=True, text=True, timeout=300,
                       env={**os.environ, "PYTHONPATH": paths})
    assert r.returncode == 0, r.stdout + r.stderr
    return r.stdout


# ----------------------------------------------------------------- threads

def test_a_calls_launches_see_its_own_stream_whatever_other_threads_call():
    # The library's entries replaced by ones that look at the stream, wait and look again, and launch nothing: another
    # thread's call on another stream, of the same functions or of a render operator, must not come in between.
    out = fresh_python("""
        import ctypes, threading, time
        import torch
        from diffrast import _lib, ops, optim
        torch.zeros(1, device="cuda")
        real, here, at, torn, calls = _lib.lib(), threading.local(), {}, [], []

        def set_stream(ctx, stream):
            at[ctx] = stream
            return 0

        def norm(ctx, rows, count, out, work):
            a = at[ctx]
            time.sleep(0.002)
            calls.append(1)
            if a != here.stream or at[ctx] != here.stream:
                torn.append((a, at[ctx], here.stream))
            return 0

        class Library:
            dr_ctx_set_stream = ctypes.CFUNCTYPE(ctypes.c_int, ctypes.c_void_p, ctypes.c_void_p)(set_stream)
            dr_grad_norm = ctypes.CFUNCTYPE(ctypes.c_int, ctypes.c_void_p, ctypes.c_void_p, ctypes.c_int,
                                            ctypes.c_void_p, ctypes.c_void_p)(norm)
            def __getattr__(self, name):
                return getattr(real, name)

        _lib._lib = Library()
        x = torch.ones(5, device="cuda")

        def use(call):
            s = torch.cuda.Stream()
            here.stream = s.cuda_stream
            with torch.cuda.stream(s):
                for _ in range(40):
                    call()

        def render():
            ops._ctx(x)
            time.sleep(0.001)

        ts = [threading.Thread(target=use, args=(c,)) for c in (lambda: optim.grad_norm([x]),) * 3 + (render,)]
        [t.start() for t in ts]
        [t.join() for t in ts]
        print(len(calls), len(torn), torn[:3])
    """)
    assert out.split()[:2] == ["120", "0"], out


def test_two_threads_step_as_one_after_the_other():
    # Clipped steps (two launches each) of two optimizers, norms and clippings in two threads on two streams, against
    # the same ones one thread after the other.
    def job(k, seed):
        torch.manual_seed(seed)
        out, s = [], torch.cuda.Stream()
        with torch.cuda.stream(s):
            gen = torch.Generator(device="cuda").manual_seed(seed)
            ps = [torch.randn(n, device="cuda", generator=gen) for n in (200_000, 31, 5000)]
            opt = optim.AdamW(ps, state_bits=8 if k else 32, max_grad_norm=0.5 + k, seed=seed, learning_rate=1e-2)
            for _ in range(60):
                gs = [torch.sin(p * 3) * 0.1 for p in ps]
                out.append(opt.step(gs))
                out.append(optim.clip_grad_norm_(gs, 0.01))
                out.append(optim.grad_norm(gs))
            s.synchronize()
        return [torch.stack(out)] + ps

    serial = [job(k, 40 + k) for k in range(2)]
    found, errors = [None, None], []

    def run(k):
        try:
            found[k] = job(k, 40 + k)
        except Exception as e:  # shown below, in the test's own thread
            errors.append(e)

    old = sys.getswitchinterval()
    sys.setswitchinterval(1e-5)
    try:
        ts = [threading.Thread(target=run, args=(k,)) for k in range(2)]
        [t.start() for t in ts]
        [t.join() for t in ts]
    finally:
        sys.setswitchinterval(old)
    assert not errors, errors
    for a, b in zip(serial, found):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_launch_counts_and_times_hold_the_optimizers_kernels():
    from diffrast import _lib
    p = torch.randn(40_000, device="cuda")
    opt = optim.AdamW([p], max_grad_norm=1.0)
    n = _lib.launch_count(0)
    _lib.set_timing(True, 0)
    opt.step([torch.randn_like(p)])
    _lib.sync(0)
    times = _lib.timing_report(0)
    _lib.set_timing(False, 0)
    assert _lib.launch_count(0) == n + 2 and times["grad_norm_parts"][0] == 1 and times["adamw"][0] == 1


def test_a_failing_call_tells_why():
    from diffrast import _lib
    with pytest.raises(_lib.DiffRastError, match="grad_norm: .*unknown type") as e:
        rows = np.zeros(1, optim._GRAD_ROW)
        rows["type"] = 9
        error = optim._rows.norm(optim._context(0), 0, rows.tobytes(), 0.0, torch.zeros(1, device="cuda").data_ptr(), None)
        _lib.failed(*error, "grad_norm")
    assert e.value.status == _lib.DR_EINVAL


# ----------------------------------------------------------------- streams

@pytest.mark.parametrize("use", ["step", "captured", "moments", "load"])
def test_an_optimizers_memory_waits_for_the_streams_it_was_used_on(use):
    # Made on one stream and used on another, which is kept busy; then the optimizer goes.  Its buffers' memory must not
    # be handed out on the first stream while the second is to use them.
    n = 3_000_001
    p, g = torch.randn(n, device="cuda"), torch.randn(n, device="cuda")
    ref = optim.AdamW([p.clone()], learning_rate=0.1)
    ref.step([g])
    opt = optim.AdamW([p], learning_rate=0.1)
    saved = {k: v.clone() if isinstance(v, torch.Tensor) else v for k, v in opt.state_dict().items()}
    here = {t.data_ptr() for t in opt.state.values()}
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):  # kernels loaded and memory at hand: neither is to wait for the stream below
        ref.moments(0)
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        if use == "captured":
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=s):
                opt.step([g])
            graph.replay()
        torch.cuda._sleep(300_000_000)
        if use == "step":
            opt.step([g])
        elif use == "moments":
            out = opt.moments(0)
        elif use == "load":
            opt.load_state_dict(saved)
        elif use == "captured":
            graph.replay()
    busy = not s.query()
    del opt
    other = [torch.full((n + k,), math.nan, device="cuda") for k in range(-300, 300, 150) for _ in range(2)]
    assert busy and not here & {t.data_ptr() for t in other}
    torch.cuda.synchronize()
    if use == "step":
        assert torch.equal(p, ref.params[0])
    if use == "moments":
        assert all(bool((x == 0).all()) for x in out)


# ------------------------------------------------- lazily negated gradients

def negated(shape, value):
    """A tensor whose memory holds -value, as the imaginary part of a conjugated one."""
    x = torch.full(shape, -value, device="cuda")
    t = torch.complex(torch.zeros_like(x), x).conj().imag
    assert t.is_neg() and bool((t == value).all())
    return t


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("shape", [(), (1,), (1, 1, 1), (3,), (2, 5)])
def test_a_lazily_negated_gradient_is_taken_at_its_value(bits, shape):
    g = negated(shape, -2.0)
    p, q = torch.zeros(shape, device="cuda"), torch.zeros(shape, device="cuda")
    a, b = (optim.AdamW([x], learning_rate=0.1, state_bits=bits, max_grad_norm=0.5) for x in (p, q))
    na, nb = a.step([g]), b.step([torch.full(shape, -2.0, device="cuda")])
    assert torch.equal(p, q) and bool((p > 0).all()) and torch.equal(na, nb)
    assert torch.equal(a.moments(0)[0], b.moments(0)[0])
    assert torch.equal(optim.grad_norm([g]), nb)


def test_the_gradient_of_one_angle():
    # Autograd gives a one-element leaf such a gradient as it is.
    def step(negate):
        b = torch.ones(1, device="cuda", requires_grad=True)
        z = torch.complex(torch.ones(1, device="cuda"), b)
        (z.conj() * torch.tensor([2.0 + 3.0j], device="cuda")).abs().sum().backward()
        if negate:
            b.grad = b.grad.resolve_neg()
        up = float(b.grad) > 0
        optim.AdamW([b], learning_rate=0.1, weight_decay=0.0).step()
        return float(b.detach()), up
    a, up = step(False)
    assert (a < 1) == up and a == step(True)[0]


def test_clipping_a_lazily_negated_gradient_scales_it():
    g = negated((1,), 3.0)
    assert float(optim.clip_grad_norm_([g], 1.5)) == 3.0
    assert abs(float(g) - 1.5) <= 3 * AO.U * 1.5 + 1.5 * 1e-6 / 3


def test_lazily_negated_parameters_and_learning_rates_are_refused():
    with pytest.raises(ValueError, match="negated"):
        optim.AdamW([negated((1,), 1.0)])
    with pytest.raises(ValueError, match="learning_rate"):
        optim.AdamW([torch.zeros(3, device="cuda")], learning_rate=negated((1,), 1.0))


# -------------------------------------------------- norms at float32's border

LARGEST = float(np.finfo(np.float32).max)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("n", [300, 50_000])
def test_a_step_is_skipped_by_the_norm_that_it_returns(bits, n):
    # Finite gradients: a norm of 4.2e38 is infinite as a float, one of 3.4028235e38 is the largest float.
    p = torch.randn(n, device="cuda")
    old, g = p.clone(), torch.zeros(n, device="cuda")
    opt = optim.AdamW([p], state_bits=bits, max_grad_norm=1.0)
    g[:2] = 3e38
    assert float(opt.step([g])) == math.inf
    assert torch.equal(p, old) and opt.state["clocks"][0].tolist() == [0, 1, 1, 0]
    assert all(bool((opt.state[k].float() == 0).all()) for k in opt.state if k != "clocks")
    g.zero_()
    g[1] = LARGEST
    assert float(opt.step([g])) == LARGEST
    assert opt.state["clocks"][0, 0] == 1 and not torch.equal(p, old) and bool(torch.isfinite(p).all())


@pytest.mark.parametrize("n", [3, 50_000])
def test_clipping_scales_by_the_norm_in_64_bits(n):
    # The factor, 1 / 5.2e38 for three of 3e38, is 1,373,000 of the smallest float's steps: rounded by 4e-7.
    x = torch.zeros(n, device="cuda")
    x[:3] = 3e38
    value = float(x[0].double())
    assert float(optim.clip_grad_norm_([x], 1.0)) == math.inf
    want = value / (value * math.sqrt(3))
    assert abs(f64(x)[:3] - want).max() <= want * (2.0 ** -150 * value * math.sqrt(3) + 2 * AO.U)
    assert bool((x[3:] == 0).all())


# ---------------------------------------------- parameters and missing leaves

def test_clipping_refuses_parameters():
    lin = torch.nn.Linear(17, 5).cuda()
    lin(torch.randn(3, 17, device="cuda")).sum().backward()
    ps = list(lin.parameters())
    old = [(p.detach().clone(), p.grad.clone()) for p in ps]
    strided = torch.zeros(4, 6, device="cuda").t().requires_grad_()
    for given in (lin.parameters(), ps, tuple(ps), ps[0], [ps[0].grad, ps[1]], [ps[0].grad, None, strided]):
        with pytest.raises(ValueError, match="not the parameters"):
            optim.clip_grad_norm_(given, 1e-3)
    for p, (w, g) in zip(ps, old):
        assert torch.equal(p.detach(), w) and torch.equal(p.grad, g)
    assert float(optim.grad_norm(ps)) > 0  # nothing is written


def test_clipping_takes_gradients_that_are_differentiated_again():
    w = torch.randn(50, device="cuda", requires_grad=True)
    g, = torch.autograd.grad((w ** 3).sum(), w, create_graph=True)
    old, n = f64(g), float(optim.grad_norm([g]).detach())
    optim.clip_grad_norm_([g], 0.5 * n)
    assert np.abs(f64(g) - old * (0.5 * n / (n + 1e-6))).max() <= 5 * AO.U * np.abs(old).max()


@pytest.mark.parametrize("strided", [False, True])
def test_missing_gradients_are_passed_over(strided):
    gs = [torch.randn(300, 7, device="cuda"), torch.randn(9, device="cuda").half()]
    if strided:
        gs[0] = torch.randn(7, 300, device="cuda").t()
    want = optim.grad_norm(gs)
    for given in ([None, gs[0], None, gs[1]], (gs[0], gs[1], None)):
        assert torch.equal(optim.grad_norm(given), want)
    old, version = [g.clone() for g in gs], gs[0]._version
    assert torch.equal(optim.clip_grad_norm_([gs[0], None, gs[1]], 1.0), want)
    optim.clip_grad_norm_(old, 1.0)
    assert all(torch.equal(a, b) for a, b in zip(gs, old)) and gs[0]._version > version
    for given in ([None], [None, None]):
        with pytest.raises(ValueError, match="no tensors"):
            optim.grad_norm(given)
        with pytest.raises(ValueError, match="no tensors"):
            optim.clip_grad_norm_(given, 1.0)


# ------------------------------------------------------------ the C entries

def test_c_entries_refuse_misaligned_scalars():
    from diffrast import _lib
    L, c = _lib.lib(), _lib.ctx_for(0)
    x = torch.zeros(4096, device="cuda")
    p = x.data_ptr()
    row = np.zeros(1, optim._GRAD_ROW)
    row["data"], row["n"] = p, 8
    step = np.zeros(1, optim._ADAMW_ROW)
    for k, at in (("param", 0), ("grad", 512), ("m", 1024), ("v", 1536), ("clock", 2048)):
        step[k] = p + at
    step["n"] = 8
    out = p + 8192
    for off in (1, 2, 3):
        assert L.dr_grad_norm(c, row.ctypes.data, 1, out + off, None) == _lib.DR_EINVAL
        assert b"aligned" in L.dr_last_error(c)
        assert L.dr_clip_grad_norm(c, row.ctypes.data, 1, 1.0, out + off, None) == _lib.DR_EINVAL
        for lr, norm, ticket in ((None, None, out + off), (out + off, None, out), (None, out + off, out)):
            assert L.dr_adamw_step(c, step.ctypes.data, 1, 0.1, lr, 0.9, 0.999, 1e-8, 32, 1.0 if norm else 0.0, norm,
                                   p + 12288, ticket) == _lib.DR_EINVAL
            assert b"aligned" in L.dr_last_error(c)
    torch.cuda.synchronize()
    assert bool((x == 0).all())


# ------------------------------------------------------------- saved states

@pytest.mark.parametrize("bits", [32, 8])
def test_a_state_of_another_order_in_memory_is_refused(bits, tmp_path):
    # States lie in the order of their parameter's memory: a channels-last parameter's are another's.
    def make(last, **kw):
        x = torch.arange(2.0 * 3 * 4 * 5, device="cuda").view(2, 3, 4, 5)
        return optim.AdamW([x.to(memory_format=torch.channels_last) if last else x.clone()], state_bits=bits, **kw)
    g = torch.randn(2, 3, 4, 5, device="cuda")
    saved = make(True)
    saved.step([g])
    torch.save(saved.state_dict(), tmp_path / "x.pt")
    state = torch.load(tmp_path / "x.pt")
    same, other = make(True), make(False)
    same.load_state_dict(state)
    assert all(torch.equal(a, b) for a, b in zip(same.moments(0), saved.moments(0)))
    with pytest.raises(ValueError, match="order"):
        other.load_state_dict(state)
    assert other.state["clocks"][0, 0] == 0
    del state["layouts"]  # of a state saved without them
    same.load_state_dict(state)


def test_a_state_with_master_weights_is_refused_where_there_are_none():
    p = torch.randn(300, device="cuda").bfloat16()
    with_master, without = optim.AdamW([p.clone()], master_weights=True), optim.AdamW([p.clone()])
    with pytest.raises(ValueError, match="master"):
        without.load_state_dict(with_master.state_dict())
    with pytest.raises(ValueError, match="master"):
        with_master.load_state_dict(without.state_dict())


# ----------------------------------------------- gradients beyond 2^64

@pytest.mark.parametrize("size", [1.8e19, 1.9e19, 3e38])
def test_gradients_whose_squares_float32_does_not_hold(size):
    # 32-bit states: v is infinite, the update 0.  8-bit states: the block of v is NaN and the element's parameter at
    # once, the block's others with the next step, other blocks never.
    p0 = torch.randn(700, device="cuda")
    g = torch.randn(700, device="cuda")
    g[5] = size
    held = size < 2.0 ** 64
    p = p0.clone()
    opt = optim.AdamW([p], learning_rate=1e-2)
    opt.step([g])
    assert bool(torch.isfinite(p).all()) and bool(torch.isfinite(opt.state["v"][5])) == held
    if not held:
        assert abs(float(p[5]) - float(p0[5]) * (1 - 1e-4)) <= 3 * AO.U * abs(float(p0[5]))
    p = p0.clone()
    opt = optim.AdamW([p], learning_rate=1e-2, state_bits=8)
    opt.step([g])
    m, r = opt.moments(0)
    assert bool(torch.isfinite(m).all()) and bool(torch.isfinite(r[256:]).all())
    assert bool(torch.isnan(r[:256]).all()) != held and bool(torch.isfinite(r[:256]).all()) == held
    assert bool(torch.isnan(p[5])) != held and bool(torch.isfinite(p[:5]).all()) and bool(torch.isfinite(p[6:]).all())
    opt.step([torch.zeros_like(g)])
    assert bool(torch.isnan(p[:256]).all()) != held and bool(torch.isfinite(p[256:]).all())
    # clipped, the same gradient is an ordinary one
    p = p0.clone()
    opt = optim.AdamW([p], learning_rate=1e-2, state_bits=8, max_grad_norm=1.0)
    for _ in range(2):
        opt.step([g])
    assert bool(torch.isfinite(p).all()) and bool(torch.isfinite(opt.moments(0)[1]).all())


# ------------------------------------------ betas, eps, a changing rate, size

U = AO.U
TINY = 2.0 ** -149


def exact(p, g, m, v, t, lr, b1, b2, eps, wd, coef, clipped):
    """One step in 64 bits from the float32 values p, m and v (with 8-bit states v is r * r, one rounding more): (p, m,
    r) and how far float32 may be from them, each rounding half a step U.
    m: beta's, the product's, the sum's; (1 - beta)'s, the product's, the sum's, with clipping the factor's and g's.
    v: the same, and the square's; clipping counts twice.  p: 1 - lr wd, its product; of the update the factors' two, two
    products, the sum with eps, the quotient (8 bits: the product with eps's sum is fused, the reciprocal is two, its
    product is fused), and what m and r carry; the last sum.  Products below float32's normal range lose TINY."""
    c = 2 if clipped else 0
    g = g * coef
    a, b = np.abs(b1 * m), np.abs((1 - b1) * g)
    x, y = b2 * v, (1 - b2) * g * g
    m2, v2, r2 = b1 * m + (1 - b1) * g, x + y, np.sqrt(x + y)
    dm, dv = U * (3 * a + (3 + c) * b) + 2 * TINY, U * (4 * x + (4 + 2 * c) * y) + 3 * TINY
    dr = np.maximum(np.sqrt(v2 + dv) - r2, r2 - np.sqrt(np.maximum(v2 - dv, 0))) + U * r2
    root, step = math.sqrt(1 - b2 ** t), lr / (1 - b1 ** t)
    denom = r2 / root + eps
    upd = step * m2 / denom
    p2 = p * (1 - lr * wd) - upd
    # 1e-5: the products of these errors
    dp = (2 * U * np.abs(p) + step * dm / denom + np.abs(upd) * (6 * U + dr / (r2 + eps * root))) * (1 + 1e-5)
    return (p2, m2, r2), (dp + U * np.abs(p2) + TINY, dm, dr)


def grads_like(rng, n, dtype):
    x = rng.normal(size=n) * 10.0 ** rng.uniform(-4, 0, size=n) * (rng.random(n) >= 0.3)
    return torch.from_numpy(x).to("cuda", dtype)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("clip", [None, 0.05])
@pytest.mark.parametrize("p,g", [(torch.float32, torch.float32), (torch.float16, torch.float16),
                                 (torch.bfloat16, torch.float32)])
@pytest.mark.parametrize("b1,b2,eps", [(0.9, 0.999, 1e-8), (0.0, 0.99, 1e-3), (0.8, 0.0, 1e-2), (0.99, 0.9999, 1.0)])
def test_adamw_of_any_betas_and_eps(b1, b2, eps, p, g, clip, bits):
    rng = np.random.default_rng(23)
    n, wd, lr = 5000, 0.1, 1e-2
    w = torch.from_numpy(rng.normal(size=n)).to("cuda", p)
    opt = optim.AdamW([w], learning_rate=lr, beta1=b1, beta2=b2, eps=eps, weight_decay=wd, state_bits=bits,
                      max_grad_norm=clip, seed=4)
    for t in range(1, 4):
        grad = grads_like(rng, n, g)
        p0, (m0, r0) = f64(w), (f64(x) for x in opt.moments(0))
        v0 = f64(opt.state["v"][:n]) if bits == 32 else r0 * r0
        norm = opt.step([grad])
        coef = AO.clip_factor(float(np.sqrt((f64(grad) ** 2).sum())), clip)
        assert (norm is None) == (clip is None) and (clip is None or coef < 1)
        (p2, m2, r2), (dp, dm, dr) = exact(p0, f64(grad), m0, v0, t, lr, b1, b2, eps, wd, coef, clip is not None)
        half = 0.0 if p == torch.float32 else torch.finfo(p).eps / 2
        least = 2.0 ** -25 if p == torch.float16 else 0.0
        assert np.all(np.abs(f64(w) - p2) <= dp + half * (np.abs(p2) + dp) + least)
        count, b1t, b2t, _ = opt.state["clocks"][0].tolist()
        assert count == t and abs(b1t - b1 ** t) <= 1e-13 * b1 ** t and abs(b2t - b2 ** t) <= 1e-13 * b2 ** t
        m1, r1 = (f64(x) for x in opt.moments(0))
        if bits == 32:
            assert np.all(np.abs(m1 - m2) <= dm) and np.all(np.abs(r1 - r2) <= dr + U * r2)
            continue
        for k, x, dx, got, step in (("m", m2, dm, m1, 2.0 ** -4), ("r", r2, dr, r1, 2.0 ** -3)):
            scale = f64(opt._flat(k + "_scale", 0))
            top = np.abs(AO.blocks(x)).max(1)
            assert np.all(np.abs(scale * 448 - top) <= AO.blocks(dx).max(1) + 2 * U * top)
            # to nearest: half a step of the grid, 2^-4 of the value or 2^-10; to a neighbour: twice that
            grid = np.maximum(step * np.abs(x), scale.repeat(256)[:n] * step * 2.0 ** -6)
            assert np.all(np.abs(got - x) <= grid * (1 + 1e-5) + dx + 4 * U * np.abs(x))


@pytest.mark.parametrize("bits", [32, 8])
def test_a_captured_clipped_step_follows_its_learning_rate(bits):
    rates = [0.5, 0.03125, 0.0, 0.0078125]
    p, g = torch.randn(5000, device="cuda"), torch.randn(5000, device="cuda")
    ref = optim.AdamW([p.clone()], state_bits=bits, max_grad_norm=1.0)
    lr = torch.tensor(1.0, device="cuda")
    opt = optim.AdamW([p], learning_rate=lr, state_bits=bits, max_grad_norm=1.0)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step([g])
    for rate in rates:
        lr.fill_(rate)
        graph.replay()
        ref.learning_rate = rate
        ref.step([g])
        assert torch.equal(p, ref.params[0])


def test_32_bit_states_and_clipping_beyond_32_bits():
    # A tensor of 2^32 + 300 elements, 52 GB with gradient and state: its last elements against a small one's.  The squares
    # of so few bits and their sums are exact in 64 bits: norm and factor do not depend on the order.
    n = (1 << 32) + 300
    if torch.cuda.mem_get_info()[0] < 60e9:
        pytest.skip("needs 52 GB")
    bf16 = torch.bfloat16
    w, g = torch.zeros(n, device="cuda", dtype=bf16), torch.zeros(n, device="cuda", dtype=bf16)
    tail, signs = torch.randn(300, device="cuda").to(bf16), torch.randint(-3, 4, (300,), device="cuda").to(bf16)
    w[-300:], g[-300:], g[:4] = tail, signs, 1.0
    small_w, small_g = [tail.clone(), torch.zeros(4, device="cuda", dtype=bf16)], [signs.clone(), g[:4].clone()]
    opt, small = optim.AdamW([w], learning_rate=0.1), optim.AdamW(small_w, learning_rate=0.1)
    for _ in range(2):
        assert torch.equal(optim.clip_grad_norm_([g], 2.0), optim.clip_grad_norm_(small_g, 2.0))
        opt.step([g])
        small.step(small_g)
    assert torch.equal(g[-300:], small_g[0]) and torch.equal(g[:4], small_g[1])
    assert torch.equal(w[-300:], small_w[0]) and torch.equal(w[:4], small_w[1])
    for k in ("m", "v"):
        assert torch.equal(opt._flat(k, 0)[-300:], small._flat(k, 0))
        assert bool((opt._flat(k, 0)[4:1 << 20] == 0).all()) and bool((opt._flat(k, 0)[-4096:-300] == 0).all())
    assert bool((w[4:1 << 20] == 0).all()) and bool((w[(1 << 32) - 4096:-300] == 0).all())
    del w, g, opt
    torch.cuda.empty_cache()


# ------------------------------------------------------------ other captures

def test_captured_norms_and_clippings_follow_their_gradients():
    # 120 tensors (two launches, a work buffer of the graph's), their values changed between replays.
    gs = [torch.zeros(1 + 37 * i, device="cuda", dtype=(torch.float32, torch.bfloat16)[i % 2]) for i in range(120)]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        before = optim.clip_grad_norm_(gs, 1.0)
        after = optim.grad_norm(gs)
    for seed in range(3):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        for g in gs:
            g.copy_(torch.randn(g.shape, device="cuda", generator=gen))
        same = [g.clone() for g in gs]
        graph.replay()
        assert torch.equal(before, optim.clip_grad_norm_(same, 1.0)) and torch.equal(after, optim.grad_norm(same))
        assert all(torch.equal(a, b) for a, b in zip(gs, same))


@pytest.mark.parametrize("bits", [32, 8])
def test_a_captured_step_with_strided_and_missing_gradients(bits):
    def make():
        torch.manual_seed(5)
        return [torch.randn(2, 3, 8, 9, device="cuda").to(memory_format=torch.channels_last),
                torch.randn(40, 30, device="cuda"), torch.randn(7, device="cuda")]
    gs = [torch.zeros(2, 3, 8, 9, device="cuda"), torch.zeros(30, 40, device="cuda").t(), None]
    ref = optim.AdamW(make(), state_bits=bits, max_grad_norm=1.0)
    opt = optim.AdamW(make(), state_bits=bits, max_grad_norm=1.0)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = opt.step(gs)
    for k in range(3):
        for g in gs[:2]:
            g.copy_(torch.randn(g.shape, device="cuda"))
        graph.replay()
        assert torch.equal(norm, ref.step(gs))
    assert all(torch.equal(a, b) for a, b in zip(opt.params, ref.params))
    assert opt.state["clocks"][:, 0].tolist() == [3, 3, 0]


def test_an_optimizer_made_in_inference_mode_steps_outside_it_on_another_stream():
    with torch.inference_mode():
        p = torch.ones(300, device="cuda")
        opt = optim.AdamW([p], learning_rate=0.1, weight_decay=0.0, master_weights=True, max_grad_norm=1.0)
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        opt.step([torch.ones(300, device="cuda")])
        m, _ = opt.moments(0)
    s.synchronize()
    assert float((p - 0.9).abs().max()) < 1e-6 and bool((m > 0).all())


def test_a_copy_of_an_optimizer_is_refused():
    import copy
    p = torch.ones(300, device="cuda")
    opt = optim.AdamW([p])
    other = copy.deepcopy(opt)
    with pytest.raises(ValueError, match="another address"):
        other.step([torch.ones(300, device="cuda")])
    assert bool((p == 1).all()) and opt.state["clocks"][0, 0] == 0
