"""The optimizer operators' workloads: gradient norm and clipping, and the AdamW step with 32-bit and with 8-bit
states, over the leaves of the scenes this framework fits.

A case names an operator and a list of tensors: a scene of the benchmark's configurations, or `tensors` sizes drawn
from `smallest` to `largest` elements.  Every tensor lies in a slot of a flat buffer that begins at a multiple of 256
elements, so outputs are few and whole; the tensors themselves are what the operators get.

Definitions, per element of a tensor at its step t (counted from 1), all rounded to float32 operation by operation:
  g' = c g with c = min(1, max_norm / (norm + 1e-6)) where the step clips, and norm the 2-norm over all tensors
  m' = b1 m + (1 - b1) g',  v' = b2 v + (1 - b2) g'^2,  r' = sqrt(v')
  p' = p (1 - lr wd) - ((lr / (1 - b1^t)) m') / (r' / sqrt(1 - b2^t) + eps)
8-bit states hold m and r as e4m3 times a scale for each block of 256 elements of a tensor, the block's largest
magnitude / 448 (0 below 2^-100): m rounded to nearest, r to one of its two neighbours by 16 random bits that are a
function of (seed, tensor, t, element), and to 2^-9 at least where r is not 0.
"""
import os
import random
import sys

import torch

own = False

BLOCK = 256
B1, B2, EPS, LR, WD = 0.9, 0.999, 1e-8, 1e-3, 1e-2
SEED = 1234
MAX32 = 0xFFFFFFFF
GOLDEN = 0x9E3779B9
LARGEST = 16 * 2048 * 2048 * 4  # elements of the largest listed case

DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}

SCENES = {
    # vertices and colours of one triangle: the smallest fit
    "triangle": [(1, 3, 4), (3, 3)],
    # 8 views' positions of an icosphere, its colours, uv and a 512^2 texture
    "sphere": [(8, 2562, 4), (2562, 3), (2562, 2), (512, 512, 3)],
    # 16 views' positions, uv and a trilinear 2048^2 texture
    "mip": [(16, 2562, 4), (2562, 2), (2048, 2048, 4)],
    # vertices and 8 attributes each of the million-triangle soup
    "soup": [(2640000, 4), (2640000, 8)],
    # a geodesic sphere's vertices and its cube map
    "cube": [(249642, 4), (6, 1024, 1024, 3)],
    # sixteen 2048^2 textures of 4 channels
    "atlas": [(2048, 2048, 4)] * 16,
}


def _case(name, op, scene="", tensors=0, smallest=0, largest=0, pick=0, param="float32", grad="float32", bits=32,
          master=False, max_norm=0.0):
    return dict(name=name, op=op, scene=scene, tensors=tensors, smallest=smallest, largest=largest, pick=pick,
                param=param, grad=grad, bits=bits, master=master, max_norm=max_norm)


def listed():
    return [
        # A fit's two small leaves: all latency.
        _case("norm triangle", "grad_norm", "triangle"),
        # The gradients of the largest benchmark scene, logged or checked each step.
        _case("norm soup", "grad_norm", "soup"),
        # Clipping before an optimizer of the user's own; the texture dominates.
        _case("clip mip", "clip", "mip", max_norm=1.0),
        # Clipping the gradients of a scene of many half-precision objects, most of them ragged.
        _case("clip 120 bf16", "clip", tensors=120, smallest=9, largest=1 << 21, pick=3, param="bfloat16",
              grad="bfloat16", max_norm=0.5),
        # The step of the smallest fit.
        _case("adamw triangle", "adamw", "triangle"),
        # The whole clipped step of the textured sphere.
        _case("adamw sphere clip", "adamw", "sphere", max_norm=1.0),
        # Many objects in bf16 with fp32 master weights, odd sizes.
        _case("adamw 120 bf16 master", "adamw", tensors=120, smallest=9, largest=1 << 21, pick=4, param="bfloat16",
              grad="bfloat16", master=True),
        # The largest: sixteen textures in fp32.
        _case("adamw atlas", "adamw", "atlas"),
        # 8-bit states of a small scene.
        _case("adamw8 sphere", "adamw", "sphere", bits=8),
        # 8-bit states of the soup, with clipping.
        _case("adamw8 soup clip", "adamw", "soup", bits=8, max_norm=1.0),
        # Half-precision textures with 8-bit states: a byte-starved atlas.
        _case("adamw8 atlas fp16", "adamw", "atlas", param="float16", grad="float16", bits=8),
        # A few ragged tensors in bf16 with fp32 gradients.
        _case("adamw8 12 bf16", "adamw", tensors=12, smallest=1000, largest=1 << 22, pick=5, param="bfloat16",
              grad="float32", bits=8),
    ]


def draw(rng):
    op = rng.choice(["grad_norm", "clip", "adamw", "adamw", "adamw", "adamw"])
    tensors = int(2 ** rng.uniform(0, 8))
    top = LARGEST // 2 // tensors
    largest = min(top, int(2 ** rng.uniform(4, 25)))
    smallest = max(1, int(largest ** rng.uniform(0.2, 1.0)))
    param = rng.choice(["float32", "bfloat16", "float16"])
    grad = rng.choice([param, "float32"])
    if op != "adamw":
        param = grad
    bits = rng.choice([32, 8]) if op == "adamw" else 32
    master = op == "adamw" and param != "float32" and rng.random() < 0.4
    max_norm = 0.0 if op == "grad_norm" else 10 ** rng.uniform(-2, 1)
    if op == "adamw" and rng.random() < 0.5:
        max_norm = 0.0
    case = _case("", op, "", tensors, smallest, largest, rng.randrange(1 << 20), param, grad, bits, master, max_norm)
    del case["name"]
    return case


def _shapes(case):
    if case["scene"]:
        return SCENES[case["scene"]]
    r = random.Random(case["pick"])
    lo, hi = case["smallest"], case["largest"]
    return [(max(lo, min(hi, int(lo * (hi / lo) ** r.random()))),) for _ in range(case["tensors"])]


def _count(shape):
    n = 1
    for d in shape:
        n *= d
    return n


def work(case):
    n = sum(_count(s) for s in _shapes(case))
    g, p = (torch.finfo(DTYPES[case[k]]).bits // 8 for k in ("grad", "param"))
    if case["op"] == "grad_norm":
        return {"bytes": n * g + 4, "flops": 2 * n}
    if case["op"] == "clip":
        return {"bytes": 2 * n * g + 4, "flops": 3 * n}
    weights = 8 + p if case["master"] else 2 * p
    state = 16 if case["bits"] == 32 else 4
    blocks = 0 if case["bits"] == 32 else sum(-(-_count(s) // BLOCK) for s in _shapes(case))
    flops = 14 + (3 if case["max_norm"] else 0) + (12 if case["bits"] == 8 else 0)
    return {"bytes": n * (weights + g + state) + 16 * blocks, "flops": flops * n}


def _package():
    if "diffrast.optim" not in sys.modules:
        sys.path.insert(0, os.path.join(os.getcwd(), "mlx-swift-diffrast_b200"))
    from diffrast import optim
    return optim


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(int(seed))
    shapes = _shapes(case)
    counts = [_count(s) for s in shapes]
    begins, total = [], 0
    for n in counts:
        begins.append(total)
        total += -(-n // BLOCK) * BLOCK

    def normal():
        return torch.randn(total, generator=gen, device=dev)

    # Gradients of a render: 3 in 10 rows of eight elements get none, the others span four decades.
    rows = torch.rand(total // 8, generator=gen, device=dev)
    seen = (torch.rand(total // 8, generator=gen, device=dev) > 0.3).float()
    size = (torch.pow(10.0, -4 * rows) * seen).repeat_interleave(8)

    def flat(x, dtype):
        for b, n in zip(begins, counts):  # nothing lies between the tensors
            x[b + n:b + -(-n // BLOCK) * BLOCK] = 0
        return x.to(dtype)

    def views(x):
        return [x[b:b + n].view(s) for b, n, s in zip(begins, counts, shapes)]

    st = dict(case=case, begins=begins, counts=counts)
    st["g"] = flat(normal() * size, DTYPES[case["grad"]])
    st["grads"] = views(st["g"])
    if case["op"] != "adamw":
        return st
    weights = flat(normal(), torch.float32)
    st["p"] = weights.to(DTYPES[case["param"]])
    st["params"] = views(st["p"])
    if case["master"]:
        st["master"] = weights
    t = 100 + int(seed) % 50
    st["clocks"] = torch.tensor([[t, B1 ** t, B2 ** t, 0.0]] * len(shapes), dtype=torch.float64, device=dev)
    m = flat(normal() * size * 0.3, torch.float32)
    r = flat(normal().square().mul_(0.3).add_(0.4).sqrt_() * size * 0.3, torch.float32)
    if case["bits"] == 32:
        st["m"], st["v"] = m, r.square()
    else:
        for key, x in (("m", m), ("r", r)):
            b = x.view(-1, BLOCK)
            top = b.abs().amax(1)
            st[key + "_scale"] = top * (1 / 448)
            inv = torch.where(top > 0, 448 / top.clamp_min(1e-30), 0.0)
            st[key] = (b * inv[:, None]).clamp_(-448, 448).to(torch.float8_e4m3fn).view(-1)
            if key == "r":
                floor = ((st[key].float() == 0) & (x > 0))
                st[key] = torch.where(floor, torch.full_like(x, 2.0 ** -9), st[key].float()).to(torch.float8_e4m3fn)
    if own:
        # The optimizer that the user's program keeps, with the state of a run in progress.
        optim = _package()
        opt = optim.AdamW(st["params"], learning_rate=LR, beta1=B1, beta2=B2, eps=EPS, weight_decay=WD,
                          state_bits=case["bits"], master_weights=case["master"],
                          max_grad_norm=case["max_norm"] or None, seed=SEED)
        names = ["clocks"] + (["master"] if case["master"] else [])
        names += ["m", "v"] if case["bits"] == 32 else ["m", "r", "m_scale", "r_scale"]
        opt.load_state_dict({**opt.state_dict(), **{k: st[k] for k in names}})
        for k in names:
            st[k] = opt.state[k]
        st["opt"] = opt
    return st


def _outputs(st, norm):
    keys = ("p", "master", "clocks", "m", "v", "r", "m_scale", "r_scale")
    out = {k: st[k] for k in keys if k in st}
    if norm is not None:
        out["norm"] = norm
    return out


def run(st):
    case = st["case"]
    if own:
        if case["op"] == "adamw":
            return _outputs(st, st["opt"].step(st["grads"]))
        optim = _package()
        if case["op"] == "grad_norm":
            return {"norm": optim.grad_norm(st["grads"])}
        return {"norm": optim.clip_grad_norm_(st["grads"], case["max_norm"]), "g": st["g"]}
    norm = coef = None
    if case["op"] != "adamw" or case["max_norm"]:
        total = torch.stack([g.double().square().sum() for g in st["grads"]]).sum().sqrt()
        norm = total.float()
        if case["max_norm"]:
            coef = (case["max_norm"] / (total + 1e-6)).clamp(max=1.0).float()
    if case["op"] == "grad_norm":
        return {"norm": norm}
    if case["op"] == "clip":
        [g.copy_(g.float() * coef) for g in st["grads"]]
        return {"norm": norm, "g": st["g"]}
    clocks = st["clocks"]
    clocks += torch.cat([torch.ones_like(clocks[:, :1]), clocks[:, 1:2] * (B1 - 1), clocks[:, 2:3] * (B2 - 1),
                         torch.zeros_like(clocks[:, 3:])], 1)
    step = (LR / (1 - clocks[:, 1])).float()
    inv = (1 / (1 - clocks[:, 2]).sqrt()).float()
    [_update(st, i, coef, step[i], inv[i]) for i in range(len(st["counts"]))]
    return _outputs(st, norm)


def _update(st, i, coef, step, inv):
    b, n = st["begins"][i], st["counts"][i]
    n = -(-n // BLOCK) * BLOCK  # the whole slot: what lies behind the tensor is 0 and stays 0
    case, p, g = st["case"], st["p"][b:b + n], st["g"][b:b + n].float()
    if coef is not None:
        g = g * coef
    if case["bits"] == 32:
        m, v = st["m"][b:b + n], st["v"][b:b + n]
        m.copy_(m * B1 + g * (1 - B1))
        v.copy_(v * B2 + g * g * (1 - B2))
        r = v.sqrt()
    else:
        at = slice(b // BLOCK, (b + n) // BLOCK)
        m = (st["m"][b:b + n].float().view(-1, BLOCK) * st["m_scale"][at, None]).view(-1)
        r = (st["r"][b:b + n].float().view(-1, BLOCK) * st["r_scale"][at, None]).view(-1)
        m = m * B1 + g * (1 - B1)
        r = (r * r * B2 + g * g * (1 - B2)).sqrt()
        mq, st["m_scale"][at] = _scaled(m)
        rq, st["r_scale"][at] = _scaled(r)
        st["m"][b:b + n] = mq.clamp(-448, 448).to(torch.float8_e4m3fn)
        st["r"][b:b + n] = _stochastic(rq, _random16(n, i, st["clocks"][i, 0].long())).to(torch.float8_e4m3fn)
    w = st["master"][b:b + n] if case["master"] else p.float()
    w = w * (1 - LR * WD) - m * step / (r * inv + EPS)
    if case["master"]:
        st["master"][b:b + n] = w
    p.copy_(w)


def _scaled(x):
    x = x.view(-1, BLOCK)
    top = x.abs().amax(1)
    top = torch.where(top < 2.0 ** -100, 0.0, top)
    inv = torch.where(top > 0, torch.full_like(top, 448.0) / top, 0.0)
    return (x * inv[:, None]).view(-1), top * (1 / 448)


def _mix(x):
    x = x & MAX32
    x = ((x ^ (x >> 16)) * 0x6A09E667) & MAX32
    x = ((x ^ (x >> 15)) * 0xBB67AE85) & MAX32
    return x ^ (x >> 16)


def _random16(n, i, t):
    """16 random bits for each of n elements of tensor i at step t: halves of one 32-bit word for each two elements."""
    key = _mix(_mix(t) ^ ((SEED + i * GOLDEN) & MAX32))
    block = _mix(key + torch.arange(n // BLOCK, device=t.device))
    word = _mix(block[:, None] + torch.arange(BLOCK // 2, device=t.device) * GOLDEN)
    return torch.stack([word & 0xFFFF, word >> 16], 2).view(-1)


def _stochastic(y, bits):
    """y >= 0 rounded to e4m3's grid (3 bits behind the leading one, steps of 2^-9 below 2^-6), up with the
    probability of its distance from the lower neighbour."""
    y = torch.where(y > 0, y.clamp_min(2.0 ** -9), 0.0)
    low = torch.where(y < 2.0 ** -6, 2.0 ** -6, 0.0)
    word = (y + low).view(torch.int32) + (bits.to(torch.int32) * 16 + 8)
    return ((word & ~0xFFFFF).view(torch.float32) - low).clamp(max=448.0)


def exact(case, seed):
    """The operators in 64 bits."""
    st = prepare(case, seed)
    f64 = torch.float64
    g = st["g"].to(f64)
    norm = torch.linalg.vector_norm(g)
    c = min(1.0, case["max_norm"] / (float(norm) + 1e-6)) if case["max_norm"] else 1.0
    if case["op"] == "grad_norm":
        return {"norm": norm}
    if case["op"] == "clip":
        return {"norm": norm, "g": g.mul_(c)}
    g.mul_(c)
    t = round(float(st["clocks"][0, 0])) + 1
    out = {"clocks": torch.tensor([[t, B1 ** t, B2 ** t, 0.0]] * len(st["counts"]), dtype=f64)}
    if case["max_norm"]:
        out["norm"] = norm
    w = (st["master"] if case["master"] else st["p"]).to(f64)
    if case["bits"] == 32:
        m, v = st["m"].to(f64), st["v"].to(f64)
    else:
        wide = {k: st[k].float().view(-1, BLOCK).to(f64) * st[k + "_scale"].to(f64)[:, None] for k in ("m", "r")}
        m, v = wide["m"].flatten(), wide["r"].flatten().square_()
        del wide
    m.mul_(B1).add_(g, alpha=1 - B1)
    v.mul_(B2).addcmul_(g, g, value=1 - B2)
    del g
    r = v.sqrt()
    if case["bits"] == 32:
        out["m"], out["v"] = m, v
    else:
        # The rounded states have no value in 64 bits where one lies between two codes by less than 32 bits show:
        # their scales have.
        del v
        out["m"] = out["r"] = None
        out["m_scale"], out["r_scale"] = (x.view(-1, BLOCK).abs().amax(1) / 448 for x in (m, r))
    denom = r.div_((1 - B2 ** t) ** 0.5).add_(EPS)
    w = w.mul_(1 - LR * WD).sub_(m.div(denom).mul_(LR / (1 - B1 ** t)))
    out["p"] = w
    if case["master"]:
        out["master"] = w
    return out
