"""Optimizers and gradient clipping, as fused CUDA passes that update in place.

Adam: the step of the example fits (MLXDiffRastExamples/Adam.swift), one
tensor at a time (dr_adam_step).  AdamW, grad_norm and clip_grad_norm_ (no
counterpart in the reference): all leaves of a scene in a launch or two,
in fp32, bf16 or fp16, AdamW's states in 32 or in 8 bits.
"""
from __future__ import annotations

import ctypes
import functools
import math
from typing import Optional, Sequence, Union

import numpy as np
import torch

from . import _lib as L
try:
    from . import _rows
except ImportError as e:
    class _Missing:
        """In place of the extension, which Adam does not need: says why it is missing at its first use."""
        reason = str(e)

        def __getattr__(self, name):
            raise ImportError("AdamW, grad_norm and clip_grad_norm_ need diffrast/_rows, which is missing or of another "
                              f"Python or torch; build it with `python mlx-swift-diffrast_b200/build.py` ({self.reason})")

    _rows = _Missing()
from .ops import _ctx, _f32, _ptr


class Adam:
    """Adam.swift:9-44: state m, v (zeros) and the step count t on the
    instance; bias-corrected update with PyTorch's defaults.  `step` updates
    `param` in place (and returns it); `mask`, if given, multiplies the
    gradient first, as the examples do with their x/y-only position masks."""

    def __init__(self, shape, learning_rate: float = 1e-2, beta1: float = 0.9, beta2: float = 0.999,
                 eps: float = 1e-8, device: Optional[torch.device] = None):
        self.learning_rate = float(learning_rate)
        self.beta1, self.beta2, self.eps = float(beta1), float(beta2), float(eps)
        dev = device if device is not None else torch.device("cuda", torch.cuda.current_device())
        self.m = torch.zeros(tuple(shape), dtype=torch.float32, device=dev)
        self.v = torch.zeros(tuple(shape), dtype=torch.float32, device=dev)
        self.t = 0

    def bias_corrections(self):
        """(1 - beta1^t, 1 - beta2^t) in float32, as the reference's Float pow."""
        b1, b2, t = np.float32(self.beta1), np.float32(self.beta2), np.float32(self.t)
        return float(np.float32(1) - np.power(b1, t)), float(np.float32(1) - np.power(b2, t))

    def step(self, param: torch.Tensor, grad: torch.Tensor, mask: Optional[torch.Tensor] = None) -> torch.Tensor:
        if tuple(param.shape) != tuple(self.m.shape) or tuple(grad.shape) != tuple(self.m.shape):
            raise ValueError(f"adam: param/grad shape must be {tuple(self.m.shape)}")
        if not (param.is_contiguous() and param.dtype == torch.float32):
            raise ValueError("adam: param must be a contiguous float32 tensor (updated in place)")
        g = _f32(grad, "grad")
        mk = _f32(mask.expand_as(param), "mask") if mask is not None else None
        self.t += 1
        c1, c2 = self.bias_corrections()
        c = _ctx(param)
        L.check(L.lib().dr_adam_step(c, _ptr(param), _ptr(g), _ptr(mk), _ptr(self.m), _ptr(self.v), param.numel(),
                                     self.learning_rate, self.beta1, self.beta2, self.eps, c1, c2), c, "adam")
        return param


# ------------------------------------------- lists of tensors (no counterpart)

BLOCK = 256  # elements that share the scale of an 8-bit state

_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}  # dr_dtype
_CUDA = [torch.device("cuda", i) for i in range(64)]

# dr_grad_tensor and dr_adamw_tensor
_GRAD_ROW = np.dtype([("data", "u8"), ("n", "i8"), ("type", "i4"), ("reserved", "i4")])
_ADAMW_ROW = np.dtype([(k, "u8") for k in ("param", "grad", "master", "m", "v", "m_scale", "v_scale", "clock")] +
                      [("n", "i8"), ("lr_ratio", "f8"), ("weight_decay", "f8"), ("seed", "u4"), ("param_type", "i4"),
                       ("grad_type", "i4"), ("reserved", "i4")])


def _dense(t: torch.Tensor) -> bool:
    """Whether t's elements fill one stretch of memory, each once, in any order of its dimensions."""
    if t.is_contiguous():
        return True
    expect = 1
    for stride, size in sorted((st, sz) for st, sz in zip(t.stride(), t.shape) if sz != 1):
        if stride != expect:
            return False
        expect *= size
    return True


def _check_list(tensors, what: str):
    """The tensors as a list, all on one CUDA device, of known types."""
    ts = [tensors] if isinstance(tensors, torch.Tensor) else list(tensors)
    if not ts:
        raise ValueError(f"{what}: no tensors")
    for t in ts:
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{what}: torch.Tensor expected (got {type(t).__name__})")
        if t.layout is not torch.strided:
            raise ValueError(f"{what}: dense tensors expected (got {t.layout})")
        if not t.is_cuda:
            raise ValueError(f"{what}: CUDA tensors expected (the library has no CPU path)")
        if t.dtype not in _TYPES:
            raise ValueError(f"{what}: float32, bfloat16 or float16 expected (got {t.dtype})")
        if t.device != ts[0].device:
            raise ValueError(f"{what}: all tensors must be on one device (got {ts[0].device} and {t.device})")
    return ts


def _check_apart(ts, what: str):
    """Refuses a list in which two tensors share memory: an element would be updated twice."""
    begin = np.array([t.data_ptr() for t in ts], np.uint64)
    size = np.array([t.numel() * t.element_size() for t in ts], np.uint64)
    begin, size = begin[size > 0], size[size > 0]
    order = np.argsort(begin)
    begin, size = begin[order], size[order]
    if (begin[:-1] + size[:-1] > begin[1:]).any():
        raise ValueError(f"{what}: two of the tensors share memory")


def _grad_table(ts):
    tab = np.zeros(len(ts), _GRAD_ROW)
    tab["data"] = [t.data_ptr() for t in ts]
    tab["n"] = [t.numel() for t in ts]
    tab["type"] = [_TYPES[t.dtype] for t in ts]
    return tab


def _written(ts) -> None:
    """Tells autograd that the tensors (or None) were changed in place; inference tensors do not count changes."""
    try:
        torch.autograd.graph.increment_version(ts)
    except (RuntimeError, TypeError):
        torch.autograd.graph.increment_version([t for t in ts if t is not None and not t.is_inference()])


@functools.lru_cache(maxsize=None)
def _context(index: int) -> int:
    """The address of the device's context of this module's lists; binds the library's functions at the first call."""
    c = L.lists_ctx_for(index)
    lib = L.lib()
    _rows.bind(*(ctypes.cast(f, ctypes.c_void_p).value
                 for f in (lib.dr_ctx_set_stream, lib.dr_last_error, lib.dr_grad_norm, lib.dr_clip_grad_norm,
                           lib.dr_adamw_step)))
    return c.value


@functools.lru_cache(maxsize=256)
def _work_len(index: int, count: int) -> int:
    return int(L.lib().dr_grad_norm_work_bytes(_context(index), count)) // 8


def _norm_work(index: int, count: int) -> torch.Tensor:
    return torch.empty(_work_len(index, count), dtype=torch.float64, device=_CUDA[index])


def _norm_call(ts, what: str, max_norm: float, dense) -> torch.Tensor:
    """The norm of the list `ts`; with max_norm > 0 the list is clipped by it.  dense: what the tensors become that are
    not contiguous."""
    found = _rows.grads(ts, max_norm > 0.0)
    if found is None:
        ts = _check_list([t for t in ts if t is not None], what)
        if max_norm > 0.0 and any(t.requires_grad and t.is_leaf for t in ts):
            raise ValueError(f"{what}: gradients expected, not the parameters (a tensor that requires grad was given)")
        ts = [t if t.is_contiguous() else dense(t) for t in ts]
        if max_norm > 0.0:
            _check_apart(ts, what)
        found = ts[0].get_device(), _grad_table(ts).tobytes(), True
    index, rows, large = found
    if torch.cuda.current_device() != index:
        with torch.cuda.device(index):
            return _norm_call(ts, what, max_norm, dense)
    c = _context(index)
    # From torch's allocator at each call: both belong to the stream (or to the
    # graph being captured) and to no other call.
    norm = torch.empty((), dtype=torch.float32, device=_CUDA[index])
    work = _norm_work(index, len(ts)) if large else None
    error = _rows.norm(c, index, rows, max_norm, norm.data_ptr(), None if work is None else work.data_ptr())
    if error:
        L.failed(*error, what)
    return norm


def grad_norm(grads) -> torch.Tensor:
    """The 2-norm over all elements of `grads` (a tensor or a sequence of
    tensors, in any mix of float32, bfloat16 and float16): a float32 scalar on
    their device, the same from run to run.  None, the gradient of a leaf that
    nothing reached, is passed over.  Squares are summed in 64 bits, so the norm
    is finite wherever float32 holds it."""
    ts = [grads] if isinstance(grads, torch.Tensor) else list(grads)
    return _norm_call(ts, "grad_norm", 0.0, lambda t: t if _dense(t) else t.detach().contiguous())


def clip_grad_norm_(grads, max_norm: float) -> torch.Tensor:
    """Scales `grads` (the gradients themselves, as grad_norm takes them; unlike
    torch's function of this name it refuses parameters) in place by
    min(1, max_norm / (norm + 1e-6)) and returns the norm they had.  The factor
    stays on the device, formed from the norm in 64 bits.  A NaN or infinite norm
    gives what the formula does; finite gradients whose norm is beyond float32,
    and returned as infinite, are scaled all the same."""
    ts = [grads] if isinstance(grads, torch.Tensor) else list(grads)
    max_norm = float(max_norm)
    if ts and not 0.0 < max_norm < 1e300:
        raise ValueError(f"clip_grad_norm_: max_norm must be positive and finite (got {max_norm})")

    def dense(t):
        if not _dense(t):
            raise ValueError("clip_grad_norm_: tensors must fill their memory (they are scaled in place)")
        return t

    norm = _norm_call(ts, "clip_grad_norm_", max_norm, dense)
    _written(ts)
    return norm


class AdamW:
    """AdamW over all `params` (a tensor or a sequence of tensors: float32,
    bfloat16, float16, in any mix, on one device) in one launch for each
    combination of types and each 300 tensors of it, updating them in place:

        g = min(1, max_grad_norm / (norm + 1e-6)) * grad      (with max_grad_norm)
        m = beta1 m + (1 - beta1) g;   v = beta2 v + (1 - beta2) g^2
        p = p (1 - lr wd) - lr (m / (1 - beta1^t)) / (sqrt(v) / sqrt(1 - beta2^t) + eps)

    computed in float32 and rounded once to the parameter's type.

    learning_rate: a float, or a float32 CUDA tensor of one element, which each
      step reads on the device (a captured step follows it).  It and
      max_grad_norm may be assigned between steps.
    lr_ratios: one factor of the learning rate for each parameter (default 1).
    weight_decay: one number, or one for each parameter.
    state_bits: 32 (m and v in float32, 8 bytes an element), or 8: m and
      sqrt(v) in e4m3 with a float32 scale for each 256 elements, 2 bytes an
      element.  m is rounded to nearest, sqrt(v) stochastically, by bits that
      depend on `seed`, the parameter's place, t and the element alone: a step
      is reproducible.  A state value that is not finite makes its block of 256
      NaN, and with the next step the block's parameters; a gradient of 2^64 or
      more (1.8e19, after clipping), whose square float32 does not hold, does so
      too and makes its parameter NaN at once.  (32-bit states keep an infinite
      v there, and the parameter stays but for its decay.)
    master_weights: bfloat16 and float16 parameters are kept in float32 too and
      rounded from there; without it, updates below half a step of their type
      are lost.
    max_grad_norm: clip by the norm over all gradients of the step.  A step whose
      norm, as returned, is not finite changes nothing.

    t is counted for each parameter on the device, so a captured step (CUDA
    graph) replays as the next one.  Parameters whose gradient is None are left
    as they are.  Steps of one optimizer must not run at the same time; those
    of different ones may, from any threads and on any streams.  A captured step
    works on this optimizer's buffers: keep it as long as the graph.
    """

    def __init__(self, params, learning_rate: Union[float, torch.Tensor] = 1e-3, beta1: float = 0.9,
                 beta2: float = 0.999, eps: float = 1e-8, weight_decay: Union[float, Sequence[float]] = 1e-2,
                 state_bits: int = 32, master_weights: bool = False, max_grad_norm: Optional[float] = None,
                 lr_ratios: Optional[Sequence[float]] = None, seed: int = 0):
        if state_bits not in (8, 32):
            raise ValueError(f"AdamW: state_bits must be 8 or 32 (got {state_bits})")
        for name, b in (("beta1", beta1), ("beta2", beta2)):
            if not 0.0 <= float(b) < 1.0:
                raise ValueError(f"AdamW: {name} must be in [0, 1) (got {b})")
        if not 2.0 ** -126 <= float(eps) < 1e30:
            raise ValueError(f"AdamW: eps must be at least 2^-126 and finite (got {eps})")
        self.beta1, self.beta2, self.eps = float(beta1), float(beta2), float(eps)
        self.state_bits, self.seed = int(state_bits), int(seed)
        self.learning_rate = learning_rate
        self.max_grad_norm = max_grad_norm
        lr_device = self._step_args()[1]
        self.params = _check_list(params, "AdamW")
        count = len(self.params)
        for p in self.params:
            if p.is_neg():
                raise ValueError("AdamW: a parameter's memory holds it negated (resolve_neg() copies it)")
            if not _dense(p):
                raise ValueError("AdamW: parameters must fill their memory (they are updated in place)")
        _check_apart(self.params, "AdamW")
        if lr_device is not None and lr_device.device != self.params[0].device:
            raise ValueError("AdamW: a learning_rate tensor must be on the parameters' device")
        decays = [float(weight_decay)] * count if np.ndim(weight_decay) == 0 else list(weight_decay)
        ratios = [1.0] * count if lr_ratios is None else list(lr_ratios)
        for name, v in (("weight_decay", decays), ("lr_ratios", ratios)):
            if len(v) != count:
                raise ValueError(f"AdamW: {name} needs {count} values (got {len(v)})")
            if not all(0.0 <= float(x) < 1e30 for x in v):
                raise ValueError(f"AdamW: {name} must be finite and not negative")

        dev = self.params[0].device
        counts = np.array([p.numel() for p in self.params], np.int64)
        slots = -(-counts // BLOCK) * BLOCK
        self._begins = begins = np.concatenate([[0], np.cumsum(slots)[:-1]]).astype(np.int64)
        total = int(slots.sum())
        self._half = [p.dtype != torch.float32 for p in self.params]
        with torch.cuda.device(dev):
            clocks = torch.tensor([[0.0, 1.0, 1.0, 0.0]] * count, dtype=torch.float64, device=dev)
            kind = torch.float32 if self.state_bits == 32 else torch.float8_e4m3fn
            names = ("m", "v") if self.state_bits == 32 else ("m", "r")
            # Each parameter's slot of a buffer begins at a multiple of BLOCK elements.
            self.state = {"clocks": clocks}
            for k in names:
                self.state[k] = torch.zeros(total, dtype=kind, device=dev)
            if self.state_bits == 8:
                for k in names:
                    self.state[k + "_scale"] = torch.zeros(total // BLOCK, dtype=torch.float32, device=dev)
            if master_weights and any(self._half):
                self.state["master"] = torch.zeros(total, dtype=torch.float32, device=dev)
                for i, p in enumerate(self.params):
                    if self._half[i]:
                        self._flat("master", i).copy_(self._memory_order(p.detach()))
            self._ticket = torch.zeros(1, dtype=torch.int32, device=dev)

        tab = np.zeros(count, _ADAMW_ROW)
        state = {k: v.data_ptr() for k, v in self.state.items()}
        one = 4 if self.state_bits == 32 else 1
        tab["m"], tab["v"] = (state[k] + begins * one for k in names)
        if self.state_bits == 8:
            tab["m_scale"], tab["v_scale"] = (state[k + "_scale"] + begins // BLOCK * 4 for k in names)
        if "master" in state:
            tab["master"] = np.where(self._half, state["master"] + begins * 4, 0)
        tab["clock"] = state["clocks"] + np.arange(count) * 32
        tab["n"] = counts
        tab["lr_ratio"], tab["weight_decay"] = ratios, decays
        tab["seed"] = (self.seed + np.arange(count, dtype=np.uint64).astype(object) * 0x9E3779B9) % (1 << 32)
        tab["param_type"] = [_TYPES[p.dtype] for p in self.params]
        self._tab = tab
        # A step updates the memory that it was given: these keep it alive, and
        # the parameters must still be there.
        self._held = [p.detach() for p in self.params] + list(self.state.values())
        self._addresses = tab["param"][:] = [p.data_ptr() for p in self.params]
        self._index, self._device, self._context = dev.index, dev, _context(dev.index)
        with torch.cuda.device(dev):
            # A step's own: steps of one optimizer never run side by side.
            self._work = _norm_work(dev.index, count)
        self._ticket_at, self._work_at = self._ticket.data_ptr(), self._work.data_ptr()
        self._streams = {_rows.stream(dev.index)}
        # What a step's gradients are held against.
        self._shapes = [p.shape for p in self.params]
        self._strides = [p.stride() for p in self.params]
        self._dtypes = [p.dtype for p in self.params]
        # The order of a parameter's elements in memory, which its state follows, where it is not that of its indices.
        self._layouts = [None if p.is_contiguous() else [list(p.shape), list(p.stride())] for p in self.params]

    @staticmethod
    def _memory_order(t: torch.Tensor) -> torch.Tensor:
        """The elements of a dense tensor in the order of their addresses."""
        return t.as_strided((t.numel(),), (1,))

    def _flat(self, name: str, i: int) -> torch.Tensor:
        """Parameter i's part of a state buffer."""
        b = int(self._begins[i])
        if name.endswith("_scale"):
            return self.state[name][b // BLOCK:b // BLOCK - (-self.params[i].numel() // BLOCK)]
        return self.state[name][b:b + self.params[i].numel()]

    def _use_here(self) -> None:
        """The buffers, which the caller does not see, are used on the current stream: once this optimizer is gone,
        their memory waits for that stream as for the one that they were made on."""
        now = _rows.stream(self._index)
        if now not in self._streams:
            self._streams.add(now)
            for t in (*self.state.values(), self._ticket, self._work):
                t.record_stream(torch.cuda.current_stream(self._index))

    def _step_args(self):
        """(lr, its device tensor or None, max_norm), checked."""
        lr, dev, top = self.learning_rate, None, self.max_grad_norm
        if isinstance(lr, torch.Tensor):
            if lr.numel() != 1 or lr.dtype != torch.float32 or not lr.is_cuda or lr.is_neg():
                raise ValueError("AdamW: a learning_rate tensor must be one float32 on the parameters' device")
            lr, dev = 0.0, lr
        elif not 0.0 <= float(lr) < 1e30:
            raise ValueError(f"AdamW: learning_rate must be finite and not negative (got {lr})")
        if top is not None and not 0.0 < float(top) < 1e300:
            raise ValueError(f"AdamW: max_grad_norm must be positive and finite (got {top})")
        return float(lr), dev, 0.0 if top is None else float(top)

    def _gradients(self, grads):
        """The given gradients, as flat memory in the order of their parameters'."""
        out = []
        for i, g in enumerate(grads):
            if g is None:
                out.append(None)
                continue
            if not isinstance(g, torch.Tensor) or g.layout is not torch.strided:
                raise ValueError(f"AdamW: gradient {i} must be a dense tensor")
            if g.shape != self._shapes[i]:
                raise ValueError(f"AdamW: gradient {i} has shape {tuple(g.shape)}, its parameter "
                                 f"{tuple(self._shapes[i])}")
            if g.get_device() != self._index:
                raise ValueError(f"AdamW: gradient {i} is not on its parameter's device")
            p = self._dtypes[i]
            if g.dtype not in _TYPES or not (g.dtype == p or torch.float32 in (p, g.dtype)):
                raise ValueError(f"AdamW: gradient {i} is {g.dtype}, its parameter {p}")
            if g.is_neg():
                g = g.detach().resolve_neg()
            if g.stride() != self._strides[i] and not (g.is_contiguous() and self.params[i].is_contiguous()):
                g = torch.empty_strided(g.shape, self._strides[i], dtype=g.dtype, device=g.device).copy_(g.detach())
            out.append(g)
        return out

    def step(self, grads: Optional[Sequence[Optional[torch.Tensor]]] = None) -> Optional[torch.Tensor]:
        """One step from `grads` (one for each parameter, or None to leave it as
        it is; default: the parameters' .grad).  Gradients have their parameter's
        shape and type, or one of the two is float32; they share no memory with
        parameters.  Returns the norm of the gradients (a float32 scalar
        on the device) with max_grad_norm, else None."""
        if torch.cuda.current_device() != self._index:
            with torch.cuda.device(self._index):
                return self.step(grads)
        ps = self.params
        lr, lr_dev, top = self._step_args()
        if lr_dev is not None and lr_dev.get_device() != self._index:
            raise ValueError("AdamW: a learning_rate tensor must be on the parameters' device")
        norm = torch.empty((), dtype=torch.float32, device=self._device) if top else None
        args = (self._index, self._context, lr, None if lr_dev is None else lr_dev.data_ptr(), self.beta1, self.beta2,
                self.eps, self.state_bits, top, None if norm is None else norm.data_ptr(), self._work_at,
                self._ticket_at)
        at = ps
        self._use_here()  # before the launches, of which one may fail behind another
        error = _rows.step(ps, grads, self._tab, *args)
        if error is False:
            gs = [p.grad for p in ps] if grads is None else list(grads)
            if len(gs) != len(ps):
                raise ValueError(f"AdamW: {len(ps)} gradients expected (got {len(gs)})")
            if [p.data_ptr() for p in ps] != self._addresses:
                raise ValueError("AdamW: a parameter is at another address than when it was given")
            gs = self._gradients(gs)
            keep = [i for i, g in enumerate(gs) if g is not None]
            at, gs, table = [ps[i] for i in keep], [gs[i] for i in keep], self._tab[keep]
            table["grad"] = [g.data_ptr() for g in gs]
            table["grad_type"] = [_TYPES[g.dtype] for g in gs]
            error = _rows.step(None, None, table.tobytes(), *args)
        if error:
            L.failed(*error, "AdamW")
        _written(at)
        return norm

    def moments(self, i: int):
        """Parameter i's first moment m and root of the second, sqrt(v), as float32 in its shape."""
        p = self.params[i]
        out = []
        self._use_here()
        for k in ("m", "v") if self.state_bits == 32 else ("m", "r"):
            x = self._flat(k, i).float()
            if self.state_bits == 8:
                x = x * self._flat(k + "_scale", i).repeat_interleave(BLOCK)[:x.numel()]
            x = x.sqrt() if k == "v" else x.clone()
            out.append(x.as_strided(p.shape, p.stride()))
        return tuple(out)

    def state_dict(self) -> dict:
        """The state's buffers (not copies) and what they were made for: save it, or load it into an optimizer of
        the same parameters."""
        return {**self.state, "state_bits": self.state_bits, "counts": [p.numel() for p in self.params],
                "layouts": self._layouts, "seed": self.seed}

    def load_state_dict(self, state: dict) -> None:
        """Copies a state_dict() into this optimizer's buffers, which keep their addresses: a captured step goes on
        from it.  The master weights are loaded, and the parameters left as they are."""
        if state.get("state_bits") != self.state_bits or list(state.get("counts", ())) != [p.numel() for p in self.params]:
            raise ValueError("AdamW: the state is of other parameters or another state_bits")
        if int(state.get("seed", -1)) != self.seed:
            raise ValueError("AdamW: the state is of another seed")
        if state.get("layouts", self._layouts) != self._layouts:
            raise ValueError("AdamW: the state is of parameters with another order in memory")
        if "master" in state and "master" not in self.state:
            raise ValueError("AdamW: the state has master weights, which this optimizer does not")
        for k, mine in self.state.items():
            x = state.get(k)
            if not isinstance(x, torch.Tensor) or x.shape != mine.shape or x.dtype != mine.dtype:
                raise ValueError(f"AdamW: the state's {k!r} must be {mine.dtype} {tuple(mine.shape)}")
        with torch.cuda.device(self.params[0].device):
            self._use_here()
            for k, mine in self.state.items():
                mine.copy_(state[k])
