"""What the many-tensor optimizer refuses, and its host-side pieces, without a
GPU: argument checks of AdamW, grad_norm and clip_grad_norm_, the density and
overlap checks, the C entries' checks, and the oracle's own arithmetic."""
import ctypes
import os
import re

import numpy as np
import pytest
import torch

import adamw_oracle as AO
from conftest import ROOT
from diffrast import _lib, optim


@pytest.mark.parametrize("kw,text", [
    (dict(state_bits=16), "state_bits"), (dict(state_bits=4), "state_bits"),
    (dict(beta1=1.0), "beta1"), (dict(beta1=-0.1), "beta1"), (dict(beta2=float("nan")), "beta2"),
    (dict(eps=0.0), "eps"), (dict(eps=1e-60), "eps"), (dict(eps=float("inf")), "eps"), (dict(eps=-1.0), "eps"),
    (dict(learning_rate=-1.0), "learning_rate"), (dict(learning_rate=float("nan")), "learning_rate"),
    (dict(learning_rate=torch.ones(1)), "learning_rate"),
    (dict(max_grad_norm=0.0), "max_grad_norm"), (dict(max_grad_norm=float("nan")), "max_grad_norm"),
    (dict(max_grad_norm=float("inf")), "max_grad_norm"),
])
def test_adamw_refuses_bad_numbers(kw, text):
    with pytest.raises(ValueError, match=text):
        optim.AdamW([torch.zeros(3)], **kw)


def test_lists_are_checked():
    for f in (optim.grad_norm, lambda x: optim.clip_grad_norm_(x, 1.0), optim.AdamW):
        with pytest.raises(ValueError, match="no tensors"):
            f([])
        with pytest.raises(ValueError, match="CUDA"):
            f([torch.zeros(3)])
        with pytest.raises(TypeError, match="Tensor"):
            f([np.zeros(3)])
        with pytest.raises(ValueError, match="dense"):
            f([torch.zeros(3, 3).to_sparse()])


def test_dense():
    x = torch.zeros(4, 6, 8)
    for t in (x, x.permute(2, 0, 1), x.transpose(0, 2), x[:, :, None], x[0], torch.zeros(()), torch.zeros(0, 3)):
        assert optim._dense(t)
    for t in (x[:, :3], x[::2], x.expand(2, 4, 6, 8), x[..., 1:], torch.zeros(1).expand(5), x.as_strided((4, 4), (1, 1))):
        assert not optim._dense(t)


def test_shared_memory_is_refused():
    x = torch.zeros(100)
    optim._check_apart([x[:50], x[50:], torch.zeros(3)], "x")
    optim._check_apart([x[:0], x, x[5:5]], "x")
    for ts in ([x, x], [x[:51], x[50:]], [x, torch.zeros(2), x[10:20]]):
        with pytest.raises(ValueError, match="share memory"):
            optim._check_apart(ts, "x")


def test_rows_match_the_header():
    # The numpy rows are the C structs, field by field.
    src = open(os.path.join(ROOT, "include", "diffrast.h")).read()
    size = {"int64_t": 8, "double": 8, "uint32_t": 4, "int32_t": 4}
    for name, row in (("dr_grad_tensor", optim._GRAD_ROW), ("dr_adamw_tensor", optim._ADAMW_ROW)):
        body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), src, re.S).group(1)
        body = re.sub(r"/\*.*?\*/", "", body, flags=re.S)
        at = 0
        fields = re.findall(r"(?:const )?(\w+)\s*(\*?)\s*(\w+);", body)
        assert [f[2] for f in fields] == list(row.names)
        for kind, star, field in fields:
            n = 8 if star else size[kind]
            assert at % n == 0 and row.fields[field][1] == at and row.fields[field][0].itemsize == n
            at += n
        assert row.itemsize == at


def test_c_entries_refuse_a_null_context():
    L = _lib.lib()
    assert L.dr_grad_norm_work_bytes(None, 4) == 0
    assert L.dr_grad_norm(None, None, 0, None, None) == _lib.DR_EINVAL
    assert L.dr_clip_grad_norm(None, None, 0, 1.0, None, None) == _lib.DR_EINVAL
    assert L.dr_adamw_step(None, None, 0, 0.0, None, 0.9, 0.999, 1e-8, 32, 0.0, None, None, None) == _lib.DR_EINVAL


# --------------------------------------------------------------- the oracle

def test_oracle_codes_are_torchs():
    codes = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).float().numpy()
    np.testing.assert_array_equal(AO.e4m3_table(), codes)


def test_oracle_step_against_torch():
    g = np.random.default_rng(3)
    p = g.normal(size=50)
    ref = torch.from_numpy(p.copy()).requires_grad_(True)
    opt = torch.optim.AdamW([ref], lr=1e-2, betas=(0.9, 0.99), eps=1e-6, weight_decay=0.1)
    m, r = np.zeros(50), np.zeros(50)
    for t in range(1, 6):
        grad = g.normal(size=50)
        ref.grad = torch.from_numpy(grad.copy())
        opt.step()
        (p, m, v), _ = AO.step(p, grad, m, r, t, 1e-2, 0.9, 0.99, 1e-6, 0.1)
        r = np.sqrt(v)
        np.testing.assert_allclose(p, ref.detach().numpy(), rtol=1e-12)


def test_random_bits_are_even_and_apart():
    # 2^18 draws of 16 bits: a mean's standard deviation is 2^16 / sqrt(12 * 2^18) = 37, a bin's (of 256, 1024 draws
    # each) about 32; six of them bound every one of the few hundred values looked at.
    n = 1 << 18
    a, b, c = AO.random16(n, 7, 1), AO.random16(n, 7, 2), AO.random16(n, 8, 1)
    for x in (a, b, c):
        assert abs(x.mean() - 32767.5) < 6 * 37
        assert np.abs(np.bincount(x >> 8, minlength=256) - 1024).max() < 6 * 32
    for x, y in ((a, b), (a, c), (a[:-1], a[1:]), (a[:-256], a[256:]), (a[::2], a[1::2])):
        assert abs(np.corrcoef(x, y)[0, 1]) < 6 / np.sqrt(len(x))


def test_oracle_rounds_to_a_neighbour_without_bias():
    g = np.random.default_rng(5)
    y = np.concatenate([g.uniform(0, 448, 200), 448 * 2.0 ** -g.uniform(0, 17, 200), [0.0, 448.0, 2.0 ** -9]])
    got = np.stack([AO.stochastic(y, g.integers(0, 1 << 16, y.size))[0] for _ in range(4000)])
    lo, hi = AO.neighbours(y)
    keep = y >= 2.0 ** -9  # less, but not 0, becomes 2^-9
    assert ((got == lo) | (got == hi))[:, keep].all() and (got[:, (y > 0) & ~keep] == 2.0 ** -9).all()
    off = np.abs(got.mean(0) - y)[keep] / (hi - lo + (hi == lo))[keep]
    assert off.max() < 6 * 0.5 / np.sqrt(4000)
    assert (got[:, y == 0] == 0).all() and (got[:, y == 448] == 448).all()
