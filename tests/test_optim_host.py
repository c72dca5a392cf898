"""The many-tensor optimizer's sources and host side, without a GPU: what holds whatever a machine's timing shows."""
import glob
import importlib.util
import os
import re
import subprocess
import sys
import sysconfig
import textwrap

import pytest

from conftest import ROOT

PKG = os.path.join(ROOT, "mlx-swift-diffrast_b200")

CSRC = os.path.join(PKG, "csrc")


def functions(*names):
    """(signature, body) of each function of these sources, comments taken out."""
    out = []
    for name in names:
        src = re.sub(r"//[^\n]*", "", open(os.path.join(CSRC, name)).read())
        out += re.findall(r"^((?:template[^\n]*\n)?(?:__global__|__device__)[^{;]*)\{\n(.*?)^\}", src, re.S | re.M)
    return out


def test_kernels_launched_early_promise_nothing_of_what_they_wait_for():
    # A kernel that starts while the one before it still writes must not declare the memory read-only (const and
    # restrict): such a load may be non-coherent, and may be moved above the wait.
    found = functions("gradnorm.cu", "adamw.cu", "optim_common.cuh")
    early = [s for s, body in found if "after_previous()" in body or "begin_step<" in body or "norm_of" in s]
    names = " ".join(early)
    for name in ("k_grad_norm_finish", "k_clip_scale", "k_adamw(", "k_adamw8(", "norm_of("):
        assert name in names, name
    for s in early:
        assert "__restrict__" not in s, s


def test_no_other_file_launches_early():
    for path in glob.glob(os.path.join(CSRC, "*")):
        if os.path.basename(path) not in ("gradnorm.cu", "adamw.cu", "optim_common.cuh"):
            assert "griddepcontrol" not in open(path).read() and "launch_early" not in open(path).read(), path


def test_the_clocks_last_block_is_ordered_behind_the_others_reads():
    # Other blocks' plain reads of the clocks and the last block's writes need an order of the memory model's.
    body = {re.sub(r"\(.*", "", s, flags=re.S).split()[-1]: b for s, b in functions("adamw.cu")}
    assert "draw(h.ticket)" in body["end_step"] and "atomicAdd" not in body["end_step"]
    assert "atom.acq_rel.gpu" in body["draw"] and '"memory"' in body["draw"]


@pytest.mark.parametrize("missing", ['sys.modules["diffrast._rows"] = None  # the file',
                                     'del torch.Tensor.__dlpack_c_exchange_api__  # what it asks of torch'])
def test_adam_goes_without_the_extension(missing):
    code = textwrap.dedent("""
        import sys
        import torch
        MISSING
        from diffrast import optim
        opt = optim.Adam((3,), device=torch.device("cpu"))
        assert opt.bias_corrections() is not None
        sys.path.insert(0, "examples")
        import fits
        for call in (lambda: optim.grad_norm([torch.zeros(3)]), lambda: optim.clip_grad_norm_([torch.zeros(3)], 1.0)):
            try:
                call()
            except ImportError as e:
                assert "build.py" in str(e)
            else:
                raise AssertionError("no extension, and no error")
    """).replace("MISSING", missing)
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300, cwd=PKG)
    assert r.returncode == 0, r.stderr


def builder():
    spec = importlib.util.spec_from_file_location("diffrast_build_test", os.path.join(PKG, "build.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


def test_the_extension_is_named_for_its_python():
    from diffrast import optim
    assert os.path.basename(optim._rows.__file__) == "_rows" + sysconfig.get_config_var("EXT_SUFFIX")
    assert os.path.samefile(builder().ROWS, optim._rows.__file__)


def test_a_build_goes_without_pythons_headers(monkeypatch, tmp_path, capsys):
    b = builder()
    monkeypatch.setattr(b.sysconfig, "get_paths", lambda: {"include": str(tmp_path)})
    assert b.build_rows(force=True) is None
    assert "Python.h" in capsys.readouterr().err
