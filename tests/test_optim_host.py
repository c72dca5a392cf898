"""The many-tensor optimizer's sources and host side, without a GPU: what holds whatever a machine's timing shows."""
import glob
import os
import re

from conftest import ROOT

CSRC = os.path.join(ROOT, "mlx-swift-diffrast_b200", "csrc")


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
