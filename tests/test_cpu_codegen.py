"""Loads in flight of kernels that wait for memory, in the assembly that hipcc makes of this repository's sources with the
build's own flags (gfx950, no GPU needed). How many loads a loop issues before its first wait is the compiler's choice, and
it has changed with a flag before: the kernels' time went with it."""
import os
import re
import shutil
import subprocess

import pytest

PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "face-inpainting-diffusion-models_amd")


def _assembly(src, tmp):
    """{kernel's mangled name: lines} of csrc/<src>.hip"""
    cmd = subprocess.run(["make", "-C", PKG, "-n", "-B", f"build/{src}.o"], capture_output=True, text=True, check=True).stdout
    cc = next(line for line in cmd.splitlines() if " -c " in line and f"csrc/{src}.hip" in line).split()
    if shutil.which(cc[0]) is None:
        pytest.skip(f"{cc[0]} is not installed")
    out = str(tmp / f"{src}.s")
    cc = [out if a == f"build/{src}.o" else "-S" if a == "-c" else a for a in cc] + ["--cuda-device-only"]
    subprocess.run(cc, cwd=PKG, check=True, capture_output=True)
    kernels, name = {}, None
    for line in open(out):
        m = re.match(r"(_Z\w+):", line)
        if m:
            name = m.group(1)
            kernels[name] = []
        elif line.startswith(".Lfunc_end"):
            name = None
        elif name:
            kernels[name].append(line.strip())
    return kernels


def _in_flight(lines):
    """The most loads from global memory issued between two waits for them (or a branch)."""
    best = run = 0
    for s in lines:
        if re.match(r"(global|buffer|flat)_load", s):
            run += 1
            best = max(best, run)
        elif (s.startswith("s_waitcnt") and "vmcnt" in s) or s.startswith(("s_cbranch", "s_branch")):
            run = 0
    return best


def _kernel(kernels, part):
    found = [v for k, v in kernels.items() if part in k]
    assert len(found) == 1, part
    return found[0]


@pytest.fixture(scope="module")
def misc(tmp_path_factory):
    return _assembly("misc", tmp_path_factory.mktemp("asm"))


def test_embedding_layers_keep_16_weight_loads_in_flight(misc):
    assert _in_flight(_kernel(misc, "skinny_kernel")) >= 16


@pytest.fixture(scope="module")
def train_ops(tmp_path_factory):
    return _assembly("train_ops", tmp_path_factory.mktemp("asm"))


def test_attention_backward_of_odd_maps_reads_a_row_at_once(train_ops):
    """Per query row: q, dout and the probabilities and their gradients of eight keys, 18 loads."""
    assert _in_flight(_kernel(train_ops, "attn_bwd_cols_kernel")) >= 18


def test_vertical_resampling_reads_rows_ahead(tmp_path):
    """Four taps: four pixels, and their coefficients in one load."""
    assert _in_flight(_kernel(_assembly("data", tmp_path), "resample_v_kernel")) >= 5
