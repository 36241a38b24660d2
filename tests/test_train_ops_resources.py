"""Registers, scratch memory and the store hazard of csrc/train_ops.hip (CPU test, as test_kernel_resources.py for the other
translation unit): no kernel there spills, and the streaming kernels keep the waves that hide their latency."""
import os
import re
import shutil
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")

# demangled prefix -> least waves per SIMD
WAVES = {
    "void norm_fwd_kernel<float, 1, ": 8,
    "void norm_fwd_kernel<unsigned short, 1, ": 8,
    "void norm_bwd_kernel<float, 1, ": 8,
    "void norm_bwd_kernel<unsigned short, 1, ": 5,
    "void norm_bwd_kernel<float, 4, 0, 512": 2,
    "void norm_bwd_kernel<unsigned short, 2, 0, 512": 3,
    "void lp_rows_kernel<": 8,
    "void lp_rows_bwd_kernel<": 8,
    "void lp_short_rows_bwd_kernel<": 8,
    "void lp_pixels_kernel<": 8,
    "void lp_pixels_bwd_kernel<": 8,
    "void adamw_kernel<": 5,
}


@pytest.fixture(scope="module")
def listing(tmp_path_factory):
    if not os.path.exists(HIPCC) or shutil.which("c++filt") is None:
        pytest.skip("hipcc / c++filt not available")
    from erfnet_pytorch_amd import _lib
    out = tmp_path_factory.mktemp("res") / "train_ops.s"
    text = subprocess.run([HIPCC, "--offload-arch=gfx950", "-O3", "-std=c++17", *_lib.DEVICE_FLAGS, "--cuda-device-only", "-S",
                           "-Rpass-analysis=kernel-resource-usage", "-o", str(out),
                           os.path.join(ROOT, "erfnet_pytorch_amd", "csrc", "train_ops.hip")],
                          capture_output=True, text=True, timeout=900).stderr
    assert out.exists(), text[-2000:]
    recs = re.findall(r"Function Name: (\S+).*?ScratchSize \[bytes/lane\]: (\d+).*?Occupancy \[waves/SIMD\]: (\d+)", text, re.S)
    names = subprocess.run(["c++filt"], input="\n".join(r[0] for r in recs), capture_output=True, text=True).stdout.split("\n")
    return {n: (int(o), int(s)) for n, (_, s, o) in zip(names, recs)}, str(out)


def test_no_kernel_spills(listing):
    kernels, _ = listing
    assert len(kernels) > 60
    assert not {n: s for n, (_, s) in kernels.items() if s}


@pytest.mark.parametrize("prefix", sorted(WAVES))
def test_kernels_keep_their_waves(listing, prefix):
    hits = {n: o for n, (o, _) in listing[0].items() if n.startswith(prefix)}
    assert hits, prefix
    assert not {n: o for n, o in hits.items() if o < WAVES[prefix]}


def test_no_wide_store_is_followed_by_a_write_of_its_data(listing):
    r = subprocess.run([sys.executable, os.path.join(ROOT, "scripts", "scan_store_hazard.py"), listing[1]],
                       capture_output=True, text=True, timeout=600)
    assert r.returncode == 0, r.stdout[-2000:] + r.stderr[-2000:]
    text = open(listing[1]).read()
    assert not re.search(r"\bv_pk_(add|mul|fma)_f32\b", text)
