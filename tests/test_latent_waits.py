"""The matrix-core products that the latent kernels issue from inline asm keep
their distances in the built library (the rules and the reader are
test_mfma_waits')."""

import re
import subprocess

import pytest
from test_mfma_waits import OBJDUMP, faults, parse

from instinct_amd import _lib

# Two widths, 1, 2 or 4 waves over heads, two types; two types.
KERNELS = {"latent_decode_kernel": 12, "latent_prefill_wide_kernel": 2}


@pytest.mark.skipif(OBJDUMP is None, reason="no llvm-objdump")
def test_built_kernels(tmp_path):
    library = tmp_path / "lib.so"
    library.symlink_to(_lib.LIBRARY_PATH)
    subprocess.run([OBJDUMP, "--offloading", library.name], cwd=tmp_path, check=True,
                   stdout=subprocess.DEVNULL)
    seen = dict.fromkeys(KERNELS, 0)
    for image in sorted(tmp_path.glob("*gfx950*")):
        code = image.read_bytes()
        if not any(kernel.encode() in code for kernel in KERNELS):
            continue
        text = subprocess.run([OBJDUMP, "-d", image.name], cwd=tmp_path, check=True,
                              capture_output=True, text=True).stdout
        for name, body in re.findall(r"^[0-9a-f]+ <(\S+)>:\n(.*?)(?=^[0-9a-f]+ <|\Z)", text,
                                     re.S | re.M):
            for kernel in KERNELS:
                if kernel in name:
                    found, products = faults(parse(body.splitlines()))
                    assert not found, f"{name}: {found[:4]}"
                    seen[kernel] += products > 0
    assert seen == KERNELS
