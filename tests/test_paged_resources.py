"""What the compiler reports of the paged serving kernels: none keeps an array on
the private stack, and only those that fill their registers (heads of 256, 17 rows
and more) a few words of addresses."""
import re
import subprocess

import pytest

from conftest import ROOT


@pytest.mark.parametrize("source", ["paged.hip", "verify.hip"])
def test_private_stack(source):
    from spock_amd import build
    r = subprocess.run([build.HIPCC, *build.FLAGS, "-Rpass-analysis=kernel-resource-usage", "--cuda-device-only", "-c",
                        str(ROOT / "spock_amd" / "csrc" / source), "-o", "/dev/null"], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-2000:]
    names = re.findall(r"Function Name: (\S+)", r.stderr)
    sizes = [int(x) for x in re.findall(r"ScratchSize \[bytes/lane\]: (\d+)", r.stderr)]
    assert names and len(names) == len(sizes)
    full = re.compile(r"paged_(mid|tiles)_kernelILi256E")
    assert not {n: s for n, s in zip(names, sizes) if s > (32 if full.search(n) else 0)}
