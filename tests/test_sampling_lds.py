"""No kernel of csrc/sample_tokens.hip reads LDS ahead of its first barrier: what a wave reads there, the others have written
(the table of powers, by the block's first half wave). From the assembly, which needs the compiler alone."""
import os
import re
import subprocess

import pytest

from q35hip import build


@pytest.fixture(scope="module")
def kernels(tmp_path_factory):
    """{kernel: [mnemonic, ...]} in the order of the text."""
    if not os.path.exists(build.HIPCC):
        pytest.skip("no hipcc")
    out = str(tmp_path_factory.mktemp("asm") / "sample_tokens.s")
    r = subprocess.run([build.HIPCC, *build.CXXFLAGS, "--cuda-device-only", "-S", os.path.join(build.CSRC, "sample_tokens.hip"),
                        "-o", out], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    with open(out) as f:
        text = f.read()
    names = re.findall(r"^\s*\.amdhsa_kernel\s+(\S+)", text, re.M)
    return {n: re.findall(r"^\s+([a-z]\w+)", re.search(rf"^{re.escape(n)}:.*?^\.Lfunc_end", text, re.M | re.S).group(0), re.M)
            for n in names}


def test_lds_is_read_behind_a_barrier(kernels):
    reads = 0
    for name, ops in kernels.items():
        first = next((i for i, op in enumerate(ops) if op.startswith("ds_read")), None)
        if first is not None:
            reads += 1
            assert "s_barrier" in ops[:first], name
    assert reads >= 4 and sum("sample_pick_kernel" in n for n in kernels) == 2
