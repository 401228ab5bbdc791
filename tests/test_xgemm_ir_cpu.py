"""The cross entropy's products as the compiler sees them: LDS bytes that hold values of one type after another's are only
accessed in ways that may alias."""
import os
import re
import subprocess

import pytest

from psgd_pro_amd import build as B


@pytest.fixture(scope="module")
def ir(tmp_path_factory):
    """LLVM IR of xgemm.hip's device code."""
    out = tmp_path_factory.mktemp("ir") / "xgemm.ll"
    subprocess.run([B.HIPCC, *B.COMMON, *B.DEVICE_FLAGS, "--cuda-device-only", "-S", "-emit-llvm", os.path.join(B.CSRC, "xgemm.hip"),
                    "-o", str(out)], check=True, capture_output=True)
    return out.read_text()


def test_no_lds_access_is_bound_to_a_type(ir):
    """A tile's references and targets (float, int) lie where its 16-bit results go: with accesses tagged by those types the
    compiler might let the reads sink below the results' writes. A tag of the character type, or none, aliases everything."""
    names = dict(re.findall(r'^!(\d+) = !\{!"([^"]*)"', ir, re.M))
    access = dict(re.findall(r"^!(\d+) = !\{!(\d+), !\d+, i64 \d+\}", ir, re.M))
    lds = [line for line in ir.splitlines() if re.search(r"\b(load|store)\b.*ptr addrspace\(3\)", line)]
    assert len(lds) > 500  # fragments, references, targets, results
    tagged = {names[access[t]] for line in lds for t in re.findall(r"!tbaa !(\d+)", line)}
    assert tagged <= {"omnipotent char"}, tagged
