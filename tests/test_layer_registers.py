"""The registers of every kernel in the built library, whichever source it was compiled from: the library holds an offload bundle for each."""
import os
import re
import shutil
import struct
import subprocess

import pytest

from conftest import ROOT

READELF = shutil.which("llvm-readelf") or "/opt/rocm/llvm/bin/llvm-readelf"


def code_objects(path, target=b"gfx950"):
    """Of each bundle - magic, number of entries, then offset, size and name of each - what is for the target."""
    with open(path, "rb") as f:
        data = f.read()
    found = []
    for match in re.finditer(b"__CLANG_OFFLOAD_BUNDLE__", data):
        start = match.start()
        at = start + 32
        for _ in range(struct.unpack_from("<Q", data, start + 24)[0]):
            offset, size, length = struct.unpack_from("<QQQ", data, at)
            if target in data[at + 24:at + 24 + length]:
                found.append(data[start + offset:start + offset + size])
            at += 24 + length
    return found


@pytest.mark.skipif(not os.path.exists(READELF), reason="no llvm-readelf")
def test_no_kernel_of_any_source_spills_but_the_allocation(tmp_path):
    kernels = []
    for n, code in enumerate(code_objects(os.path.join(ROOT, "gact-icml_amd", "gact", "lib", "libgact_hip.so"))):
        held = tmp_path / ("code%d.o" % n)
        held.write_bytes(code)
        notes = subprocess.run([READELF, "--notes", str(held)], check=True, capture_output=True, text=True).stdout
        kernels += notes.split("- .agpr_count")[1:]
    field = lambda kernel, name: re.search(r"\.%s:\s+(\S+)" % name, kernel).group(1)  # noqa: E731
    names = [field(k, "name") for k in kernels]
    # both sources
    assert sum("quantize_strips_kernel" in n for n in names) == 42
    assert sum("product_kernel" in n for n in names) > 50 and sum("norm_backward_kernel" in n for n in names) > 30
    # one workgroup, and nothing waits for its bandwidth: 16 candidates a thread
    spilled = {n: field(k, "vgpr_spill_count") for n, k in zip(names, kernels) if field(k, "vgpr_spill_count") != "0"}
    assert [n for n in spilled if "calc_precision" not in n] == []
    # and no kernel of the layers has memory of its own, which an array that is indexed at run time would be
    assert [n for n, k in zip(names, kernels) if "GLOBAL__N_1" in n and field(k, "private_segment_fixed_size") != "0"] == []
