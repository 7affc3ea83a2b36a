"""The device code of the cross entropy's products, as built: the loads to LDS set m0 by themselves, in inline assembly that
the compiler is not told of (it keeps m0 to itself and takes no such word), so nothing else in these kernels may use it."""
import os
import re
import shutil

import pytest

import gptc
from test_kernel_code import BIN, tool

pytestmark = pytest.mark.skipif(not os.path.exists(os.path.join(BIN, "llvm-objdump")), reason="no llvm-objdump")

LOAD = re.compile(r"(global_load_lds_dwordx4|buffer_load_dwordx4 .* lds)\b")
IMPLICIT = re.compile(r"v_movrel|s_movrel|v_interp|ds_gws|ds_append|ds_consume|s_sendmsg|_load_lds_|\blds\b")


def uses_of_m0(lines):
    """Places where m0 is used for anything but the loads right behind the word that sets it."""
    armed = False
    for line in lines:
        if re.match(r"s_mov_b32 m0, s\d+$", line):
            armed = True
        elif LOAD.match(line):
            if not armed:
                yield line
        elif re.search(r"\bm0\b", line) or IMPLICIT.search(line):
            yield line
        elif not line.startswith("s_nop"):
            armed = False


def test_nothing_else_uses_m0(tmp_path):
    if not os.path.exists(gptc.LIB_PATH):
        pytest.skip("the library is not built")
    lib = shutil.copy(gptc.LIB_PATH, tmp_path / "lib.so")
    tool("llvm-objdump", "--offloading", str(lib))
    seen = {}
    for path in tmp_path.iterdir():
        if "gfx950" not in path.name or not re.search("few_kernel|logits_kernel", tool("llvm-readelf", "-s", "-W", str(path))):
            continue
        for part in re.split(r"\n(?=[0-9a-f]{16} <)", tool("llvm-objdump", "-d", str(path)))[1:]:
            name = re.match(r"[0-9a-f]+ <(\S+)>:", part).group(1)
            lines = [re.sub(r"\s+", " ", line.split("//")[0]).strip() for line in part.splitlines()[1:]]
            if any(LOAD.match(line) for line in lines):
                seen[name] = list(uses_of_m0(lines))
    assert len(seen) == 6 + 1 + 3, sorted(seen)  # few_kernel, logits_kernel, product_kernel
    assert not any(seen.values()), seen


def test_the_scan_finds_other_uses():
    load = "global_load_lds_dwordx4 v1, s[2:3]"
    assert not list(uses_of_m0(["s_mov_b32 m0, s4", "s_nop 0", load, load + " offset:1024", "v_add_f32 v1, v2, v3"]))
    assert list(uses_of_m0(["s_mov_b32 m0, s4", "v_add_f32 v1, v2, v3", load])) == [load]
    assert list(uses_of_m0(["s_mov_b32 m0, -1", "ds_gws_init v0 gds"])) == ["s_mov_b32 m0, -1", "ds_gws_init v0 gds"]
