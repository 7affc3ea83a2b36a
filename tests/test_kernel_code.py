"""The device code of the paged attention kernels, as built: what their launches and their products count on.

A matrix instruction's result must not be touched before a number of instruction slots have passed: 8 for
v_mfma_f32_16x16x32_bf16 (16 cycles), 10 for v_mfma_f32_16x16x4_f32 (32 cycles).  The hardware does not wait by itself.
"""
import os
import re
import shutil
import subprocess

import pytest

import gptc

BIN = os.path.join(os.environ.get("ROCM_PATH", "/opt/rocm"), "llvm", "bin")
SLOTS = {"v_mfma_f32_16x16x32_bf16": 8, "v_mfma_f32_16x16x4_f32": 10}

pytestmark = pytest.mark.skipif(not os.path.exists(os.path.join(BIN, "llvm-objdump")), reason="no llvm-objdump")


def tool(name, *args):
    return subprocess.run([os.path.join(BIN, name), *args], check=True, capture_output=True, text=True, timeout=120).stdout


@pytest.fixture(scope="module")
def objects(tmp_path_factory):
    """The library's gfx950 code objects that hold paged attention kernels."""
    if not os.path.exists(gptc.LIB_PATH):
        pytest.skip("the library is not built")
    at = tmp_path_factory.mktemp("code")
    lib = shutil.copy(gptc.LIB_PATH, at / "lib.so")
    tool("llvm-objdump", "--offloading", str(lib))
    found = [str(p) for p in at.iterdir() if "gfx950" in p.name and re.search("paged_(attn|wide)_kernel", tool("llvm-readelf", "-s", "-W", str(p)))]
    assert len(found) == 2
    return found


def registers(text):
    return {(kind, i) for kind, lo, hi in re.findall(r"\b([va])\[?(\d+)(?::(\d+))?", text)
            for i in range(int(lo), int(hi or lo) + 1)}


def kernels(path):
    """(name, instructions, successors): an instruction is its name, its registers, and those it writes if a product."""
    for part in re.split(r"\n(?=[0-9a-f]{16} <)", tool("llvm-objdump", "-d", path))[1:]:
        name = re.match(r"[0-9a-f]+ <(\S+)>:", part).group(1)
        if "paged_attn_kernel" not in name and "paged_wide_kernel" not in name:
            continue
        start, code, at, to = int(part[:16], 16), [], {}, []
        for line in part.splitlines()[1:]:
            m = re.match(r"\s+(\S+)\s*(.*?)\s*// ([0-9A-F]+):.*?(?:<\S+?(?:\+0x([0-9a-f]+))?>)?$", line)
            if m:
                at[int(m.group(3), 16)] = len(code)
                code.append((m.group(1), m.group(2)))
                to.append(start + int(m.group(4), 16) if m.group(4) and "branch" in m.group(1) else None)
        after = [[] if op == "s_endpgm" else [at[t]] if op == "s_branch" else [i + 1] + ([at[t]] if t else [])
                 for i, ((op, _), t) in enumerate(zip(code, to))]
        assert all(t is not None for (op, _), t in zip(code, to) if "branch" in op)
        yield name, code, after


def early_reads(code, after):
    used = [registers(args) for _, args in code]
    for i, (op, args) in enumerate(code):
        if not op.startswith("v_mfma"):
            continue
        result = registers(args.split(",")[0])
        todo, best = [(j, 0) for j in after[i]], {}
        while todo:
            j, slots = todo.pop()
            if j >= len(code) or slots >= SLOTS[op] or best.get(j, 99) <= slots:
                continue
            best[j] = slots
            op2, args2 = code[j]
            if op2.startswith("v_mfma"):
                to, a, b = args2.split(",")[:3]
                early = result & registers(a + b)
                if not early and result & registers(to):
                    continue  # adds to it, or forms the next one there: the hardware keeps these in order
            else:
                early = result & used[j]
            if early:
                yield f"{slots} slots after {op} {args}: {op2} {args2}"
                continue
            slots += 1 + (int(args2, 0) if op2 == "s_nop" else 0)
            todo += [(k, slots) for k in after[j]]


def test_no_result_is_read_early(objects):
    """On any path through a kernel, across branches too."""
    seen, products = 0, set()
    for path in objects:
        for name, code, after in kernels(path):
            products |= {op for op, _ in code if op.startswith("v_mfma")}
            early = list(early_reads(code, after))
            assert not early, (name, early)
            seen += 1
    assert seen == 12 + 27 and products == set(SLOTS)


def test_the_scan_finds_early_reads():
    code = [("v_mfma_f32_16x16x32_bf16", "v[0:3], v[8:11], v[12:15], v[0:3]"), ("s_cbranch_scc0", "2"), ("s_nop", "7"),
            ("v_mul_f32_e32", "v4, v3, v4"), ("s_endpgm", "")]
    assert list(early_reads(code, [[1], [2, 3], [3], [4], []])) == [
        "1 slots after v_mfma_f32_16x16x32_bf16 v[0:3], v[8:11], v[12:15], v[0:3]: v_mul_f32_e32 v4, v3, v4"]
    assert not list(early_reads(code, [[1], [2], [3], [4], []]))


def test_two_workgroups_share_a_cu_where_the_plan_counts_on_it(objects):
    """256 registers a lane are half of a SIMD's: heads up to 64, and all wide kernels."""
    for path in objects:
        for name, count in re.findall(r"\.name:\s+(\S+)\n(?:.*\n)*?\s+\.vgpr_count:\s+(\d+)", tool("llvm-readelf", "--notes", path)):
            if "paged_wide_kernel" in name or re.search(r"paged_attn_kernelI(f|DF16b)Li64E", name):
                assert int(count) <= 256, name
