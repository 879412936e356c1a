"""What the serving kernels' built code and host code hold, without a GPU: the
prompt attention kernels' loads into LDS have landed where a barrier publishes
them, on every path, and the serving operators' host tests pass under
AddressSanitizer and UndefinedBehaviorSanitizer."""
import os
import re
import shutil
import subprocess
import sys

import pytest

from test_direct_lds_waits import LIB, LLVM, code_objects, unwaited_barriers
from test_sanitized_host import ORACLE, ROOT, SAN_FMX, SAN_ORACLE, asan_runtime


@pytest.fixture(scope="module")
def tile_kernels(tmp_path_factory):
    """{symbol: [(address, mnemonic, operands, branch target or None)]} of the
    kernels whose loads go straight into LDS, as the few-row products' test reads
    its own."""
    if not LIB.exists():
        from freemoe_amd import build
        build.build()
    found = {}
    for code in code_objects():
        if b"attention_tiles_kernel" not in code:
            continue
        obj = tmp_path_factory.mktemp("code") / "code.elf"
        obj.write_bytes(code)
        text = subprocess.run([LLVM / "llvm-objdump", "-d", "--no-show-raw-insn", obj], check=True, text=True,
                              capture_output=True).stdout
        base, body = {}, None
        for line in text.splitlines():
            head = re.match(r"^([0-9a-f]+) <(.+)>:$", line)
            if head:
                base[head[2]] = int(head[1], 16)
                body = found.setdefault(head[2], []) if "attention_tiles_kernel" in head[2] else None
                continue
            ins = body is not None and re.match(r"^\s+(\S+)\s*(.*?)\s*// ([0-9A-F]+):(.*)$", line)
            if ins:
                to = re.search(r"<([^>+]+)(?:\+0x([0-9a-f]+))?>", ins[4])
                target = base[to[1]] + int(to[2] or "0", 16) if to and "branch" in ins[1] else None
                body.append((int(ins[3], 16), ins[1], ins[2], target))
    return {name: code for name, code in found.items() if code}


def publishing(code):
    """The code with only the barriers that publish loads: those right behind a
    wait for vector memory. (A reduction over the workgroup, where values that
    are not finite are looked for, has barriers of its own, which later blocks'
    loads may pass.)"""
    return [ins if ins[1] != "s_barrier" or code[i - 1][1] == "s_waitcnt" and "vmcnt" in code[i - 1][2]
            else (ins[0], "s_nop", "0", None) for i, ins in enumerate(code)]


def test_prompt_attention_waits_for_its_direct_lds_loads(tile_kernels):
    assert len(tile_kernels) >= 20  # three types, one or several parts, four widths, pages that split loads or not
    for name, code in tile_kernels.items():
        kept = publishing(code)
        assert sum("load_lds" in ins[1] for ins in kept) > 0 and sum(ins[1] == "s_barrier" for ins in kept) >= 2, name
        assert unwaited_barriers(kept) == set(), name


def test_publishing_keeps_the_barriers_behind_waits():
    code = [(0, "global_load_lds_dwordx4", "", None), (4, "s_barrier", "", None), (8, "s_waitcnt", "lgkmcnt(0)", None),
            (12, "s_barrier", "", None), (16, "s_waitcnt", "vmcnt(0) lgkmcnt(0)", None), (20, "s_barrier", "", None),
            (24, "global_load_lds_dwordx4", "", None), (28, "global_load_lds_dwordx4", "", None),
            (32, "s_waitcnt", "vmcnt(2) lgkmcnt(0)", None), (36, "s_barrier", "", None),
            (40, "s_waitcnt", "vmcnt(1) lgkmcnt(0)", None), (44, "s_barrier", "", None), (48, "s_endpgm", "", None)]
    assert [ins[0] for ins in publishing(code) if ins[1] == "s_barrier"] == [20, 36, 44]
    assert unwaited_barriers(publishing(code)) == {44}


def test_serving_host_code_under_asan_and_ubsan():
    rt = asan_runtime()
    if rt is None or shutil.which("make") is None or not os.path.exists("/opt/rocm/bin/hipcc"):
        pytest.skip("clang's sanitizer runtime or hipcc is not in this image")
    build = subprocess.run(["make", "-C", str(ORACLE), "-j8", "sanitize"], capture_output=True, text=True, timeout=1200)
    assert build.returncode == 0, build.stderr[-4000:]
    env = dict(os.environ, LD_PRELOAD=str(rt), FMX_LIBRARY=str(SAN_FMX), FMORACLE_LIBRARY=str(SAN_ORACLE),
               ASAN_OPTIONS="detect_leaks=0:abort_on_error=1", UBSAN_OPTIONS="halt_on_error=1:print_stacktrace=1")
    run = subprocess.run([sys.executable, "-m", "pytest", "-x", "-q", "-p", "no:cacheprovider", "-m", "not gpu",
                          "tests/test_serving_host.py"], cwd=ROOT, env=env, capture_output=True, text=True, timeout=1200)
    report = run.stdout[-3000:] + run.stderr[-3000:]
    assert run.returncode == 0, report
    assert "ERROR: AddressSanitizer" not in report and "runtime error:" not in report, report
