"""What the comments in the kernels' sources promise of the compiled code, read from the objects that the build leaves (no device needed)."""
import os
import re
import subprocess

import pytest

from aicity_action_amd import _hip

LLVM = "/opt/rocm/llvm/bin"
OBJECTS = [os.path.join(os.path.dirname(_hip.LIB_PATH), d) for d in ("obj", "obj_f16")]


def code_object(path, tmp_path):
    """The gfx950 part of an object file."""
    if not os.path.exists(path) or not os.path.exists(LLVM + "/llvm-objdump"):
        pytest.skip("%s is not there: the library was built elsewhere" % path)
    fat, code = str(tmp_path / "fat"), str(tmp_path / "code")
    subprocess.check_call([LLVM + "/llvm-objcopy", "--dump-section", ".hip_fatbin=" + fat, path, os.devnull])
    subprocess.check_call([LLVM + "/clang-offload-bundler", "--unbundle", "--type=o", "--targets=hipv4-amdgcn-amd-amdhsa--gfx950", "--input=" + fat,
                           "--output=" + code])
    return code


def listing(path, tmp_path):
    """Its instructions, in order."""
    text = subprocess.run([LLVM + "/llvm-objdump", "-d", code_object(path, tmp_path)], check=True, capture_output=True, text=True).stdout
    return [line.split("//")[0].strip() for line in text.splitlines() if line.startswith("\t")]


@pytest.mark.parametrize("objects", OBJECTS, ids=os.path.basename)
def test_nothing_but_the_lds_loads_uses_m0_in_newton_schulz(objects, tmp_path):
    """ns_dma writes M0 in inline asm, which cannot name it as overwritten: right as long as the compiler keeps nothing of its own there."""
    code = listing(os.path.join(objects, "newton_schulz.o"), tmp_path)
    loads = 0
    for i, line in enumerate(code):
        if re.search(r"\bm0\b", line):
            assert re.match(r"s_mov_b32 m0, s\d+$", line), line
            assert code[i + 1] == "s_nop 0" and code[i + 2].startswith("global_load_lds_dwordx4 "), code[i:i + 3]
            loads += 1
        assert not re.match(r"[sv]_movrel|s_sendmsg|ds_gws|ds_\w*_gs_|v_interp|buffer_load_\w+ .*\blds\b", line), line
    assert loads == sum(line.startswith("global_load_lds") for line in code) > 0


@pytest.mark.parametrize("objects", OBJECTS, ids=os.path.basename)
@pytest.mark.parametrize("name", ["newton_schulz", "rotary", "rowops", "attention"])
def test_no_packed_fp32_instructions(name, objects, tmp_path):
    for line in listing(os.path.join(objects, name + ".o"), tmp_path):
        assert not re.match(r"v_pk_(add|mul|fma)_f32", line), line


def test_newton_schulz_holds_the_tile_kernels_that_its_dispatch_names(tmp_path):
    """ns_gemm_kernel<tile side, wave groups, stages, phase, split>: variants that no call reaches are not compiled."""
    code = code_object(os.path.join(OBJECTS[0], "newton_schulz.o"), tmp_path)
    names = subprocess.run([LLVM + "/llvm-objdump", "-t", "-C", code], check=True, capture_output=True, text=True).stdout
    found = set(re.findall(r"ns_gemm_kernel<(\d+), (\d+), (\d+), (\d+), (true|false)>", names))
    phases = [str(p) for p in range(6)]           # the products of an iteration, and the last one to 16 bits, fp32 and the weights
    want = {v + (p, s) for p in phases for s in ("true", "false") for v in (("128", "1", "2"), ("64", "1", "2"))}
    want |= {v + (p, "false") for p in phases for v in (("64", "1", "5"), ("64", "2", "5"))}
    want |= {("64", "2", "2", p, "true") for p in phases + ["6"]} | {("64", "1", "2", "7", "true")}       # 6, 7: pieces of long sums
    assert found == want


@pytest.mark.parametrize("half", ["bf16", "fp16"])
def test_hand_packed_records_are_the_library_s(half):
    """The sizes, and each record's fields by what the host side makes of them."""
    import numpy as np

    from aicity_action_amd import muon, rotary
    L = _hip.lib_with_record(half, "mvit_rotary_tensor_bytes", rotary._RECORD.size)
    assert L is _hip.lib(half) and muon._library(half) is L
    with pytest.raises(RuntimeError, match="build it again"):
        _hip.lib_with_record(half, "mvit_ns_matrix_bytes", muon._REC.itemsize - 4)
    # rows and columns: a matrix of 65 rows and 200 columns is no one-workgroup matrix once its columns are far apart, and one of 65 x 2000 never is
    size = lambda *m: L.mvit_newton_schulz_workspace_bytes(np.array([m], dtype=muon._REC).ctypes.data, 1, 0)  # noqa: E731
    assert size(8, 8, 8, 8, 200, 1, 65, 200, 0.0, 0) == 0
    tables = 72 * 256 * 8
    assert size(8, 8, 8, 8, 200, 1 << 28, 65, 200, 0.0, 0) == tables + 2 * (3 * 128 * 256 + 2 * 128 * 128)
    assert size(8, 8, 8, 8, 2000, 1, 65, 2000, 0.0, 0) == tables + 2 * (3 * 128 * 2048 + 2 * 128 * 128)
    assert size(8, 8, 8, 8, 1, 1, 0, 5, 0.0, 0) < 0


def test_the_build_entry_compiles_where_a_library_is_there(monkeypatch):
    import __graft_entry__
    calls = []
    monkeypatch.setattr(_hip.subprocess, "check_call", lambda cmd, **kw: calls.append(cmd))
    __graft_entry__.build()
    assert len(calls) == 1 and calls[0][0] == "make" and "-B" in calls[0]
    _hip.build()                       # the library is newer than its sources now
    assert len(calls) == 1 or "-B" not in calls[1]
