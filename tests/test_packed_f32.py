"""No HIP code of this library holds a packed f32 instruction (v_pk_add_f32, v_pk_mul_f32, v_pk_fma_f32): some of their
operand forms have given wrong results on the MI355X now and then, with no error, so every build turns the feature off.
Read from the code objects built here; no device is needed."""
from __future__ import annotations

import re
import shutil
import subprocess
from pathlib import Path

import pytest

import torch  # noqa: F401  first, as in every process that renders

import cuda_raytracing_amd as rt
from cuda_raytracing_amd import _abi

PACKED = re.compile(r"\bv_pk_(?:add|mul|fma)_f32\b")


def _objdump():
    tool = shutil.which("llvm-objdump") or "/opt/rocm/lib/llvm/bin/llvm-objdump"
    if not Path(tool).exists():
        pytest.skip("llvm-objdump not available")
    return tool


def _disassemble(path):
    out = subprocess.run([_objdump(), "-d", "--mcpu=gfx950", str(path)], capture_output=True, text=True, check=True).stdout
    assert "s_endpgm" in out, f"{path}: no kernel in the listing"
    return out


def _packed(isa):
    return [ln.strip() for ln in isa.splitlines() if PACKED.search(ln)]


def test_offline_kernels_hold_no_packed_f32(tmp_path):
    lib = tmp_path / "lib.so"                       # the tool writes the bundles it extracts next to its input
    shutil.copy(_abi.HIP_LIB, lib)
    subprocess.run([_objdump(), "--offloading", str(lib)], capture_output=True, check=True, cwd=tmp_path)
    objects = [p for p in tmp_path.iterdir() if "gfx950" in p.name]
    assert len(objects) == 1, sorted(p.name for p in tmp_path.iterdir())
    bad = _packed(_disassemble(objects[0]))
    assert not bad, bad[:5]


# slp "1": the vectoriser that forms f32 pairs is let loose (RT_JIT_SLP); the pairs still end up in scalar instructions
@pytest.mark.parametrize("slp", ["0", "1"])
@pytest.mark.parametrize("scene,trav,mb", [(0, rt.RT_TRAV_STATIC, 16), (17, rt.RT_TRAV_STATIC, 50),
                                           (20, rt.RT_TRAV_ACCEL, 16), (3, rt.RT_TRAV_MIXED, 40),
                                           (0, rt.RT_TRAV_LANE, 8)])
def test_run_time_kernels_hold_no_packed_f32(tmp_path, monkeypatch, scene, trav, mb, slp):
    monkeypatch.setenv("RT_JIT_CACHE_DIR", "0")
    monkeypatch.setenv("RT_JIT_DUMP", str(tmp_path))
    monkeypatch.setenv("RT_JIT_SLP", slp)
    w, _ = rt.build_scene(scene)
    rt.kernel_build(w.scene(), trav, mb)
    objects = list(tmp_path.glob("*.co"))
    assert objects, "no code object dumped"
    bad = [ln for co in objects for ln in _packed(_disassemble(co))]
    assert not bad, bad[:5]
