"""tools/ holds measurements and offline analysis: no script brings a failed GPU build back, and the index in
tools/README.md names files that are there."""
from __future__ import annotations

import re
from pathlib import Path

TOOLS = Path(__file__).resolve().parents[1] / "tools"
SUFFIXES = (".sh", ".py", ".c", ".cpp", ".hip", ".patch")


def _sources():
    # (path below tools/, text with continued shell lines joined)
    for p in sorted(TOOLS.rglob("*")):
        if p.is_file() and p.suffix in SUFFIXES:
            yield p.relative_to(TOOLS).as_posix(), p.read_text().replace("\\\n", " ")


def test_no_script_loads_a_code_object_over_the_compiled_kernels():
    # the run-time kernels a script runs are the ones the tree compiles, never a code object kept from a miscompiled
    # build; nor does a script run the checkout (_old) that such a build was made in
    pat = re.compile(r"RT_JIT_LOAD\w*|/_old\b")
    bad = [f"{name}: {m.group(0)}" for name, text in _sources() for m in pat.finditer(text)]
    assert not bad, bad


def test_index_names_files_that_exist():
    # a name without a folder stands in the folder of the name before it on its line, as the index writes its rows
    missing = []
    for line in (TOOLS / "README.md").read_text().splitlines():
        if not line.startswith("|"):
            continue
        folder = ""
        for token in re.findall(r"`([^`]+)`", line.split("|")[1]):
            for word in token.split():
                if not word.endswith(SUFFIXES):
                    continue
                if "/" in word:
                    folder, word = word.rsplit("/", 1)
                at = TOOLS / folder
                if at.is_dir() and not list(at.glob(word)):
                    missing.append(f"{folder}/{word}")
    assert not missing, missing


def test_scene20_probe_runs_default_builds_only():
    # dbg20.py compares frames of the 10k-sphere scene with the oracle under environment variants given as "label|ENV=V".
    # A 6-wave build of that scene faulted the GPU, so scripts run the probe on the default build alone ("label|"): no
    # forced register budget, no code compiled out, no other library
    bad = []
    for name, text in _sources():
        if not name.endswith(".sh"):
            continue
        for line in text.splitlines():
            if line.lstrip().startswith("#") or "dbg20.py" not in line:
                continue
            before, after = line.split("dbg20.py", 1)
            variants = re.findall(r'"([^"|]*)\|([^"]*)"', after)
            if "RT_HIP_LIB" in before or not variants or any(env for _, env in variants):
                bad.append(f"{name}: {line.strip()[:90]}")
    assert not bad, bad
