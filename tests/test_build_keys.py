"""A library is rebuilt when a file that it is compiled from changes, and the module of the host's calls is held to the launchers' prototypes."""
import os
import re
import shutil
import subprocess

import pytest

from qwen_decoder_b200.csrc import build


@pytest.fixture
def sources(tmp_path, monkeypatch):
    """A copy of the sources, which the build then goes by."""
    to = tmp_path / "csrc"
    shutil.copytree(build.CSRC, to, ignore=shutil.ignore_patterns("_build", "__pycache__"))
    monkeypatch.setattr(build, "CSRC", str(to))
    return to


def included(folder, name, seen=None):
    """The files of the folder that ``name`` includes, and those that they do."""
    seen = set() if seen is None else seen
    for f in re.findall(r'^\s*#include "([^"]+)"', (folder / name).read_text(), re.M):
        if f not in seen and (folder / f).exists():
            seen.add(f)
            included(folder, f, seen)
    return seen


@pytest.mark.parametrize("name", sorted(build.LIBRARIES))
def test_a_library_is_rebuilt_when_what_it_includes_changes(name, sources):
    nvcc = build.find_nvcc()
    before = build._key(name, nvcc)
    assert before == build._key(name, nvcc)
    for f in sorted(included(sources, build.LIBRARIES[name]) | {build.LIBRARIES[name]}):
        text = (sources / f).read_text()
        (sources / f).write_text(text + "// changed\n")
        assert build._key(name, nvcc) != before, f
        (sources / f).write_text(text)


@pytest.mark.skipif(shutil.which("g++") is None, reason="no g++")
def test_a_prototype_that_drifts_does_not_compile(sources):
    """The host's calls go by ``entry_points.h``: with a pointer or a length of a launcher changed there they are an error."""
    source = os.path.join(build.CSRC, build.LIBRARIES["host_calls"])
    command = [a for a in build._extension_command(source, os.devnull) if not a.startswith(("-l", "-Wl", "-shared", "-O"))] + ["-fsyntax-only", "-w"]
    header = sources / "entry_points.h"
    text = header.read_text()
    assert subprocess.run(command, capture_output=True).returncode == 0
    for before, after in (("int qd_rows_fp8(const void* x, int dtype, long long ldx,", "int qd_rows_fp8(const void* x, int dtype, const void* ldx,"),
                          ("int qd_token_logprobs(const void* logits, int dtype,", "int qd_token_logprobs(const void* logits,")):
        assert before in text
        header.write_text(text.replace(before, after))
        assert subprocess.run(command, capture_output=True).returncode != 0, after
