"""What an installed package holds: everything its kernels are built from."""

import os
import shutil
import subprocess
import sys
import zipfile

import pytest

from lily_b200.csrc import build


def test_a_wheel_holds_every_source_of_the_kernels(tmp_path):
    pytest.importorskip("setuptools")
    pytest.importorskip("wheel")
    package = os.path.dirname(build.HERE)
    shutil.copytree(package, tmp_path / "lily_b200", ignore=shutil.ignore_patterns("_build", "__pycache__"))
    for name in ("pyproject.toml", "README.md"):
        shutil.copy(os.path.join(os.path.dirname(package), name), tmp_path)
    made = subprocess.run([sys.executable, "-c", "from setuptools import build_meta; print(build_meta.build_wheel('out'))"], cwd=tmp_path, capture_output=True, text=True, timeout=300)
    assert made.returncode == 0, made.stderr[-2000:]
    (wheel,) = (tmp_path / "out").glob("*.whl")
    held = set(zipfile.ZipFile(wheel).namelist())
    for name in [*build.SOURCES, *build.HEADERS, build.FACES]:
        assert f"lily_b200/csrc/{name}" in held, name
    assert not [n for n in held if n.endswith((".so", ".o"))]
