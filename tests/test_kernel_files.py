"""Every kernel file around the GEMVs names what it uses: it compiles by
itself, not only after the files that happen to come before it in the
library's translation unit."""

from __future__ import annotations

import subprocess

from se12_b200 import _build

FILES = ("se12_kv.cu", "se12_attend.cu", "se12_attend_tile.cu", "se12_logprobs.cu")


def test_each_kernel_file_compiles_by_itself(tmp_path):
    runs = [(name, subprocess.Popen([_build.nvcc_path(), "-std=c++17", "-gencode", _build.GENCODE, "--cuda", "-o",
                                     str(tmp_path / f"{name}.ii"), str(_build.PACKAGE_DIR / "csrc" / name)],
                                    stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)) for name in FILES]
    for name, run in runs:
        output, _ = run.communicate()
        assert run.returncode == 0, f"{name}:\n{output}"
