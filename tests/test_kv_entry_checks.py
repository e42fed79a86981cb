"""What the C entries of the 4-bit cache and of the norms refuse, on the GPU (a
cache handle needs one), and that their kernel files compile by themselves."""

from __future__ import annotations

import subprocess

import pytest
import torch

from se12_b200 import _build


def test_the_4_bit_kernel_files_compile_by_themselves(tmp_path):
    for name in ("se12_kv4.cu", "se12_attend4.cu"):
        run = subprocess.run([_build.nvcc_path(), "-std=c++17", "-gencode", _build.GENCODE, "--cuda", "-o", str(tmp_path / f"{name}.ii"),
                              str(_build.PACKAGE_DIR / "csrc" / name)], capture_output=True, text=True)
        assert run.returncode == 0, f"{name}:\n{run.stdout}{run.stderr}"


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["int8", "int4"])
def test_norms_are_refused_before_anything_runs(kind):
    from se12_b200 import _lib
    from se12_b200.kv_cache import PagedKvCache

    lib = _lib.load()
    x = torch.ones(1, 1, 64, device="cuda")
    out = torch.full((1, 1, 64), 3.0, dtype=torch.bfloat16, device="cuda")
    cache, ints = PagedKvCache(1, 16, 1, 64, kind), torch.ones(1, 1, dtype=torch.int32, device="cuda")
    page = torch.zeros(1, 1, dtype=torch.int32, device="cuda")
    codes = cache.k_codes.clone()
    batch = _lib.KV_BATCH.pack(1, 1, ints.data_ptr(), 0, page.data_ptr(), 1, 1)
    args = _lib.KV_APPEND.pack(False, 1, x.data_ptr(), x.data_ptr(), x.data_ptr(), *[64] * 6, 0, 0, 0, 0, 0, False, out.data_ptr(), 64, 64)
    w = x.data_ptr()

    def call(*norms):
        return lib.se12_kv_append_normed(cache.handle, batch, args, _lib.KV_NORMS.pack(*norms), torch.cuda.current_stream().cuda_stream)

    for norms in ((w + 2, 0, 0, 0, 1e-6), (0, w + 2, 0, 0, 1e-6), (w + 1, 0, 1, 0, 1e-6), (0, w + 1, 0, 1, 1e-6)):
        assert call(*norms) == 3 and b"aligned" in lib.se12_last_error(), norms
    for eps in (-1.0, -1e-300, float("inf"), float("nan")):
        assert call(w, w, 0, 0, eps) == 1 and b"eps" in lib.se12_last_error(), eps
    torch.cuda.synchronize()
    assert bool((out == 3).all()) and torch.equal(cache.k_codes, codes)
    assert call(w, w, 0, 0, 0.0) == 0 and call(w + 2, 0, 1, 0, 1e-6) == 0
    torch.cuda.synchronize()
    assert bool((out != 3).all())
