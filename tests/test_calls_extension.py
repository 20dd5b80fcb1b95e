"""The CPython extension of the ordinary 4-bit calls can be missing, of another PyTorch or broken: the library still
builds, and the calls go through ctypes (CPU)."""

import subprocess

import pytest
import torch

from mini_infra_b200 import _native as nat
from mini_infra_b200 import build as build_mod
from mini_infra_b200 import ops


@pytest.mark.parametrize("broken", [False, True])
def test_calls_go_through_ctypes_where_there_is_no_extension(monkeypatch, tmp_path, broken):
    path = tmp_path / "_mi_calls.so"
    if broken:
        path.write_bytes(b"not a shared object")
    monkeypatch.setattr(nat, "calls_path", lambda: path)
    monkeypatch.setattr(nat, "_calls", None)
    with pytest.warns(RuntimeWarning, match="ctypes"):
        calls = nat.calls()
    assert nat.calls() is calls
    for name in ("kv4_paged_decode", "kv4_append", "kv4_store_chunks", "kv4_gather_blocks", "kv_copy_blocks"):
        assert getattr(calls, name)(1, 2, 3) is None
    x = torch.zeros((1, 2, 64), dtype=torch.bfloat16)
    pool = torch.zeros((2, 2, ops.kv4_page_bytes(16, 64)), dtype=torch.uint8)
    with pytest.raises(RuntimeError, match="CUDA tensors"):  # the ordinary path's own refusal
        ops.kv4_scatter(x, x, None, None, torch.zeros(1, dtype=torch.long), pool, pool)


def test_another_pytorch_has_another_extension(monkeypatch):
    here = build_mod.calls_path()
    monkeypatch.setattr(torch, "__version__", "99.0")
    assert build_mod.calls_path() != here and build_mod.calls_path().parent == here.parent


@pytest.mark.parametrize("error", [FileNotFoundError("g++"), subprocess.CalledProcessError(1, "g++")])
def test_the_library_builds_where_the_extension_does_not(monkeypatch, tmp_path, error):
    ran = []

    def run(cmd, check):
        ran.append(cmd)
        raise error

    monkeypatch.setattr(build_mod, "calls_path", lambda: tmp_path / "_mi_calls.so")
    monkeypatch.setattr(build_mod, "needs_build", lambda: False)
    monkeypatch.setattr(build_mod.subprocess, "run", run)
    with pytest.warns(RuntimeWarning, match="ctypes"):
        assert build_mod.build() == build_mod.LIB_PATH
    assert len(ran) == 1 and not (tmp_path / "_mi_calls.so").exists()


@pytest.mark.skipif(not build_mod.calls_path().exists(), reason="built without the extension")
def test_the_extension_that_was_built_loads():
    assert not isinstance(nat.calls(), nat._NoCalls)
