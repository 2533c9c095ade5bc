"""When the build rebuilds the torch extension module."""

from __future__ import annotations

import os

from qwen_image_shardedit_mlx_b200 import build


def test_extension_is_rebuilt_for_another_torch(tmp_path, monkeypatch):
    ext = tmp_path / "_q6torch.so"
    monkeypatch.setattr(build, "EXT", ext)
    monkeypatch.setattr(build, "BUILD", tmp_path)
    monkeypatch.setattr(build, "LIB", tmp_path / "lib.so")
    assert build._extension_stale()  # not there
    build.LIB.write_bytes(b"")
    ext.write_bytes(b"")
    later = max(p.stat().st_mtime for p in (build.EXT_SOURCE, build.INCLUDE / "q6_b200.h", build.LIB)) + 10
    os.utime(ext, (later, later))
    assert build._extension_stale()  # newer than its sources, but nothing says for which torch
    build._stamp().write_text(build._torch_abi())
    assert not build._extension_stale()
    monkeypatch.setattr(build.importlib.metadata, "version", lambda name: "0.0.0")
    assert build._extension_stale()  # torch was replaced since
    build._stamp().write_text(build._torch_abi())
    assert not build._extension_stale()
    os.utime(ext, (1, 1))
    assert build._extension_stale()  # older than its sources
