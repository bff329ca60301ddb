"""Where the reference's library and source are both absent, what compares
with it is skipped with that reason, and does not end a run."""

import unittest

import pytest


def test_an_absent_reference_skips(igo_mod, monkeypatch, tmp_path):
    monkeypatch.setattr(igo_mod, "_REF", None)
    monkeypatch.setattr(igo_mod, "_REF_CUDA", None)
    monkeypatch.setattr(igo_mod, "ref_lib_path", lambda: str(tmp_path / "libref.so"))
    monkeypatch.setattr(igo_mod, "REF_CUDA_PATH", str(tmp_path / "libref_cuda.so"))
    monkeypatch.setattr(igo_mod, "build", lambda: None)
    for load in (igo_mod.ref_lib, igo_mod.ref_cuda_lib):
        with pytest.raises(unittest.SkipTest, match="missing"):
            load()
