"""The compiled binding counts as built only for the torch, C++ ABI and interpreter that it was compiled against."""
import pytest

from electrock_infer_b200 import _C, build


def test_a_binding_for_another_torch_is_stale(tmp_path, monkeypatch):
    build.build()
    assert not build.binding_is_stale()
    stamp = tmp_path / "stamp"
    monkeypatch.setattr(build, "BINDING_STAMP", stamp)
    assert build.binding_is_stale()                      # nothing known about it
    stamp.write_text(build.binding_target())
    assert not build.binding_is_stale()
    stamp.write_text(build.binding_target().replace("torch ", "torch 1."))
    assert build.binding_is_stale()


def test_a_binding_for_another_torch_is_not_used(monkeypatch):
    assert _C._native().built_for == build.binding_target()
    monkeypatch.setattr(_C, "_binding", None)
    from electrock_infer_b200 import _binding
    monkeypatch.setattr(_binding, "built_for", "torch 1.0")
    with pytest.raises(RuntimeError, match="electrock_infer_b200.build"):
        _C._native()
    with pytest.raises(RuntimeError, match="torch 1.0"):
        _C.paged_store_kvcache_fp8(None, None, None, None, None, None, None)
