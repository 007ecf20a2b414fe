"""The helper behind the comparisons with the reference's own modules: no tree skips them, a tree without the module does
not."""
import pytest

import refkern


def test_an_absent_tree_skips_with_its_reason(monkeypatch, tmp_path):
    monkeypatch.setattr(refkern, "REF_DIR", str(tmp_path / "none"))
    for call in (lambda: refkern.available("k3_mxfp8"), lambda: refkern.function("k3_mxfp8", "kern_k3_mxfp8_quant")):
        with pytest.raises(pytest.skip.Exception, match="oracle/_ref is absent"):
            call()


def test_a_tree_without_the_module_does_not_skip(monkeypatch, tmp_path):
    monkeypatch.setattr(refkern, "REF_DIR", str(tmp_path))
    assert refkern.available("k3_mxfp8") is False
    (tmp_path / "k3_mxfp8.cubin").touch()
    assert refkern.available("k3_mxfp8") is True
