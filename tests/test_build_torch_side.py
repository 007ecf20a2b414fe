"""When the compiled torch side counts as built."""
import os
import time

import pytest

import k3moe_build as kb


@pytest.fixture
def built(monkeypatch, tmp_path):
    monkeypatch.setattr(kb, "TORCH_OUT", str(tmp_path / "k3moe_torch.so"))
    monkeypatch.setattr(kb, "TORCH_STAMP", str(tmp_path / "k3moe_torch.stamp"))
    (tmp_path / "k3moe_torch.so").touch()
    (tmp_path / "k3moe_torch.stamp").write_text(kb.torch_stamp())
    return tmp_path


def test_of_this_torch(built):
    assert kb.torch_up_to_date()


def test_of_another_torch(built):
    """Its sources are older than it, and still it has to be built again."""
    (built / "k3moe_torch.stamp").write_text("torch 1.0, cpython-38\n")
    assert not kb.torch_up_to_date()
    (built / "k3moe_torch.stamp").unlink()
    assert not kb.torch_up_to_date()


def test_older_than_its_sources(built):
    then = time.time() - 10 * 365 * 86400
    os.utime(built / "k3moe_torch.so", (then, then))
    assert not kb.torch_up_to_date()
    (built / "k3moe_torch.so").unlink()
    assert not kb.torch_up_to_date()
