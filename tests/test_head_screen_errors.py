"""What the screens say to a GPU that is not there, or that is too small: one line and exit status 2."""

import pytest
import torch

from triton_kubernetes_amd.ops import cli


@pytest.mark.parametrize("command", ["loss", "gemv"])
def test_a_device_that_does_not_exist(command, capsys, monkeypatch):
    monkeypatch.setattr(torch.cuda, "is_available", lambda: True)
    monkeypatch.setattr(torch.cuda, "device_count", lambda: 2)
    assert cli.main([command, "--device", "2"]) == 2
    assert capsys.readouterr().err.strip() == "tk-gpu: no GPU 2 (there are 2)"


class _Here:
    """torch.cuda.device on a machine without one."""

    def __init__(self, dev):
        pass

    def __enter__(self):
        pass

    def __exit__(self, *error):
        pass


@pytest.mark.parametrize("command", ["loss", "gemv"])
def test_sizes_that_the_memory_does_not_hold(command, capsys, monkeypatch):
    def full(*args, **kwargs):
        raise torch.OutOfMemoryError("out of memory. Tried to allocate 1024.00 GiB.\nMore lines")

    monkeypatch.setattr(torch.cuda, "is_available", lambda: True)
    monkeypatch.setattr(torch.cuda, "device_count", lambda: 1)
    monkeypatch.setattr(torch.cuda, "device", _Here)
    monkeypatch.setattr(torch, "Generator", full)
    assert cli.main([command]) == 2
    err = capsys.readouterr().err.strip().splitlines()
    assert len(err) == 1 and err[0].startswith("tk-gpu: the GPU's memory does not hold")
