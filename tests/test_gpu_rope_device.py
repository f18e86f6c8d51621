"""The rotation table of a prefix on another device than the current one is built with that device current."""
import pytest
import torch

from starkv import RopeConfig, _lib, rope_table

pytestmark = pytest.mark.gpu


def test_table_is_built_on_its_own_device(monkeypatch):
    inside, seen = [], []
    device = torch.cuda.device

    class Recorded(device):
        def __enter__(self):
            inside.append(self.idx)
            return super().__enter__()

        def __exit__(self, *a):
            inside.pop()
            return super().__exit__(*a)

    build = _lib.lib().starkv_rope_build
    monkeypatch.setattr(torch.cuda, "device", Recorded)
    monkeypatch.setattr(_lib.lib(), "starkv_rope_build", lambda *a: seen.append(list(inside)) or build(*a))
    rope_table(RopeConfig(theta=4321.0), 100, torch.device("cuda", 0))
    assert seen == [[0]]
