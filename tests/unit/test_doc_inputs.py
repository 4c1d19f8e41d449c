"""Document bounds of inference tensors, with the kernel replaced by a record (CPU)."""

import importlib

import torch

from mint_b200.ops import _ext

attention = importlib.import_module("mint_b200.ops.attention")  # the package has a function of that name


class FakeKernels:
    def __init__(self):
        self.calls = 0

    def doc_bounds(self, d):
        self.calls += 1
        return torch.full((*d.shape, 2), self.calls)


def test_inference_tensors_are_taken_and_not_kept(monkeypatch):
    fake = FakeKernels()
    monkeypatch.setattr(_ext, "require", lambda: fake)
    with torch.inference_mode():
        ids = torch.zeros(1, 8, dtype=torch.int32)
        assert int(attention._doc_inputs(ids)[1][0, 0, 0]) == 1
        ids[0, 4:] = 1
        assert int(attention._doc_inputs(ids)[1][0, 0, 0]) == 2  # computed from the ids as they are now
    ids = torch.zeros(1, 8, dtype=torch.int32)
    a, b = attention._doc_inputs(ids), attention._doc_inputs(ids)
    assert fake.calls == 3 and a[1] is b[1]
    ids[0, 4:] = 1
    assert int(attention._doc_inputs(ids)[1][0, 0, 0]) == 4
