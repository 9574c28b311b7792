"""Packed weights that Engine.ctpt_project_ takes, without a GPU: as many bytes as the
matrix needs, one after the other in memory, before anything is passed on."""
import types

import pytest
import torch


def test_packed_weights_have_to_be_there(pkg):
    passed = []
    e = types.SimpleNamespace(gemm_weight_bytes=lambda n_in, n_out, limbs: 64 * n_in * n_out * limbs, hp=0, device=0,
                              _check=lambda rc: None,
                              K=types.SimpleNamespace(ctpt_project=lambda *a: passed.append(a)))
    x, y, g = [None] * 3, [None] * 2, [0, 1]
    whole = torch.zeros(64 * 12, dtype=torch.uint8)
    for packed in (whole, torch.zeros(1000, dtype=torch.uint8), whole.view(12, 64), whole.view(torch.int32)):
        passed.clear()
        pkg.Engine.ctpt_project_(e, y, x, packed, g)
        assert len(passed) == 1
    passed.clear()
    for packed in (whole[:-1], whole[:1].expand(64 * 12), whole.view(64, 12).t(), torch.zeros(2 * 64 * 12, dtype=torch.uint8)[::2],
                   whole[:64 * 3].view(torch.int32)):
        with pytest.raises(ValueError):
            pkg.Engine.ctpt_project_(e, y, x, packed, g)
    assert not passed
