"""Bounds that a caller of the packed cache's attention may give, without a GPU."""

import pytest
import torch

from packed_plain import Cache


@pytest.mark.parametrize("bounds", [{"max_kv_len": -1}, {"max_kv_len": -(1 << 40)}, {"max_q_len": -1}])
def test_negative_bounds_are_refused(monkeypatch, bounds):
    from yalis_b200.ops import packed
    from yalis_b200.ops._lib import KernelError
    monkeypatch.setattr(packed, "_need_here", lambda *a: "cpu")
    pages, table = Cache([40], 2, 64, 16).to("cpu")
    i32 = lambda v: torch.tensor(v, dtype=torch.int32)
    with pytest.raises(KernelError, match="negative"):
        packed.packed_attention(torch.zeros(200, 256), pages, torch.arange(200).int(), i32([0, 200]), table, num_heads=4,
                                **{"max_q_len": 200, **bounds})
