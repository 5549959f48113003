"""What the drafted step refuses, without a GPU: types that are not the kernels' own, arrays that overlap."""
import pytest
import torch

from tests.test_draft_host import P, be, refused, step  # noqa: F401


def test_rope_vecs_of_another_type(be):
    """Two bytes wide is not bf16: halves and integers would be turned as the bf16 that their bits spell."""
    x = torch.zeros((3, 4, 64), dtype=torch.bfloat16)
    be.rope_vecs(x, torch.zeros_like(x))
    for t in (torch.float16, torch.int16):
        for bad in ((x.to(t),), (x, x.to(t)), (x.to(t), x)):
            with pytest.raises(ValueError):
                be.rope_vecs(*bad)
