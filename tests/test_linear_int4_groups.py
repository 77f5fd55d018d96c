"""linear_int4 without group_size: taken where the number of groups says it, refused where it does not."""
import pytest
import torch

from forge import engine


def _call(C, G, **kw):
    rec = dict(weight_packed=torch.zeros(3, (C + 7) // 8, dtype=torch.int32), weight_scale=torch.ones(3, G),
               weight_shape=torch.tensor([3, C]))
    return engine.linear_int4(torch.zeros(2, C, dtype=torch.bfloat16), rec, **kw)


def _on_the_way_to_the_gpu(C, G, **kw):
    """accepted: the next thing that a tensor on the CPU meets is that it is not on a GPU"""
    with pytest.raises(RuntimeError) as e:
        _call(C, G, **kw)
    assert not isinstance(e.value, ValueError)


@pytest.mark.parametrize("C,G,size", [(192, 2, 128), (320, 5, 64), (1000, 2, 512), (96, 2, 64), (160, 2, 128), (480, 4, 128)])
def test_ambiguous_groups_are_refused(C, G, size):
    if C % G or (C // G & (C // G - 1)) == 0:
        _on_the_way_to_the_gpu(C, G)
    else:
        assert -(-C // size) == G                      # the other reading
        with pytest.raises(ValueError, match="pass group_size"):
            _call(C, G)
    _on_the_way_to_the_gpu(C, G, group_size=size)
    _on_the_way_to_the_gpu(C, G, group_size=C // G)


@pytest.mark.parametrize("C,G", [(256, 4), (2048, 16), (7168, 56), (768, 8), (96, 1), (100, 1), (12, 12), (128, 1)])
def test_clear_groups_are_taken(C, G):
    _on_the_way_to_the_gpu(C, G)
