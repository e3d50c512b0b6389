"""Corner calls of the serving operators that need no GPU."""

import itertools

import pytest
import torch

from pdattention_b200.ops import _ext

needs_ext = pytest.mark.skipif(not _ext.available(), reason="extension not built")


def views():
    """Tensors [..., heads, head_dim] whose leading dimensions have sizes of 1 with strides of any kind."""
    base = torch.arange(3 * 2 * 3 * 2 * 4).view(3, 2, 3, 2, 4)
    yield base[:, ::2]                                  # [3, 1, 3]: the middle stride is two rows
    yield base[:1].permute(1, 2, 0, 3, 4)               # [2, 3, 1]: the inner stride is the whole tensor
    yield base[:, :1, :1].transpose(0, 2)               # [1, 1, 3]
    yield base[:, :, ::3]                               # [3, 2, 1]
    yield base[:, 1]                                    # [3, 3]
    yield base.transpose(0, 1)                          # no one stride
    yield base[::2].transpose(0, 2)
    yield base[0, 0]
    yield base[:1, :1, :1]
    yield base[0, 0, 0]                                 # a single token without leading dimensions
    yield base[:, :1, 0, :1].expand(3, 4, 1, 4)         # broadcast: stride 0
    yield base[0, 0, :1].expand(5, 2, 4)
    for order in itertools.permutations(range(3)):
        for cut in itertools.product((slice(None), slice(0, 1), slice(None, None, 2)), repeat=3):
            yield base[cut].permute(*order, 3, 4)


@needs_ext
def test_token_stride_ignores_dimensions_of_one():
    found = 0
    for x in views():
        stride = _ext.require().token_stride(list(x.shape), list(x.stride()))
        tokens = x.shape[:-2].numel()
        first = x.reshape(tokens, *x.shape[-2:])[:, 0, 0]  # where each token begins, in elements of the base
        if stride >= 0:
            found += 1
            assert torch.equal(first, first[0] + stride * torch.arange(tokens)), (x.shape, x.stride())
        else:
            steps = first.diff()
            assert not (steps == steps[0]).all()  # there is none
    assert found > 50
