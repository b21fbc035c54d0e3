"""Without a GPU: what the calls on kept activations refuse."""

import pytest
import torch

from tensorforge_amd import _lib
from tensorforge_amd import tforge_nn as nn


def test_masked_refusals():
    lib = _lib.lib()
    for args, words in (((256, 64, 4, 64, 3, 0, 256), "type = 3"), ((256, 63, 4, 64, 1, 0, 256), "x: 63 elements"), ((256, 64, 4, 64, 1, 2, 256), "positive = 2"),
                        ((256, 64, 4, 64, 1, 0, 264), "not 16-byte aligned"), ((None, 64, 4, 64, 1, 0, 256), "x is a null pointer")):
        assert lib.tf_keep8_masked(*args, None) == -4
        got = lib.tf_last_error().decode()
        assert got.startswith("tf_keep8_masked: ") and words in got, got
    assert lib.tf_keep8_masked(None, 0, 0, 64, 1, 0, None, None) == 0
    x = torch.zeros(4, 40, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="not on a GPU"):
        nn.keep8(x, masked=True)
    with pytest.raises(ValueError, match="no gradient"):
        nn.keep8(x.requires_grad_(), masked=True)
