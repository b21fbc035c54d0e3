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


def test_what_is_no_tensor_is_a_type_error():
    """Beside kept activations as beside tensors."""
    kept = lambda m, n: nn.Kept8(torch.zeros(m * (-(-n // 32)) * 33, dtype=torch.uint8), (m, n), torch.bfloat16)  # noqa: E731
    dy, w, v = (torch.zeros(n, dtype=torch.bfloat16) for n in ((4, 16), (40, 16), (40,)))
    for call, words in ((lambda: nn.linear_grad(None, kept(4, 40), w), "dy is not a tensor"),
                        (lambda: nn.linear_grad([1.0], kept(4, 40), w), "dy is not a tensor"),
                        (lambda: nn.linear_grad(dy, kept(4, 40), None), "w is not a tensor"),
                        (lambda: nn.linear_grad(dy, None, w, kept(4, 16), "gelu"), "x is not a tensor"),
                        (lambda: nn.linear_grad(kept(4, 16), kept(4, 40), w), "dy is not a tensor"),
                        (lambda: nn.linear_grad(dy, kept(4, 40), kept(40, 16)), "w is not a tensor"),
                        (lambda: nn.rms_norm_grad(None, kept(4, 40), v), "dy is not a tensor"),
                        (lambda: nn.rms_norm_grad(kept(4, 40), kept(4, 40), v), "dy is not a tensor"),
                        (lambda: nn.rms_norm_grad(torch.zeros(4, 40).bfloat16(), kept(4, 40), 1.0), "weight is not a tensor"),
                        (lambda: nn.keep8([1.0, 2.0]), "x is not a tensor"),
                        (lambda: nn.keep8(kept(4, 40)), "x is not a tensor"),
                        (lambda: nn.linear(kept(4, 40), w), "x is not a tensor"),
                        (lambda: nn.linear_cross_entropy(kept(4, 40), w, torch.zeros(4, dtype=torch.int64)), "x is not a tensor")):
        with pytest.raises(TypeError, match=words):
            call()
