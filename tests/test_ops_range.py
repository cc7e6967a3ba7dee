"""Stream operators without a GPU: sizes beyond 32 bits, kinds of tensors, gradients, alignment."""
import pytest
import torch

from fast_audiovae import ops

MANY = 2 ** 31


def wide(*shape, dtype=torch.float32):
    """A tensor of any shape that holds one element."""
    return torch.zeros((1,) * len(shape), dtype=dtype).expand(shape)


@pytest.mark.parametrize("call,words", [
    (lambda: ops.causal_conv(wide(MANY, 8), torch.zeros(8, 4)), "too many rows"),
    (lambda: ops.causal_conv(wide(2, MANY // 2, 8), torch.zeros(8, 4)), "too many rows"),
    (lambda: ops.selective_scan(wide(MANY, 8), wide(MANY, 8), torch.zeros(4, 8), wide(MANY, 1, 4), wide(MANY, 1, 4)),
     "too many rows"),
    (lambda: ops.group_norm(wide(MANY, 8), 4), "too many rows"),
    (lambda: ops.group_norm(wide(1, MANY), 4), "too many rows or channels"),
    (lambda: ops.group_norm(torch.zeros(2, 8), 2 ** 32 + 4), "divides the channels"),
    (lambda: ops.project_int4(wide(MANY, 64), torch.zeros(8, 32, dtype=torch.uint8), torch.zeros(8, 2), group=32), "too large"),
    (lambda: ops.project_int4(torch.zeros(2, 64), torch.zeros(8, 32, dtype=torch.uint8), torch.zeros(8, 2),
                              group=2 ** 32 + 32), "scales must be"),
])
def test_sizes_beyond_32_bits_are_refused(call, words):
    with pytest.raises(ValueError, match=words):
        call()
