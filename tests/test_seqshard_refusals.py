"""What sequence sharding refuses, without a GPU."""
import pytest
import torch

from holonomyawareattention_b200 import PathOrderedGeometricMHA, seqshard


def test_gradients_are_refused():
    """The sharded forward is not differentiable: its kernels would leave all but the last linear without gradients."""
    m = PathOrderedGeometricMHA(32, n_heads=4)
    x = torch.zeros(1, 8, 32)
    with pytest.raises(NotImplementedError, match="forward-only"):
        seqshard.sequence_sharded_forward(m, x)
    with torch.no_grad(), pytest.raises(NotImplementedError, match="CUDA"):
        seqshard.sequence_sharded_forward(m, x)
    m.requires_grad_(False)
    with pytest.raises(NotImplementedError, match="CUDA"):
        seqshard.sequence_sharded_forward(m, x)
    with pytest.raises(NotImplementedError, match="forward-only"):
        seqshard.sequence_sharded_forward(m, x.requires_grad_())
