"""The prefetcher's batches stay what they are until their step has run."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_a_batch_is_not_overwritten_while_it_is_used():
    """Steps that the host queues far ahead of the GPU see their own batch."""
    from deeplearning_cfn_amd.data import HostPinnedPrefetcher
    n, size = 60, 1 << 20

    def source():
        for i in range(n):
            yield (torch.full((size,), float(i)),)

    pipe = HostPinnedPrefetcher(source(), torch.device("cuda"))
    busy = torch.randn(2048, 2048, device="cuda")
    low = torch.empty(n, device="cuda")
    high = torch.empty(n, device="cuda")
    for i, (x,) in enumerate(pipe):
        for _ in range(4):
            busy = torch.tanh(busy @ busy)      # the step in front of the use
        low[i], high[i] = x.min(), x.max()
        del x
    want = torch.arange(n, device="cuda", dtype=torch.float32)
    assert torch.equal(low, want) and torch.equal(high, want)
    pipe.close()
