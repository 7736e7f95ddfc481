"""The filter layout that reduced-precision library convolutions are handed, without a GPU."""
import types

import pytest
import torch

from nextou_amd.network_architecture import channel_pad


@pytest.mark.parametrize("setting", [None, "stored", "contiguous"])
def test_reduced_precision_filters_are_contiguous_whatever_the_environment(monkeypatch, setting):
    """A 16-bit convolution never gets a channels-last filter: a library solver faults the GPU on it."""
    if setting is None:
        monkeypatch.delenv("NEXTOU_REDUCED_PRECISION_FILTERS", raising=False)
    else:
        monkeypatch.setenv("NEXTOU_REDUCED_PRECISION_FILTERS", setting)
    x = torch.randn(2, 8, 4, 4, dtype=torch.bfloat16).contiguous(memory_format=torch.channels_last)
    on_gpu = types.SimpleNamespace(is_cuda=True, dtype=x.dtype, dim=x.dim, stride=x.stride)      # what the rule looks at, of a device tensor
    w = torch.randn(8, 8, 2, 2, dtype=torch.bfloat16).contiguous(memory_format=torch.channels_last)
    got = channel_pad.filter_layout_for(on_gpu, w)
    assert got.is_contiguous() and torch.equal(got, w)
