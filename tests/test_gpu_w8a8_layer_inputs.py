"""The 8-bit layer on inputs as a model hands them over."""

import pytest
import torch

from conftest import announce

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_layer_on_slices(dev, dtype):
    """Slices along tokens, channels and batch, transposed and expanded inputs: the bits of a contiguous copy."""
    from nunchaku_amd.models import W8A8Linear

    torch.manual_seed(4)
    m = W8A8Linear.from_linear(torch.nn.Linear(64, 40, dtype=dtype), device=dev)
    hidden = torch.randn(3, 12, 192, dtype=dtype).to(dev)
    cases = {
        "tokens": torch.randn(2, 12, 64, dtype=dtype).to(dev)[:, :7],
        "tokens and channels": hidden[:, 2:9, 64:128],
        "channels": hidden[..., 64:128],
        "every other batch entry": hidden[::2, :, :64],
        "channels off 16 bytes": hidden[..., 4:68],
        "rows off 16 bytes": torch.randn(3, 12, 68, dtype=dtype).to(dev)[..., :64],
        "transposed": torch.randn(64, 9, dtype=dtype).to(dev).t(),
        "tokens first": torch.randn(12, 3, 64, dtype=dtype).to(dev).transpose(0, 1),
        "one row for all": hidden[0, :1, :64].expand(5, -1),
        "one entry for all": hidden[:1, :, :64].expand(4, -1, -1),
        "one token": hidden[0, 0, 4:68],
        "no token": hidden[:, :0, :64],
    }
    for name, x in cases.items():
        announce(f"layer on {name} {dtype}")
        y = m(x)
        assert y.shape == (*x.shape[:-1], 40) and y.dtype == dtype
        assert torch.equal(y, m(x.clone(memory_format=torch.contiguous_format))), name


def test_slices_in_a_graph(dev):
    """The copy that a slice needs is part of a captured graph: replays see new inputs."""
    from nunchaku_amd.models import W8A8Linear

    announce("slices in a graph")
    torch.manual_seed(5)
    m = W8A8Linear.from_linear(torch.nn.Linear(64, 40, dtype=torch.bfloat16), device=dev)
    hidden = torch.randn(2, 12, 64, dtype=torch.bfloat16).to(dev)
    m(hidden[:, :7])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = m(hidden[:, :7])
    for turn in range(3):
        hidden.mul_(-1.5)
        want = m(hidden[:, :7])
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
