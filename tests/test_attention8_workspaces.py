"""The workspaces that HotPath.attention8 keeps, one for each stream that it was called on."""
import numpy as np
import pytest

from redshift_b200 import HotPath

from .test_attention8 import Layer


def test_only_so_many_workspaces_are_kept(monkeypatch):
    import torch
    stream, made = [0], []
    monkeypatch.setattr(torch._C, '_cuda_getCurrentRawStream', lambda device: stream[0], raising=False)
    hot = HotPath()
    monkeypatch.setattr(hot, 'attention8_workspace', lambda device: made.append(stream[0]) or object())
    first = hot.kept_workspace8(0)
    assert hot.kept_workspace8(0) is first and hot.kept_workspace8(1) is not first
    for stream[0] in range(1, 100):
        one = hot.kept_workspace8(0)
        assert hot.kept_workspace8(0) is one
        assert len(hot._workspaces8) <= hot.KEPT_WORKSPACES8
    assert made == [0, 0] + list(range(1, 100))
    for stream[0] in range(99, 99 - hot.KEPT_WORKSPACES8, -1):      # the newest ones are still there
        hot.kept_workspace8(0)
    assert len(made) == 101


@pytest.mark.gpu
def test_calls_on_many_streams(hot):
    """More streams than workspaces are kept, one behind the other, twice over."""
    import torch
    many = HotPath()
    layers = [Layer(1 + i % 3, 500 + 64 * i, 448 + 64 * i, 128, 9800 + i) for i in range(4)]
    want = [layer.run(hot).copy() for layer in layers]
    streams = [torch.cuda.Stream() for _ in range(many.KEPT_WORKSPACES8 + 8)]
    outs, before = [], torch.cuda.current_stream()
    for _ in range(2):
        for i, stream in enumerate(streams):
            layer = layers[i % 4]
            layer.out = torch.full_like(layer.out, float('nan'))
            stream.wait_stream(torch.cuda.current_stream())
            stream.wait_stream(before)
            before = stream
            with torch.cuda.stream(stream):
                layer.again(many)
            outs.append((layer.out, want[i % 4]))
    torch.cuda.synchronize()
    assert many.status() == 0 and len(many._workspaces8) <= many.KEPT_WORKSPACES8
    assert all(np.array_equal(out.cpu().numpy(), w) for out, w in outs)
