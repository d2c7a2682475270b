"""What Cache8 counts on the host: positions packed, positions that hold a row.  No GPU: the calls are recorded."""
import pytest

from redshift_b200 import Cache8


class Recorder:
    """Stands for HotPath: notes the calls; `capture` says whether the stream of a device is being captured."""

    def __init__(self, capture=False):
        self.calls, self.capture = [], capture

    def capturing(self, *device):
        return self.capture

    def __getattr__(self, name):
        return lambda *args: self.calls.append(name)


def _cache(context=256, **kw):
    return Cache8(Recorder(**kw), context, device='cpu:0')


def _step(cache, batch, position):
    cache.attention(None, None, None, None, None, None, batch, position)


@pytest.mark.parametrize('position', [71, 128, -1, 257])
def test_rows_that_are_not_there_are_not_packed(position):
    """Rows behind the last one are stale or were never written."""
    cache = _cache()
    for at in range(0, 70, 10):
        _step(cache, 10, at)
    before = len(cache.hot.calls), cache.packed, cache.rows
    with pytest.raises(ValueError, match='70 rows'):
        cache.pack(position)
    assert (len(cache.hot.calls), cache.packed, cache.rows) == before
    cache.pack(70)
    assert cache.packed == 64
    _step(cache, 1, 70)


def test_nothing_is_counted_under_capture():
    """A captured call writes no row yet, and its replays would write the tail rows of one position, which hold
    others once the ring has gone on."""
    import torch
    cache = _cache()
    _step(cache, 10, 0)
    cache.hot.capture = True
    rows = torch.zeros((200, 4, 256), dtype=torch.float16)
    for call in (lambda: _step(cache, 1, 10), lambda: cache.load(rows, rows, 130)):
        with pytest.raises(RuntimeError, match='capture'):
            call()
    assert (cache.packed, cache.rows) == (0, 10) and cache.hot.calls == ['attention8']
    cache.hot.capture = False
    with pytest.raises(ValueError, match='leaves a gap'):
        _step(cache, 1, 11)
    _step(cache, 1, 10)
    cache.load(rows, rows, 130)
    assert (cache.packed, cache.rows) == (128, 130)


def test_capture_is_looked_for_on_the_device_of_the_tensors(monkeypatch):
    """The calls run on the current stream of the tensors' device, whichever device is current."""
    import torch
    from redshift_b200 import HotPath
    current = [0]

    class Current:
        def __init__(self, device):
            self.device = device

        def __enter__(self):
            self.before, current[0] = current[0], torch.device('cuda', self.device).index if isinstance(self.device, int) else self.device.index

        def __exit__(self, *_):
            current[0] = self.before
    monkeypatch.setattr(torch.cuda, 'device', Current)
    monkeypatch.setattr(torch.cuda, 'is_current_stream_capturing', lambda: current[0] == 1)
    monkeypatch.setattr(torch._C, '_cuda_getDevice', lambda: current[0], raising=False)
    hot = object.__new__(HotPath)
    assert hot.capturing(1) and hot.capturing(torch.device('cuda', 1))
    assert not hot.capturing(0) and not hot.capturing()
    current[0] = 1
    assert not hot.capturing(0) and hot.capturing(1) and hot.capturing()
    asked = []
    cache = _cache()
    cache.hot.capturing = lambda *device: asked.append(device)
    _step(cache, 10, 0)
    assert asked and all(device == (cache.key_codes.device,) for device in asked)


def test_a_prefill_of_no_tokens_and_rows_of_two_lengths():
    """`rows` may be anything up to the shorter buffer's length, zero with empty buffers among it."""
    import torch
    calls = []

    class Shapes(Recorder):
        def cache8_pack(self, *args):
            calls.append([tuple(a.shape) for a in args[4:6]] + list(args[6:]))

        def cache8_unpack(self, *args):
            calls.append([tuple(a.shape) for a in args[:2]] + list(args[6:]))
    cache = Cache8(Shapes(), 256, device='cpu:0')
    none, short, long = (torch.zeros((n, 4, 256), dtype=torch.float16) for n in (0, 130, 200))
    cache.load(none, none, 0)
    cache.unload(none, none, 0)
    assert calls == [] and (cache.packed, cache.rows) == (0, 0)
    _step(cache, 10, 0)
    cache.load(long, short, 130)
    cache.unload(short, long, 130)
    assert calls == [[(130, 4, 256), (130, 4, 256), 0, 128], [(130, 4, 256), (130, 4, 256), 0, 128]]
    assert (cache.packed, cache.rows) == (128, 130)
    cache.load(none, none, 0)                            # a new conversation
    assert (cache.packed, cache.rows) == (0, 0)
    _step(cache, 1, 0)
