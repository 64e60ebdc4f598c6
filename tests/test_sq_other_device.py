"""SQRows on a device that is not the current one: a large write takes scratch of
its own where the stream that it runs on is captured, whatever the current
device's stream does.  torch.cuda is a fake of two devices here (no GPU)."""
import types

import pytest
import torch

import insitu_b200 as ib


class FakeCuda:
    """the current device, and which devices' current streams are being captured"""

    def __init__(self, current, captured):
        self.current, self.captured, self.made = current, captured, []

    def device(self, device):
        fake = self

        class Scope:
            def __enter__(self):
                self.before, fake.current = fake.current, device.index

            def __exit__(self, *_):
                fake.current = self.before

        return Scope()

    def install(self, monkeypatch):
        monkeypatch.setattr(torch.cuda, "current_device", lambda: self.current)
        monkeypatch.setattr(torch.cuda, "device", self.device)
        monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: self.current in self.captured)
        monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda index: 100 + index, raising=False)
        monkeypatch.setattr(torch, "empty", lambda *a, **k: self.made.append(object()) or Scratch())


class Scratch:
    def data_ptr(self):
        return 4096


def store(device):
    rows = ib.SQRows.__new__(ib.SQRows)
    rows.L = types.SimpleNamespace(ivf_sq_write=None)
    rows._codes = rows._scales = Scratch()
    rows.capacity, rows.d, rows.bits, rows.group = 1000, 32, 8, 0
    rows.device, rows._ldc, rows._lds = device, 32, 1
    rows._claim = rows._claim_stream = None
    rows._rows = lambda x: (Scratch(), 32, 600, 0)
    rows._slots = lambda slots, n: Scratch()
    return rows


@pytest.mark.parametrize("current", [0, 1])
@pytest.mark.parametrize("captured", [(), (0,), (1,), (0, 1)])
def test_scratch_follows_the_stores_stream(monkeypatch, current, captured):
    fake = FakeCuda(current, captured)
    fake.install(monkeypatch)
    monkeypatch.setattr(ib, "_sq_call", lambda *a: None)
    rows = store(torch.device("cuda", 1))
    rows.write("rows", "slots")
    assert (rows._claim is None) == (1 in captured)      # a captured write's scratch is not kept
    assert len(fake.made) == 1 and fake.current == current
    rows.write("rows", "slots")
    assert len(fake.made) == (2 if 1 in captured else 1)
