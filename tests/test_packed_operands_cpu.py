"""Which weights a kept bf16 operand is taken for: the bookkeeping alone, with packing, streams and events replaced by plain
objects."""
import copy
import pickle

import numpy as np
import pytest
import torch


class FakeStream:
    def __init__(self, ident):
        self.ident, self.waited = ident, []

    def wait_event(self, e):
        self.waited.append(e)


class FakeEvent:
    def record(self):
        pass


class FakeOperand:
    def __init__(self, values):
        self.values, self.streams = values, []

    def record_stream(self, s):
        self.streams.append(s)


@pytest.fixture
def world(monkeypatch):
    """current stream and capture state, settable; packing gives the matrix that it was asked to pack"""
    from vc3d import packed
    w = type("World", (), dict(stream=FakeStream(0), capturing=False, packs=0))()

    def pack(m):
        w.packs += 1
        return FakeOperand(m.clone()), FakeOperand(m.clone())
    monkeypatch.setattr(packed, "_matrix_pack", pack)
    monkeypatch.setattr(packed, "cur_stream", lambda: w.stream.ident)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: w.capturing)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda *a: w.stream)
    monkeypatch.setattr(torch.cuda, "Event", FakeEvent)
    return w


def operands():
    from vc3d.lstm import _PackedLSTMWeights
    from vc3d.scan import PackedGateWeight
    return [(PackedGateWeight, 1), (_PackedLSTMWeights, 2)]


def weights_at(memory, count):
    """`count` parameters over one block of memory, as an allocator hands it out again: same address, same version"""
    return [torch.nn.Parameter(torch.from_numpy(memory).view(4, 4)) for _ in range(count)]


@pytest.mark.parametrize("make,count", operands())
def test_unchanged_weights_are_packed_once(world, make, count):
    ws, p = [torch.nn.Parameter(torch.randn(4, 4)) for _ in range(count)], make()
    first = p.get(*ws)
    assert p.get(*ws) is first and world.packs == 1 and not world.stream.waited
    for w in ws:
        with torch.no_grad():
            w.mul_(2)
        again = p.get(*ws)
        assert again is not first and torch.equal(again[0].values, p.matrix(*ws))
        first = again


@pytest.mark.parametrize("make,count", operands())
def test_another_parameter_at_the_same_address_is_another(world, make, count):
    memory, p = np.zeros(16, np.float32), make()
    others = [torch.nn.Parameter(torch.randn(4, 4)) for _ in range(count - 1)]
    (old,) = weights_at(memory, 1)
    p.get(old, *others)
    where, version = old.data_ptr(), old._version
    del old
    memory[:] = 1.0
    (new,) = weights_at(memory, 1)
    assert (new.data_ptr(), new._version) == (where, version)
    assert torch.equal(p.get(new, *others)[0].values, p.matrix(new, *others))


@pytest.mark.parametrize("make,count", operands())
def test_memory_of_kept_weights_is_not_given_to_others(world, make, count):
    """param.data replaced twice may come back to its first address at the same version: not while what was packed is held"""
    ws, p = [torch.nn.Parameter(torch.randn(4, 4)) for _ in range(count)], make()
    p.get(*ws)
    held = ws[0].data_ptr()
    ws[0].data = torch.randn(4, 4)
    assert any(t is not None and t.data_ptr() == held for t in p.kept[2])
    assert torch.equal(p.get(*ws)[0].values, p.matrix(*ws))


@pytest.mark.parametrize("make,count", operands())
def test_another_stream_waits_for_the_packing(world, make, count):
    ws, p = [torch.nn.Parameter(torch.randn(4, 4)) for _ in range(count)], make()
    home, away = world.stream, FakeStream(7)
    ops = p.get(*ws)
    world.stream = away
    assert p.get(*ws) is ops and len(away.waited) == 1 and all(o.streams == [away] for o in ops)
    world.stream = home
    assert p.get(*ws) is ops and not home.waited


@pytest.mark.parametrize("make,count", operands())
def test_a_captured_call_packs_for_itself(world, make, count):
    ws, p = [torch.nn.Parameter(torch.randn(4, 4)) for _ in range(count)], make()
    world.capturing = True
    in_graph = p.get(*ws)  # without a warm-up: nothing has run yet that an eager call could use
    world.capturing = False
    eager = p.get(*ws)
    assert eager is not in_graph and world.packs == 2
    world.capturing = True
    assert p.get(*ws) is not eager and world.packs == 3
    world.capturing = False
    assert p.get(*ws) is eager


@pytest.mark.parametrize("make,count", operands())
def test_a_copy_packs_for_itself(world, make, count):
    ws, p = [torch.nn.Parameter(torch.randn(4, 4)) for _ in range(count)], make()
    p.get(*ws)
    for q in (copy.deepcopy(p), pickle.loads(pickle.dumps(p))):
        assert type(q) is make and q.kept is None
