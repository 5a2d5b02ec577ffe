"""The split-K workspace of a captured conv is the graph's own: bookkeeping without a GPU."""
import torch


def test_a_captured_call_shares_no_workspace(monkeypatch):
    from vc3d import ops
    cpu, now = torch.device("cpu"), [False]
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: now[0])
    monkeypatch.setattr(torch.cuda, "current_stream", lambda *a: type("S", (), dict(cuda_stream=5)))
    monkeypatch.setattr(ops, "_WS", {})
    eager = ops._workspace(None, 0, cpu, need=3 << 20)
    assert ops._workspace(None, 0, cpu, need=1000) == eager  # shared from call to call
    epoch, now[0] = ops.WS_EPOCH, True
    got = [ops._workspace(None, 0, cpu, need=n) for n in (1000, 2000, 5 << 20)]
    assert [n for _, n in got] == [1000, 2000, 5 << 20]
    assert len({int(at) for at, _ in got} | {int(eager[0])}) == 4
    assert all(at.tensor.data_ptr() == at and at.tensor.numel() == n for at, n in got)  # alive as long as its address is
    assert list(ops._WS.values())[0].numel() == 3 << 20 and ops.WS_EPOCH == epoch
    now[0] = False
    assert ops._workspace(None, 0, cpu, need=1000) == eager
    assert ops._workspace(None, 0, cpu, need=0) == (None, 0)
