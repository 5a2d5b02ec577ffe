"""The gate projection's packed operands where calls share them: streams, graphs, weights that change in between."""
import copy

import pytest
import torch

pytestmark = pytest.mark.gpu


def cell_of(F, H, seed):
    from models.recurrence import GatedScan
    torch.manual_seed(seed)
    return GatedScan(F, H).cuda()


def expected(cell, x):
    """what a module without any history computes"""
    with torch.no_grad():
        out = copy.deepcopy(cell).sequence(x)
    torch.cuda.synchronize()
    return out


def equal(got, want):
    return all(torch.equal(a, b) for a, b in zip(got, want))


def test_sequences_on_two_streams_after_a_change_of_weights():
    """the first call packs behind 50 ms of other work on its stream; the second, on another stream, may not overtake it"""
    cell, g = cell_of(128, 64, 1), torch.Generator().manual_seed(2)
    xs = [torch.randn(3, 40, 128, generator=g).cuda() for _ in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    for step in range(3):
        with torch.no_grad():
            cell.gates.weight.normal_()
        want = [expected(cell, x) for x in xs]
        with torch.no_grad():
            with torch.cuda.stream(streams[step % 2]):
                torch.cuda._sleep(100_000_000)
                first = cell.sequence(xs[0])
            with torch.cuda.stream(streams[1 - step % 2]):
                second = cell.sequence(xs[1])
        torch.cuda.synchronize()
        assert equal(first, want[0]) and equal(second, want[1]), step


@pytest.mark.parametrize("warm", [True, False])
def test_a_captured_sequence_follows_the_weights(warm):
    """replays with what the weights hold then, eager calls between the replays, the graph's memory its own"""
    cell, g = cell_of(128, 64, 3), torch.Generator().manual_seed(4)
    x = torch.randn(3, 40, 128, generator=g).cuda()
    expected(cell_of(128, 64, 5), x)  # (kernels loaded)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.no_grad():
        if warm:
            with torch.cuda.stream(side):
                cell.sequence(x)
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=side):
            out = cell.sequence(x)
        want = expected(cell, x)
        assert equal(cell.sequence(x), want)  # before the first replay
        for k in range(4):
            graph.replay()
            torch.cuda.synchronize()
            assert equal(out, want), k
            cell.gates.weight.normal_()
            want = expected(cell, x)
            if k % 2:
                assert equal(cell.sequence(x), want)  # packs anew: what it replaces is not the graph's
                junk = [torch.full((256, 128), float("nan"), dtype=torch.bfloat16, device="cuda") for _ in range(64)]
                torch.cuda.synchronize()
                del junk
