"""A wait inside the 8-bit product that gives up is reported (ivf_sq_status), and
leaves the device usable.  With a limit of 0 no wait waits: the first poll finds
nothing copied and nothing multiplied yet.  What is in flight then still ends
before the kernel returns, so nothing is read or written out of place."""
import pytest
import torch

import insitu_b200 as ib

pytestmark = pytest.mark.gpu


def operands(m, n, k, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    a = torch.randint(-128, 128, (m, k), generator=g, device="cuda", dtype=torch.int8)
    b = torch.randint(-128, 128, (n, k), generator=g, device="cuda", dtype=torch.int8)
    return a, torch.ones(m, device="cuda"), b, torch.ones(n, device="cuda")


# few tokens with k split over a cluster; several tiles a block, of 16 and of 256 tokens
@pytest.mark.parametrize("m,n,k", [(16, 1024, 8192), (16, 80000, 4096), (600, 20000, 4096)])
def test_a_wait_that_gives_up_is_reported_once(cuda_ok, monkeypatch, m, n, k):
    ops = operands(m, n, k, m)
    want = ib.sq_matmul(*ops)
    ib.sq_status()
    monkeypatch.setenv("INSITU_SQ_WAIT_NS", "0")
    out = torch.full((m + 2, n), 3.0, device="cuda")
    ib.sq_matmul(*ops, out=out[1:-1])
    with pytest.raises(ib.InsituError, match="gave up"):
        ib.sq_status()
    ib.sq_status()                                       # reported once
    assert (out[0] == 3).all() and (out[-1] == 3).all()
    monkeypatch.delenv("INSITU_SQ_WAIT_NS")
    assert torch.equal(ib.sq_matmul(*ops), want)         # the device is as it was
    ib.sq_status()


def test_scores_report_too_on_a_stream_of_their_own(cuda_ok, monkeypatch):
    store = ib.SQRows(5000, 128).write(torch.randn(5000, 128, device="cuda"))
    q = torch.randn(64, 128, device="cuda")
    want = store.scores(q)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    monkeypatch.setenv("INSITU_SQ_WAIT_NS", "0")
    with torch.cuda.stream(side):
        store.scores(q)
        with pytest.raises(ib.InsituError):
            ib.sq_status()
    for limit in ("", "-1", "x", "99999999999999999999"):        # none of them a shorter limit
        monkeypatch.setenv("INSITU_SQ_WAIT_NS", limit)
        assert torch.equal(store.scores(q), want)
    ib.sq_status("cuda")


def test_status_is_refused_in_a_capture(cuda_ok):
    ops = operands(32, 500, 64, 1)
    ib.sq_matmul(*ops)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = ib.sq_matmul(*ops)
        with pytest.raises(ib.InsituError, match="captured"):
            ib.sq_status()
    graph.replay()
    ib.sq_status()
    assert torch.equal(y, ib.sq_matmul(*ops))
