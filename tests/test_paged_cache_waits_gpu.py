"""What a PagedKVCache does on the host: no call waits for the GPU, and none can be captured."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def make(dev, fmt=None):
    from mase_amd.quantized import PagedKVCache

    return PagedKVCache(2, 2, 64, 128, page_size=16, kv_format=fmt, device=dev, track_weights=True)


@pytest.mark.parametrize("fmt", [None, "mxint8"])
def test_no_call_waits_for_the_gpu(dev, fmt):
    c = make(dev, fmt)
    x = torch.randn(2, 2, 20, 64, generator=torch.Generator().manual_seed(90)).bfloat16().to(dev)
    q = torch.randn(2, 4, 64, generator=torch.Generator().manual_seed(91)).bfloat16().to(dev)
    one = x[:, :, :1].contiguous()

    def work():
        c.append(x, x, counts=[20, 15])          # pages taken, counts sent
        for _ in range(15):
            c.append(one, one)                   # across borders of pages
            c.attend(q)
        c.update(one, one)
        c.evict(18, recent=4, first=2)           # pages given back
        c.append(one, one)
        return c.attend(q), c.lengths()

    want, held = work()
    table = c._table.clone()
    c.reset()
    torch.cuda.synchronize()
    torch.cuda.set_sync_debug_mode("error")
    try:
        got, again = work()
    finally:
        torch.cuda.set_sync_debug_mode("default")
    assert again == held and torch.equal(got, want) and torch.equal(c._table, table)
    assert c._held_dev[0].tolist() == held


def test_staged_page_numbers_arrive_in_order(dev):
    """many appends queued behind work that keeps the stream busy: each sees its own pages and counts"""
    c, d = make(dev), make(dev)
    x = torch.randn(2, 2, 9, 64, generator=torch.Generator().manual_seed(92)).bfloat16().to(dev)
    busy = torch.randn(4096, 4096, device=dev)
    counts = [[9, 0], [0, 9], [7, 8], [9, 9], [1, 2], [0, 0], [9, 5]]
    torch.cuda.synchronize()
    for _ in range(30):
        busy = busy @ busy * 1e-4
    for n in counts:
        c.append(x, x, counts=n)
    for n in counts:
        d.append(x, x, counts=n)
        torch.cuda.synchronize()
    assert torch.equal(c._table, d._table) and c._held_dev[0].tolist() == c.lengths() == [35, 33]
    for a, b in zip(c.gather(), d.gather()):
        assert torch.equal(a.view(torch.int16), b.view(torch.int16))


def test_steps_refuse_to_be_captured(dev):
    """a replay would not move the host's lengths on"""
    c = make(dev)
    x = torch.randn(2, 2, 4, 64, generator=torch.Generator().manual_seed(93)).bfloat16().to(dev)
    q = torch.randn(2, 4, 64, generator=torch.Generator().manual_seed(94)).bfloat16().to(dev)
    c.update(x, x)
    want = c.attend(q)
    other = torch.zeros(8, device=dev)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        other += 1
        for call in (lambda: c.append(x, x), lambda: c.update(x, x), lambda: c.gather(), lambda: c.attend(q),
                     lambda: c.add_weights(torch.empty(2, 2, 1, 4, device=dev)), lambda: c.evict(2), lambda: c.reset()):
            with pytest.raises(RuntimeError, match="captured"):
                call()
    graph.replay()
    torch.cuda.synchronize()
    assert c.lengths() == [4, 4] and other.tolist() == [1.0] * 8
    c.reset()
    c.update(x, x)
    assert torch.equal(c.attend(q), want)
