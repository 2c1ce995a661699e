"""The eviction's selection at the lengths where its form changes: the same choice on both sides."""
import pytest
import torch

from paged_reference import evict

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("capacity,lengths", [(2048, [2048, 2047, 1, 1500]), (2064, [2064, 2049, 2048, 30]), (4112, [4096, 4112, 4097, 4095])])
@pytest.mark.parametrize("ties", [False, True])
def test_rows_around_the_change_of_form(dev, capacity, lengths, ties):
    from mase_amd.quantized import functional as F

    g = torch.Generator().manual_seed(120)
    pages = capacity // 16
    k, v = (torch.randn(4 * pages, 2, 16, 64, generator=g).bfloat16() for _ in range(2))
    table = torch.randperm(4 * pages, generator=g).view(4, pages).to(torch.int32)
    w = torch.rand(4, 2, capacity, generator=g)
    if ties:
        w = w.mul_(3).floor_()
    pos = torch.arange(capacity, dtype=torch.int32).expand(4, 2, capacity).contiguous()
    kd, vd = k.to(dev), v.to(dev)
    nw, npos, n = F.paged_kv_evict(kd, vd, table.to(dev), torch.tensor(lengths, dtype=torch.int32, device=dev), w.to(dev), pos.to(dev), capacity,
                                   900, recent=40, first=3)
    assert n.tolist() == [min(m, 900) for m in lengths]
    flat = lambda t, b: t[table[b].long()].transpose(0, 1).flatten(1, 2)  # noqa: E731  [heads, slots, dim]
    for b, m in enumerate(lengths):
        for h in range(2):
            src = evict(pos[b, h].tolist(), w[b, h].tolist(), m, 900, 40, 3)
            assert npos[b, h, :len(src)].tolist() == src and torch.equal(nw[b, h, :len(src)].cpu(), w[b, h, src])
            assert not bool(nw[b, h, len(src):].any()) and bool((npos[b, h, len(src):] == -1).all())
            for new, old in ((kd, k), (vd, v)):
                assert torch.equal(flat(new.cpu(), b)[h, :len(src)], flat(old, b)[h, src])
                assert torch.equal(flat(new.cpu(), b)[h, len(src):], flat(old, b)[h, len(src):])
