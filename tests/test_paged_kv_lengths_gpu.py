"""Lengths in device memory beyond what a call or its table holds: cut, for every reader, with the results looked at."""
import math

import pytest
import torch

from paged_reference import HALF, Pool, attend

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt", [None, "mxint8", "mxfp4"])
@pytest.mark.parametrize("max_length", [150, 100])
def test_lengths_past_the_table_count_for_max_length(dev, fmt, max_length):
    """150 slots in tables of 160; a length of 2^30 counts for max_length, slots in pages that are not there apart"""
    from mase_amd.quantized import functional as F

    p = Pool(torch.Generator().manual_seed(100), [150, 150], 2, 64, 16, fmt, torch.bfloat16)
    absent = torch.zeros(2, 160, dtype=torch.bool)
    good = p.table.clone()
    for b, at, bad in ((0, 0, -1), (0, 5, p.k.shape[0]), (1, 2, 1 << 20), (1, 3, -0x80000000)):
        p.table[b, at] = bad
        absent[b, 16 * at:16 * at + 16] = True
    kw = p.to(dev)
    p.table = good
    n = torch.tensor([1 << 30, 0x7FFFFFFF], dtype=torch.int32, device=dev)
    q = torch.randn(2, 4, 64, generator=torch.Generator().manual_seed(101)).bfloat16()
    w = torch.full((2, 2, 160), 0.25, device=dev)
    out = F.paged_attention_decode(q.to(dev), **kw, lengths=n, max_length=max_length, weights=w).cpu().double()
    k, v = (t.cpu().double() for t in F.paged_kv_gather(**kw, lengths=n, max_length=max_length, dtype=torch.bfloat16))
    got = w.cpu().double()
    for b in range(2):
        kk, vv = p.rows(b, max_length)
        gone = absent[b, :max_length]
        row = torch.zeros(max_length, dtype=torch.float64).masked_fill(gone, -math.inf)
        o, pr, to, tp = attend(q[b], kk, vv, 64 ** -0.5, row, torch.bfloat16)
        assert bool(((out[b] - o).abs() <= to).all())
        add = pr.view(2, 2, -1).sum(1)
        assert bool(((got[b, :, :max_length] - 0.25 - add).abs() <= tp.view(2, 2, -1).sum(1) + 3 * HALF[torch.float32] * (add + 0.25)).all())
        assert bool((got[b, :, :max_length][:, gone] == 0.25).all()) and bool((got[b, :, max_length:] == 0.25).all())
        for have, want in ((k, kk), (v, vv)):
            assert not bool(have[b][:, gone].any()) and torch.equal(have[b][:, ~gone], want[:, ~gone])


@pytest.mark.parametrize("max_length,keep", [(150, 40), (100, 40), (150, 120)])
def test_evictions_cut_such_lengths_too(dev, max_length, keep):
    from mase_amd.quantized import functional as F

    g = torch.Generator().manual_seed(102)
    p = Pool(g, [150, 150], 2, 64, 16, None, torch.bfloat16)
    w = torch.rand(2, 2, 160, generator=g)
    pos = torch.arange(160, dtype=torch.int32).expand(2, 2, 160).contiguous()
    lengths = [1 << 30, max_length]
    nw, npos, nlen = F.paged_kv_evict(**p.to(dev), lengths=torch.tensor(lengths, dtype=torch.int32, device=dev), weights=w.to(dev),
                                      positions=pos.to(dev), max_length=max_length, keep=keep, recent=5, first=2)
    assert nlen.tolist() == [keep, keep]
    from paged_reference import evict

    for b in range(2):
        for h in range(2):
            src = evict(pos[b, h].tolist(), w[b, h].tolist(), max_length, keep, 5, 2)
            assert npos[b, h, :keep].tolist() == src and torch.equal(nw[b, h, :keep].cpu(), w[b, h, src])
            assert not bool(nw[b, h, keep:].any()) and bool((npos[b, h, keep:] == -1).all())
