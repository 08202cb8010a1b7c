"""Every cached position counts exactly once in the decode and prompt attention: rows in which each one is decisive
(tests/paged_coverage.py) over the splits by clusters and by ranges, at page, tile and range borders, beside pages that
are not there."""
import numpy as np
import pytest
import torch

import soinfer.ops as ops
from tests import paged_coverage as cover

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _cum(lens):
    return torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int32, device=DEV)


def _cat(parts, *shape):
    return torch.from_numpy(np.concatenate(parts) if parts else np.zeros((0, *shape), np.float16)).to(DEV)


def _decode(lens, page, nq, nkv, hd, bits, cols, missing=0):
    need = [-(-n // page) for n in lens]
    rng = np.random.default_rng(sum(lens) + page + bits)
    order = rng.permutation(sum(need) + 3).astype(np.int32)
    table = np.full((len(lens), max([cols // page] + need)), -1, np.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at : at + n]
        at += n
    for b in rng.choice(len(lens), missing):  # (a page of a sequence, its last one too)
        if need[b]:
            table[b, rng.integers(need[b])] = -1
    on = [np.repeat(table[b, : need[b]] >= 0, page)[:n].astype(np.float64) for b, n in enumerate(lens)]
    table_d = torch.from_numpy(table).to(DEV)
    lens_d, start = torch.tensor(lens, dtype=torch.int32, device=DEV), torch.zeros(len(lens), dtype=torch.int32, device=DEV)
    one = torch.ones(max(max(lens), 1), hd // 2, device=DEV)
    keys = [cover.key_classes(n, nkv, hd) for n in lens]
    lift, _ = cover.large(hd)
    k = _cat([cover.rows(c, hd) for c in keys], nkv, hd)
    for layout in ("stripes", "random"):
        classes = [cover.value_classes(n, nkv, hd, layout, b + n) for b, n in enumerate(lens)]
        v = _cat([cover.rows(c, hd) for c in classes], nkv, hd)
        pools = ops.paged_kv_alloc(sum(need) + 3, nkv, page, hd, bits, DEV)
        for t in pools:
            t.view(torch.uint8).fill_(0xFF)  # what is not written reads as NaN
        ops.paged_kv_append(None, k, v, *pools, table_d, start, one, 0 * one, cu_seqlens=_cum(lens))
        q = torch.zeros(len(lens), nq, hd, dtype=torch.float16, device=DEV)
        got = ops.paged_decode_attention(q, *pools, table_d, lens_d).cpu().numpy().astype(np.float64)
        for b, n in enumerate(lens):
            want = np.repeat(cover.even(classes[b], on[b], hd), nq // nkv, 0)
            assert cover.off(got[b], want, cover.EVEN) <= 1, (layout, b, cover.off(got[b], want, cover.EVEN))
    for c0 in range(0, hd, max(nq, hd // 4)):  # key classes, a few calls of all of them
        wanted = (c0 + np.arange(nq)) % hd
        q = torch.zeros(len(lens), nq, hd, dtype=torch.float16)
        q[:, torch.arange(nq), torch.from_numpy(wanted)] = float(lift)
        got = ops.paged_decode_attention(q.to(DEV), *pools, table_d, lens_d).cpu().numpy().astype(np.float64)
        for b, n in enumerate(lens):
            want = cover.chosen(classes[b], keys[b], on[b], hd, wanted)
            assert cover.off(got[b], want, cover.CHOSEN) <= 1, (c0, b, cover.off(got[b], want, cover.CHOSEN))


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("lens,page,nq,nkv,hd", [([1], 16, 16, 8, 128), ([15, 16, 17, 31, 32, 33], 16, 4, 4, 128),
                                                 ([127, 128, 129, 1], 32, 10, 2, 128), ([777], 64, 8, 1, 64),
                                                 ([640, 3, 200], 16, 24, 2, 128), ([2000, 0, 900], 32, 2, 2, 128),
                                                 ([4096], 16, 8, 1, 64), ([4000, 255, 257], 128, 3, 1, 128)])
def test_decode_by_clusters(lens, page, nq, nkv, hd, bits):
    _decode(lens, page, nq, nkv, hd, bits, 0)


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("missing", [0, 4])
@pytest.mark.parametrize("lens,page,nq,nkv,hd", [([3000, 0, 17, 12000], 16, 5, 1, 64), ([255, 256, 257, 513, 70], 32, 12, 1, 128),
                                                 ([40] * 40 + [2000], 128, 2, 1, 64), ([20011], 64, 8, 1, 128),
                                                 ([20011], 16, 2, 2, 64), ([16003, 64], 32, 8, 8, 128),
                                                 ([5000, 0, 40, 3000], 32, 24, 2, 128)])
def test_decode_by_ranges(lens, page, nq, nkv, hd, missing, bits):
    _decode(lens, page, nq, nkv, hd, bits, 9000, missing)


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("lens,page,nq,nkv,hd", [
    ([30 + i * 37 % 300 for i in range(60)] + [0] * 20 + [7000] + [5] * 45, 16, 4, 4, 64),
    ([100] * 298 + [101, 99], 16, 2, 1, 128),
    ([257, 64, 65, 1024, 256] * 4 + [0, 1], 64, 10, 2, 64),
    ([777] * 70, 32, 16, 8, 128),
])
def test_decode_of_batches(lens, page, nq, nkv, hd, bits):
    _decode(lens, page, nq, nkv, hd, bits, 9000)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("new,past,nq,nkv", [
    ([600], [0], 2, 2),
    ([257, 256, 1, 128, 129], [0] * 5, 4, 2),
    ([70, 1, 33], [130, 500, 0], 8, 2),
    ([1, 0, 7, 26, 3, 1, 60], [0, 300, 130, 5, 125, 128, 0], 10, 2),
    ([9, 4] * 20, [40, 127] * 20, 3, 1),
    ([16], [8000], 8, 2),         # few tiles over long contexts: shared by clusters of CTAs
    ([1], [5000], 16, 1),
    ([200, 3], [3000, 10], 5, 1),
    ([300, 0, 2], [-200, 700, 6000], 3, 1),
    ([5], [16003], 4, 1),
])
def test_prompts(new, past, nq, nkv, hd):
    ctx = [a + b for a, b in zip(new, past)]
    keys = [cover.key_classes(c, nkv, hd) for c in ctx]
    k = _cat([cover.rows(c, hd) for c in keys], nkv, hd)
    lift, weight = cover.large(hd)
    T, rep = sum(new), nq // nkv
    wanted = [(np.arange(n)[:, None] * 5 + np.arange(nq) * 11) % hd for n in new]  # key classes of rows and heads
    asks = np.zeros((T, nq, hd), np.float16)
    np.put_along_axis(asks, np.concatenate(wanted)[..., None], lift, -1)
    for layout in ("stripes", "random"):
        classes = [cover.value_classes(c, nkv, hd, layout, b) for b, c in enumerate(ctx)]
        values = [cover.rows(c, hd) for c in classes]
        v = _cat(values, nkv, hd)
        for q, tolerance in ((np.zeros((T, nq, hd), np.float16), cover.EVEN), (asks, cover.CHOSEN)):
            got = ops.prefill_attention(torch.from_numpy(q).to(DEV), k, v, _cum(new), cu_seqlens_k=_cum(ctx))
            got = got.cpu().numpy().astype(np.float64)
            at = 0
            for b, (n, c) in enumerate(zip(new, ctx)):
                seen = (np.arange(c)[None] <= np.arange(n)[:, None] + c - n).astype(np.float64)
                for h in range(nq):
                    w = seen
                    if tolerance == cover.CHOSEN:
                        w = seen * np.where(keys[b][None, :, h // rep] == wanted[b][:, h, None], weight, 1.0)
                    total = w.sum(1, keepdims=True)
                    want = w @ values[b][:, h // rep].astype(np.float64) / np.where(total == 0, 1, total)
                    err = cover.off(got[at : at + n, h], want, tolerance)
                    assert err <= 1, (layout, tolerance, b, h, err)
                at += n


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("seqs", [33, 34, 37, 38])
def test_decode_where_clusters_just_fit(seqs, hd, bits):
    """The most sequences that clusters take, and one more."""
    _decode([300 + 7 * i for i in range(seqs)], 16, 8, 1, hd, bits, 0)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("seqs,past", [(15, 8200), (16, 4200), (33, 2100), (34, 1100), (74, 1100), (75, 1100)])
def test_prompts_where_clusters_just_fit(seqs, past, hd):
    """Contexts shared by eight, four and two CTAs in as many clusters as the GPU holds, and in one more."""
    test_prompts([1] * (seqs - 1) + [17], [past] * seqs, 8, 1, hd)  # (17 of 16 rows: the last one's second tile)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("new,nq,nkv", [([17] * 5, 8, 1), ([16, 33, 1, 0, 17], 8, 1), ([129, 1, 128], 1, 1), ([129] * 3, 130, 1),
                                        ([26, 25, 51], 5, 1), ([1] * 9, 384, 2)])
def test_prompts_that_need_every_pair_of_tiles(new, nq, nkv, hd):
    """Lengths one beyond a tile, in layouts with one and several head groups: the grid holds every pair there may be."""
    test_prompts(new, [0] * len(new), nq, nkv, hd)
