"""The paged KV cache (append, read), attention over it and prompt attention
against float64 definitions (tests/paged_oracle.py), at the lengths, pages,
masks, strides and layouts where they can go wrong, and a run of them together."""
import numpy as np
import pytest
import torch

import soinfer.ops as ops
from tests import paged_oracle as oracle

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _cum(lens):
    return torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int32, device=DEV)


def _table(lens, page, seed, spare=2, cols=None):
    """Shuffled pages for sequences of the given lengths (-1 where there is none) and the pool's size."""
    need = [-(-n // page) for n in lens]
    order = torch.randperm(sum(need) + spare, generator=_gen(seed)).int()
    table = torch.full((len(lens), cols or max([1] + need)), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at : at + n]
        at += n
    return table, sum(need) + spare


def _pools(pages, nkv, page, hd, bits, fill=0xFF):
    """Pools whose every byte says NaN (fp16 0xFFFF, code -1 with a NaN scale): what is not written must not count."""
    k, v = ops.paged_kv_alloc(pages, nkv, page, hd, bits, DEV)
    for t in (k, v):
        t.view(torch.uint8).fill_(fill)
    return k, v


def _np(*ts):
    return [t.cpu().numpy() for t in ts]


def _fill(k_pages, v_pages, bits, table, lens, k, v):
    """Rows k (float32), v (float16) of packed positions into device pools, by the oracle."""
    kp, vp = _np(k_pages, v_pages)
    page, at = kp.shape[2], 0
    for b, n in enumerate(lens):
        for p in range(n):
            oracle.put((kp, vp), bits, page, int(table[b, p // page]), p % page, k[at], v[at])
            at += 1
    k_pages.copy_(torch.from_numpy(kp))
    v_pages.copy_(torch.from_numpy(vp))


# ------------------------------------------------------------------ append
APPEND = [  # new, past, page, nq, nkv, hd, norm
    ([1], [0], 16, 16, 8, 128, True),
    ([1, 1, 1], [5, 31, 100], 16, 40, 8, 128, True),
    ([3, 0, 17, 1], [0, 9, 15, 47], 32, 4, 2, 64, False),
    ([33, 70], [31, 0], 64, 5, 5, 128, False),
    ([20], [1], 16, 3, 1, 64, True),
    ([9, 8], [0, 127], 128, 0, 3, 128, True),
    ([300, 41], [2, 14], 16, 32, 4, 128, True),  # enough rows for four steps per warp
]


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("new,past,page,nq,nkv,hd,norm", APPEND)
def test_append(new, past, page, nq, nkv, hd, norm, bits):
    T, B, eps = sum(new), len(new), 1e-6
    g = _gen(T + hd + bits)
    qkv = torch.randn(T, nq + 2 * nkv, hd, generator=g).half()
    ctx = [a + b for a, b in zip(new, past)]
    table, pages = _table(ctx, page, T)
    cos, sin = (t.cpu() for t in ops.precompute_rope_table(hd, 1e6, max(ctx) + 1, "cpu"))
    qw, kw = ((1 + 0.2 * torch.randn(hd, generator=g)).half() for _ in range(2))
    pools = _pools(pages, nkv, page, hd, bits)
    d = qkv.to(DEV)
    one = all(n == 1 for n in new)
    q, k = ops.paged_kv_append(d[:, :nq] if nq else None, d[:, nq : nq + nkv], d[:, nq + nkv :], *pools, table.to(DEV),
                               torch.tensor(past, dtype=torch.int32, device=DEV), cos.to(DEV), sin.to(DEV),
                               cu_seqlens=None if one else _cum(new), q_norm=qw.to(DEV) if norm else None,
                               k_norm=kw.to(DEV) if norm else None, eps=eps, return_k=True)
    pos = np.concatenate([np.arange(p, p + n) for p, n in zip(past, new)])
    x, c, s = qkv.numpy(), cos.numpy()[pos], sin.numpy()[pos]
    wq, wk = (w.numpy() if norm else None for w in (qw, kw))
    for got, rows, w in ((q, x[:, :nq], wq), (k, x[:, nq : nq + nkv], wk)):
        if got is None:
            assert nq == 0
            continue
        want = oracle.rotate(rows, w, eps, c, s)
        # half a step of fp16 and about twelve fp32 roundings of each of the two terms
        size = oracle.rotate(np.abs(rows), None if w is None else np.abs(w), eps, np.abs(c), -np.abs(s))
        size = np.abs(size) + np.abs(oracle.rotate(np.abs(rows), None if w is None else np.abs(w), eps, np.abs(c), np.abs(s)))
        assert np.all(np.abs(got.cpu().numpy().astype(np.float64) - want) <=
                      oracle.HALF_ULP16 * np.abs(want) + 12 * 2.0**-24 * size + 2.0**-25)
    # the pools, byte for byte: nothing but the new positions' rows has changed
    kx = oracle.rotate(x[:, nq : nq + nkv], wk, eps, c, s, np.float32)
    want = [t.cpu().numpy() for t in _pools(pages, nkv, page, hd, bits)]
    at = 0
    for b in range(B):
        for p in range(past[b], past[b] + new[b]):
            oracle.put(want, bits, page, int(table[b, p // page]), p % page, kx[at], x[at, nq + nkv :])
            at += 1
    for got, w in zip(pools, want):
        assert np.array_equal(got.cpu().numpy().view(np.uint8), w.view(np.uint8))


def test_append_of_tokens_without_a_place():
    """Tokens before and behind the sequences, beyond the tables, without a page: zeros or rotated, never stored."""
    hd, page, nkv = 64, 16, 2
    cos, sin = ops.precompute_rope_table(hd, 1e4, 40, DEV)
    x = torch.randn(9, 3 * nkv, hd, generator=_gen(1)).half().to(DEV)
    for bits in (16, 4):
        pools = _pools(3, nkv, page, hd, bits)
        table = torch.tensor([[0, 7, 1], [-1, 2, 2]], dtype=torch.int32, device=DEV)  # page 7 is outside the pool
        cu = torch.tensor([2, 4, 7], dtype=torch.int32, device=DEV)
        start = torch.tensor([15, 38], dtype=torch.int32, device=DEV)
        q, k = ops.paged_kv_append(x[:, :2], x[:, 2:4], x[:, 4:], *pools, table, start, cos, sin, cu_seqlens=cu, return_k=True)
        # rows 2, 3: positions 15 (page 0), 16 (page 7); rows 4..6: positions 38, 39 (page 2), 40 (beyond the tables)
        zero = [0, 1, 6, 7, 8]
        assert torch.count_nonzero(q[zero]) == 0 and torch.count_nonzero(k[zero]) == 0
        assert torch.all(q[2:6].abs().sum((1, 2)) > 0)
        kb, vb = (t.view(torch.uint8) for t in pools)
        for t in (kb, vb):
            assert torch.all(t[1] == 0xFF)
        if bits == 16:
            written = torch.zeros(3, page, dtype=torch.bool)
            written[0, 15] = written[2, 38 % 16] = written[2, 39 % 16] = True
            for t in pools:
                assert torch.equal(~torch.isnan(t).all(-1).all(1).cpu(), written)
    # one token per sequence, more table rows than tokens is refused; a negative start is no place
    pools = _pools(3, nkv, page, hd, 16)
    start = torch.tensor([-1, 3], dtype=torch.int32, device=DEV)
    table = torch.tensor([[0], [1]], dtype=torch.int32, device=DEV)
    q, k = ops.paged_kv_append(x[:2, :2], x[:2, 2:4], x[:2, 4:], *pools, table, start, cos, sin, return_k=True)
    assert torch.count_nonzero(q[0]) == 0 and torch.isnan(pools[0][0]).all()
    assert not torch.isnan(pools[0][1, :, 3]).any() and torch.isnan(pools[0][1, :, 2]).all()


@pytest.mark.parametrize("hd", [64, 128])
def test_four_bit_rows_at_the_ends_of_the_range(hd):
    """Zeros, subnormals, the largest fp16 values, infinities and NaN through append and read."""
    page, nkv = 16, 1
    v = torch.zeros(8, nkv, hd)
    v[1, 0, 3] = 2.0**-24
    v[2] = 65504
    v[3, 0] = torch.linspace(-65504, 65504, hd)
    v[4, 0, hd - 1] = float("inf")
    v[5, 0, 0] = float("nan")
    v[6, 0, ::2] = -1e-3
    v[7, 0, 40] = -float("inf")
    v = v.half()
    cos, sin = torch.ones(8, hd // 2, device=DEV), torch.zeros(8, hd // 2, device=DEV)  # no rotation
    pools = ops.paged_kv_alloc(1, nkv, page, hd, 4, DEV)
    table, start, cu = (torch.tensor(x, dtype=torch.int32, device=DEV) for x in ([[0]], [0], [0, 8]))
    d = v.to(DEV)
    ops.paged_kv_append(None, d, d, *pools, table, start, cos, sin, cu_seqlens=cu)
    k_got, v_got = ops.paged_kv_read(*pools, table, cu, 8)
    want = [t.cpu().numpy() for t in ops.paged_kv_alloc(1, nkv, page, hd, 4, DEV)]
    kf = v.numpy().astype(np.float32)
    with np.errstate(invalid="ignore"):  # 0 * x - 0 * y, as the rotation computes it
        h = hd // 2
        kf = np.concatenate([kf[..., :h] * 1 - kf[..., h:] * 0, kf[..., h:] * 1 + kf[..., :h] * 0], -1).astype(np.float32)
    for p in range(8):
        oracle.put(want, 4, page, 0, p, kf[p], v.numpy()[p])
    for p in range(8):
        k_want, v_want = oracle.get(want, 4, page, hd, 0, p)
        with np.errstate(over="ignore"):
            for got, w in ((k_got, k_want), (v_got, v_want)):
                assert np.array_equal(got[p].cpu().numpy(), w.astype(np.float16), equal_nan=True), p
    assert torch.isnan(v_got[4]).all() and torch.isnan(v_got[5]).all() and not torch.isnan(v_got[6]).any()
    assert torch.isnan(k_got[5, 0, :32]).all()


# ------------------------------------------------------------------ read
@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("lens,page,nkv,hd", [([1], 16, 1, 128), ([0, 40, 17, 0, 1], 16, 3, 64), ([129, 64], 64, 8, 128),
                                              ([300], 128, 2, 64)])
def test_read(lens, page, nkv, hd, bits):
    T = sum(lens)
    g = _gen(T + bits)
    table, pages = _table(lens, page, T)
    pools = _pools(pages, nkv, page, hd, bits)
    k, v = (torch.randn(T, nkv, hd, generator=g) for _ in range(2))
    _fill(*pools, bits, table, lens, k.half().float().numpy(), v.half().numpy())
    out = tuple(torch.full((T + 3, nkv, hd), 9.0, dtype=torch.float16, device=DEV) for _ in range(2))
    table = table.to(DEV)
    if lens[-1] > page:
        table[-1, 1] = pages + 5  # a page that the pool does not have reads as zeros
    got = ops.paged_kv_read(*pools, table, _cum(lens), T + 3, out=out)
    assert got[0] is out[0] and torch.all(out[0][T:] == 9) and torch.all(out[1][T:] == 9)
    host, at = _np(*pools), 0
    for b, n in enumerate(lens):
        want_k, want_v, _ = oracle.context(host, bits, page, hd, table[b].cpu().numpy(), n, pages)
        assert np.array_equal(out[0][at : at + n].cpu().numpy(), want_k.astype(np.float16))
        assert np.array_equal(out[1][at : at + n].cpu().numpy(), want_v.astype(np.float16))
        at += n


# ------------------------------------------------------------------ decode attention
DECODE = [  # lens, page, nq, nkv, hd
    ([1], 16, 16, 8, 128),
    ([0, 5, 0], 16, 4, 2, 64),
    ([15, 16, 17, 31, 32, 33], 16, 4, 4, 128),
    ([127, 128, 129, 1], 32, 10, 2, 128),   # 5 heads a group
    ([777], 64, 8, 1, 64),
    ([640, 3, 200], 16, 24, 2, 128),        # 12 heads a group: two column groups
    ([1500, 1], 128, 16, 1, 64),            # 16 heads a group
    ([2100, 0, 900], 32, 2, 2, 128),
]


def _decode_case(lens, page, nq, nkv, hd, bits, seed):
    g = _gen(seed)
    T = sum(lens)
    table, pages = _table(lens, page, seed)
    pools = _pools(pages, nkv, page, hd, bits)
    k = torch.randn(T, nkv, hd, generator=g) * (0.5 * torch.randn(nkv, hd, generator=g)).exp()
    v = torch.randn(T, nkv, hd, generator=g).half()
    _fill(*pools, bits, table, lens, k.half().float().numpy(), v.numpy())
    q = torch.randn(len(lens), nq + 1, hd, generator=g).half()[:, :nq]
    return q, pools, table, pages


def _check_decode(got, q, pools, bits, table, lens, pages):
    host, page, hd = _np(*pools), pools[0].shape[2], q.shape[2]
    for b, n in enumerate(lens):
        k, v, on = oracle.context(host, bits, page, hd, table[b].cpu().numpy(), n, pages)
        qb = q[b : b + 1].cpu().numpy()
        out, mag, dot = oracle.attention(qb, k, v, on[None])
        scale = np.abs(k).max() / 7 * 1.01 if bits == 4 and n else 0.0
        bound = oracle.attention_bound(out, mag, dot, qb if bits == 4 else None, scale)
        err = np.abs(got[b : b + 1].cpu().numpy().astype(np.float64) - out)
        assert np.all(err <= bound), f"sequence {b}: {np.max(err / bound):.2f} of the bound"


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("lens,page,nq,nkv,hd", DECODE)
def test_decode_attention(lens, page, nq, nkv, hd, bits):
    q, pools, table, pages = _decode_case(lens, page, nq, nkv, hd, bits, sum(lens) + bits)
    dq = torch.full((len(lens), nq + 1, hd), float("nan"), dtype=torch.float16, device=DEV)
    dq[:, :nq] = q.to(DEV)
    out = torch.full((len(lens), nq, hd), 7.0, dtype=torch.float16, device=DEV)
    got = ops.paged_decode_attention(dq[:, :nq], *pools, table.to(DEV),
                                     torch.tensor(lens, dtype=torch.int32, device=DEV), out=out)
    assert got is out
    _check_decode(got, q, pools, bits, table, lens, pages)
    for b, n in enumerate(lens):
        if n == 0:
            assert torch.count_nonzero(got[b]) == 0


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("lens,page,nq,nkv,hd", [([3000, 0, 17, 12000], 16, 5, 1, 64), ([1], 64, 4, 2, 128),
                                                 ([255, 256, 257, 513, 70], 32, 12, 1, 128),
                                                 ([40] * 40 + [2000], 128, 2, 1, 64), ([20011], 64, 8, 1, 128)])
def test_decode_attention_with_wide_tables(lens, page, nq, nkv, hd, bits):
    """Tables that can name long sequences: positions cut into chunks over the GPU, joined afterwards."""
    T, g = sum(lens), _gen(len(lens) + bits)
    table, pages = _table(lens, page, T, cols=max(9000, max(lens) + 500) // page)
    pools = _pools(pages, nkv, page, hd, bits)
    q = torch.randn(len(lens), nq, hd, generator=g).half().to(DEV)
    k, v = (torch.randn(T, nkv, hd, generator=g).half().to(DEV) for _ in range(2))
    one, zero = torch.ones(max(lens), hd // 2, device=DEV), torch.zeros(max(lens), hd // 2, device=DEV)
    start = torch.zeros(len(lens), dtype=torch.int32, device=DEV)
    ops.paged_kv_append(None, k, v, *pools, table.to(DEV), start, one, zero, cu_seqlens=_cum(lens))
    got = ops.paged_decode_attention(q, *pools, table.to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV))
    _check_decode(got, q, pools, bits, table, lens, pages)


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("lens,page,nq,nkv,hd", [
    ([30 + i * 37 % 300 for i in range(60)] + [0] * 20 + [7000] + [5] * 45, 16, 4, 4, 64),  # more units than CTAs
    ([100] * 298 + [101, 99], 16, 2, 1, 128),
    ([5000, 0, 40, 3000], 32, 24, 2, 128),  # 12 heads a group: two column groups, split sequences
    ([0] * 50, 64, 8, 8, 64),
    ([257, 64, 65, 1024, 256] * 4 + [0, 1], 64, 10, 2, 64),
])
def test_decode_attention_of_batches(lens, page, nq, nkv, hd, bits):
    """Ranges over many sequences: several to a CTA, some over many CTAs, empty ones, units noted per sequence or CTA."""
    test_decode_attention_with_wide_tables(lens, page, nq, nkv, hd, bits)


@pytest.mark.parametrize("bits", [16, 4])
def test_decode_attention_over_missing_pages_and_odd_lengths(bits):
    """Pages that are not there are skipped; lengths below zero and beyond the table are cut."""
    lens, page, nq, nkv, hd = [700, 64, 90, 33], 32, 4, 2, 128
    q, pools, table, pages = _decode_case(lens, page, nq, nkv, hd, bits, 3)
    table[0, 3], table[0, 9], table[1, :] = -1, pages, -7
    asked = torch.tensor([700, 64, -3, 10_000_000], dtype=torch.int32, device=DEV)
    table[3] = table[0]
    seen = [700, 64, 0, table.shape[1] * page]  # the last page's unwritten slots are NaN: write them first
    full = torch.randn(seen[3], nkv, hd, generator=_gen(5)).half()
    good = table.clone()
    good[(good < 0) | (good >= pages)] = 0
    _fill(*pools, bits, good[3:4], [seen[3]], full.float().numpy(), full.numpy())
    got = ops.paged_decode_attention(q.to(DEV), *pools, table.to(DEV), asked)
    _check_decode(got, q, pools, bits, table, seen, pages)
    assert torch.count_nonzero(got[1:3]) == 0


@pytest.mark.parametrize("cols", [70, 640])
@pytest.mark.parametrize("bits", [16, 4])
def test_decode_attention_over_pages_as_allocated(bits, cols):
    """Zeroed pages hold zero keys and values (4 bits: with the scale 0), alone and next to written rows."""
    lens, page, nq, nkv, hd = [1, 40, 1000], 16, 6, 2, 128
    table, pages = _table([cols * page] * 3, page, 4)
    pools = ops.paged_kv_alloc(pages, nkv, page, hd, bits, device=DEV)
    q = torch.randn(3, nq, hd, generator=_gen(6)).half().to(DEV)
    lens_d = torch.tensor(lens, dtype=torch.int32, device=DEV)
    assert torch.count_nonzero(ops.paged_decode_attention(q, *pools, table.to(DEV), lens_d)) == 0
    k, v = (torch.randn(30, nkv, hd, generator=_gen(7)).half().to(DEV) for _ in range(2))
    one = torch.ones(1000, hd // 2, device=DEV)
    start = torch.tensor([0, 5, 500], dtype=torch.int32, device=DEV)
    ops.paged_kv_append(None, k, v, *pools, table.to(DEV), start, one, 0 * one, cu_seqlens=_cum([0, 10, 20]))
    got = ops.paged_decode_attention(q, *pools, table.to(DEV), lens_d)
    _check_decode(got, q, pools, bits, table, lens, pages)


@pytest.mark.parametrize("cols", [80, 640])
@pytest.mark.parametrize("bits", [16, 4])
def test_decode_attention_with_nan(bits, cols):
    """A NaN in a query makes its head NaN and no other; in a cached key the heads that read it, if it lies within."""
    lens, page, nq, nkv, hd = [777, 1, 300, 300], 16, 6, 2, 128
    table, pages = _table(lens, page, 4, cols=cols)
    pools = _pools(pages, nkv, page, hd, bits)
    T, g = sum(lens), _gen(16)
    q = torch.randn(4, nq, hd, generator=g).half()
    k, v = (torch.randn(T, nkv, hd, generator=g).half().to(DEV) for _ in range(2))
    k[778 + 123, 1, 70] = k[1078 + 299, 0, 5] = float("nan")
    one = torch.ones(800, hd // 2, device=DEV)
    ops.paged_kv_append(None, k, v, *pools, table.to(DEV), torch.zeros(4, dtype=torch.int32, device=DEV), one, 0 * one,
                        cu_seqlens=_cum(lens))
    bad = q.clone()
    bad[0, 1, 3] = bad[1, 5, 100] = float("nan")
    seen = [777, 1, 300, 299]  # the last sequence's NaN lies behind
    got = ops.paged_decode_attention(bad.to(DEV), *pools, table.to(DEV), torch.tensor(seen, dtype=torch.int32, device=DEV))
    for b, h in ((0, [1]), (1, [5]), (2, [3, 4, 5])):
        assert torch.isnan(got[b, h]).all(), (b, h)
        got[b, h] = 0
    assert torch.isfinite(got).all()
    pools = [torch.where(torch.isnan(t), 0, t) if bits == 16 else t for t in pools]
    if bits == 4:  # the groups that the NaN made unreadable
        ks = pools[0].view(pages, nkv, -1)[:, :, page * hd // 2 :].view(torch.float16)
        ks[torch.isnan(ks)] = 0
    want = ops.paged_decode_attention(q.to(DEV), *pools, table.to(DEV), torch.tensor(seen, dtype=torch.int32, device=DEV))
    _check_decode(want, q, pools, bits, table, seen, pages)
    for b, h in ((0, [1]), (1, [5]), (2, [3, 4, 5])):
        want[b, h] = 0
    torch.testing.assert_close(got.float(), want.float(), rtol=4 * 2.0**-11, atol=4 * 2.0**-11)


@pytest.mark.parametrize("bits", [16, 4])
def test_decode_attention_captured_replayed_and_repeatable(bits):
    """A captured call follows the lengths it finds at replay; two graphs on one pool do not share scratch; the same
    call gives the same bits, on another stream too."""
    lens, page, nq, nkv, hd = [900, 20, 333], 16, 16, 8, 128
    q, pools, table, pages = _decode_case(lens, page, nq, nkv, hd, bits, 11)
    q, table_d = q.contiguous().to(DEV), table.to(DEV)
    n = torch.tensor(lens, dtype=torch.int32, device=DEV)
    q2 = torch.randn_like(q)
    eager = ops.paged_decode_attention(q, *pools, table_d, n)
    eager2 = ops.paged_decode_attention(q2, *pools, table_d, n)
    graphs, outs, streams = [], [], [torch.cuda.Stream() for _ in range(2)]
    for x in (q, q2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(ops.paged_decode_attention(x, *pools, table_d, n))
        graphs.append(gr)
    torch.cuda.synchronize()
    for _ in range(20):
        for gr, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                gr.replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], eager) and torch.equal(outs[1], eager2)
    n.copy_(torch.tensor([1, 20, 64], dtype=torch.int32))
    graphs[0].replay()
    with torch.cuda.stream(streams[1]):
        streams[1].wait_stream(torch.cuda.current_stream())
        again = ops.paged_decode_attention(q, *pools, table_d, n)
    torch.cuda.synchronize()
    assert torch.equal(outs[0], again)
    _check_decode(again, q, pools, bits, table, [1, 20, 64], pages)


def test_append_captured_and_replayed_over_growing_lengths():
    """One captured decode step (append, then attention over start + 1 positions) follows the lengths on the device."""
    nq, nkv, hd, page, B = 4, 2, 64, 16, 3
    table, pages = _table([40, 40, 40], page, 1)
    pools = _pools(pages, nkv, page, hd, 4)
    host = [ops.paged_kv_alloc(pages, nkv, page, hd, 4, DEV) for _ in range(1)][0]
    for t, h in zip(pools, host):
        h.copy_(t)
    cos, sin = ops.precompute_rope_table(hd, 1e4, 64, DEV)
    x = torch.zeros(B, nq + 2 * nkv, hd, dtype=torch.float16, device=DEV)
    start = torch.tensor([0, 7, 30], dtype=torch.int32, device=DEV)
    steps = [torch.randn(B, nq + 2 * nkv, hd, generator=_gen(30 + i)).half().to(DEV) for i in range(5)]
    # what the cache holds before: rows of the longer sequences
    past = [0, 7, 30]
    rows = torch.randn(sum(past), 2 * nkv, hd, generator=_gen(9)).half().to(DEV)
    for p in (pools, host):
        ops.paged_kv_append(None, rows[:, :nkv], rows[:, nkv:], *p, table.to(DEV), torch.zeros_like(start), cos, sin,
                            cu_seqlens=_cum(past))
    table_d = table.to(DEV)

    def step(p, at):
        q, _ = ops.paged_kv_append(x[:, :nq], x[:, nq : nq + nkv], x[:, nq + nkv :], *p, table_d, at, cos, sin)
        return ops.paged_decode_attention(q, *p, table_d, at + 1)

    torch.cuda.synchronize()
    spare = ops.paged_kv_alloc(pages, nkv, page, hd, 4, DEV)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):  # warm-up
        step(spare, start)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(pools, start)
        start.add_(1)
    at = torch.tensor(past, dtype=torch.int32, device=DEV)
    for s in steps:
        x.copy_(s)
        graph.replay()
        want = step(host, at)
        assert torch.equal(out, want)
        at += 1
    assert all(torch.equal(a, b) for a, b in zip(pools, host))


@pytest.mark.parametrize("bits", [16, 4])
def test_pools_beyond_four_gigabytes(bits):
    """Append, read and attention on pages whose byte offsets pass 32 bits."""
    nkv, page, hd = 8, 128, 128
    per_page = nkv * page * (2 * hd if bits == 16 else hd // 2 + 2)
    pages = (1 << 32) // per_page + 6
    pools = ops.paged_kv_alloc(pages, nkv, page, hd, bits, DEV)
    lens = [200, 100]
    table = torch.tensor([[pages - 1, pages - 3], [1, pages - 2]], dtype=torch.int32, device=DEV)
    x = torch.randn(sum(lens), 4 * nkv, hd, generator=_gen(2)).half().to(DEV)
    cos, sin = ops.precompute_rope_table(hd, 1e6, 256, DEV)
    start = torch.zeros(2, dtype=torch.int32, device=DEV)
    q, k = ops.paged_kv_append(x[:, : 2 * nkv], x[:, 2 * nkv : 3 * nkv], x[:, 3 * nkv :], *pools, table, start, cos, sin,
                               cu_seqlens=_cum(lens), return_k=True)
    kr, vr = ops.paged_kv_read(*pools, table, _cum(lens), sum(lens))
    if bits == 16:
        assert torch.equal(kr, k) and torch.equal(vr, x[:, 3 * nkv :])
    last = q[torch.tensor([199, 299], device=DEV)].contiguous()
    got = ops.paged_decode_attention(last, *pools, table, torch.tensor(lens, dtype=torch.int32, device=DEV))
    for b, (a, n) in enumerate(((0, 200), (200, 100))):
        kk, vv = (t[a : a + n].cpu().numpy().astype(np.float64) for t in (kr, vr))
        qb = last[b : b + 1].cpu().numpy()
        out, mag, dot = oracle.attention(qb, kk, vv, np.ones((1, n), bool))
        bound = oracle.attention_bound(out, mag, dot, qb, np.abs(kk).max() / 7 * 1.01)
        # the rows come back rounded to fp16 from 4 bits: half a step more on scores and values
        if bits == 4:
            bound += mag * (2.0**-11 * (1 + 2 * dot))
        assert np.all(np.abs(got[b : b + 1].cpu().numpy().astype(np.float64) - out) <= bound)
    del pools


# ------------------------------------------------------------------ prompt attention
PREFILL = [  # new, past, nq, nkv, hd
    ([1], [0], 2, 1, 128),
    ([37], [0], 16, 8, 128),
    ([128, 127, 129], [0, 0, 0], 4, 2, 128),
    ([5, 0, 64, 1, 0, 200], [0, 0, 0, 0, 0, 0], 6, 2, 64),
    ([300], [0], 5, 1, 128),
    ([257, 256, 1], [0, 0, 0], 8, 8, 64),
    ([70, 1, 33], [130, 500, 0], 8, 2, 128),
    ([140, 17], [1, 300], 16, 1, 64),
    ([600], [0], 2, 2, 128),
]


def _check_prefill(got, q, k, v, new, ctx):
    iq = ik = 0
    for n, c in zip(new, ctx):
        qb, kb, vb = q[iq : iq + n].cpu().numpy(), *(t[ik : ik + c].cpu().numpy().astype(np.float64) for t in (k, v))
        seen = np.arange(c)[None] <= np.arange(n)[:, None] + c - n
        kb, vb = np.where(np.isnan(kb), 0, kb), vb
        out, mag, dot = oracle.attention(qb, kb, vb, seen)
        err = np.abs(got[iq : iq + n].cpu().numpy().astype(np.float64) - out)
        bound = oracle.attention_bound(out, mag, dot)
        assert np.all(err <= bound), f"rows {iq}..: {np.nanmax(err / bound):.2f} of the bound"
        iq, ik = iq + n, ik + c


@pytest.mark.parametrize("new,past,nq,nkv,hd", PREFILL)
def test_prefill_attention(new, past, nq, nkv, hd):
    g = _gen(sum(new) + hd)
    ctx = [a + b for a, b in zip(new, past)]
    x = torch.randn(sum(new) + 2, nq + 3, hd, generator=g).half().to(DEV)
    kv = torch.randn(sum(ctx) + 2, 2 * nkv, hd, generator=g).half().to(DEV)
    kv[sum(ctx) :] = float("nan")  # rows behind the last sequence
    x[sum(new) :] = float("nan")
    q, k, v = x[:, 1 : nq + 1], kv[:, :nkv], kv[:, nkv:]
    out = torch.full((sum(new) + 2, nq, hd), 7.0, dtype=torch.float16, device=DEV)
    got = ops.prefill_attention(q, k, v, _cum(new), cu_seqlens_k=_cum(ctx), out=out)
    assert got is out and torch.all(out[sum(new) :] == 7)
    _check_prefill(got, q, k, v, new, ctx)
    if not any(past):
        same = ops.prefill_attention(q[: sum(new)], k[: sum(new)], v[: sum(new)], _cum(new))
        assert torch.equal(same, out[: sum(new)])


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("rep,nkv", [(2, 4), (3, 1), (5, 2), (12, 1), (40, 2), (128, 1), (130, 1)])
def test_prefill_of_few_tokens_each(rep, nkv, hd):
    """A tile holds all query heads of a kv head for a few rows: groups that fill it and that do not, contexts, rows behind."""
    new, past = [1, 0, 7, 26, 3, 1, 60], [0, 300, 130, 5, 125, 128, 0]
    test_prefill_attention(new, past, rep * nkv, nkv, hd)


SPLIT = [  # new, past, nq, nkv: few tiles over long contexts, which several CTAs share
    ([16], [8000], 8, 2),
    ([1], [5000], 16, 1),
    ([200, 3], [3000, 10], 5, 1),
    ([130], [4100], 2, 1),
    ([300, 0, 2], [-200, 700, 6000], 3, 1),  # rows without keys beside a long context
    ([40, 9], [2600, 2047], 24, 2),
    ([1], [1100], 3, 3),
]


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("new,past,nq,nkv", SPLIT)
def test_prefill_over_long_contexts(new, past, nq, nkv, hd):
    test_prefill_attention(new, past, nq, nkv, hd)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_prefill_over_long_contexts_with_non_finite_values(bad, hd):
    """A non-finite key or value anywhere in a shared context: the rows that see it are what the formula gives."""
    n, ctx, nq, nkv = 20, 4500, 4, 2
    g = _gen(18)
    q = torch.randn(n, nq, hd, generator=g).half()
    k, v = (torch.randn(ctx, nkv, hd, generator=g).half() for _ in range(2))
    for at in (3, 1500, ctx - 5):
        kb, vb = k.clone(), v.clone()
        kb[at, 0, 9] = bad
        vb[at + 1, 1, 7] = bad
        cu = torch.tensor([0, n], dtype=torch.int32, device=DEV)
        got = ops.prefill_attention(q.to(DEV), kb.to(DEV), vb.to(DEV), cu, cu_seqlens_k=_cum([ctx])).cpu().numpy()
        seen = np.arange(ctx)[None] <= np.arange(n)[:, None] + ctx - n
        with np.errstate(invalid="ignore"):
            out, _, _ = oracle.attention(*(t.numpy().astype(np.float64) for t in (q, kb, vb)), seen)
        _, mag, dot = oracle.attention(*(t.numpy().astype(np.float64) for t in (q, k, v)), seen)
        mag = np.maximum(mag, np.abs(v.numpy().astype(np.float64)).max())
        fine = np.isfinite(out)
        assert np.array_equal(got[~fine], out[~fine], equal_nan=True), at
        err = np.abs(got[fine].astype(np.float64) - out[fine])
        assert np.all(err <= oracle.attention_bound(np.where(fine, out, 0), mag, dot)[fine]), at


def test_prefill_and_decode_of_two_streams_at_once_captured():
    """Shared contexts (clusters) and ranges beside one another on two streams, eager and from graphs: the same bits."""
    nq, nkv, hd, page = 8, 2, 128, 16
    g = _gen(19)
    lens = [9000, 300, 70, 2000]
    table, pages = _table(lens, page, 3)
    pools = ops.paged_kv_alloc(pages, nkv, page, hd, 4, device=DEV)
    k, v = (torch.randn(sum(lens), nkv, hd, generator=g).half().to(DEV) for _ in range(2))
    one = torch.ones(9000, hd // 2, device=DEV)
    table = table.to(DEV)
    ops.paged_kv_append(None, k, v, *pools, table, torch.zeros(4, dtype=torch.int32, device=DEV), one, 0 * one,
                        cu_seqlens=_cum(lens))
    q = torch.randn(4, nq, hd, generator=g).half().to(DEV)
    lens_d = torch.tensor(lens, dtype=torch.int32, device=DEV)
    x = torch.randn(24, nq, hd, generator=g).half().to(DEV)
    cu, ctx = _cum([17, 7]), _cum([9000, 300])
    calls = [lambda: ops.prefill_attention(x, k[:9300], v[:9300], cu, cu_seqlens_k=ctx),
             lambda: ops.paged_decode_attention(q, *pools, table, lens_d)]
    want = [call().clone() for call in calls]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in calls]
    graphs, outs = [], []
    for call, stream in zip(calls, streams):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            outs.append(call())
        graphs.append(graph)
    for _ in range(5):
        got = []
        for call, stream in zip(calls, streams):
            with torch.cuda.stream(stream):
                got.append(call())
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        for out in outs:
            out.zero_()
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))


def test_prefill_of_many_sequences_longest_anywhere():
    """More sequences than a warp has lanes, and a few with the longest in the middle."""
    g = _gen(21)
    for new in ([3, 0, 17, 130] * 10 + [260], [5, 400, 1, 129]):
        T, nq, nkv, hd = sum(new), 6, 2, 64
        q = torch.randn(T, nq, hd, generator=g).half().to(DEV)
        k, v = (torch.randn(T, nkv, hd, generator=g).half().to(DEV) for _ in range(2))
        _check_prefill(ops.prefill_attention(q, k, v, _cum(new)), q, k, v, new, new)


@pytest.mark.parametrize("hd", [64, 128])
def test_prefill_layouts(hd):
    """Heads-major rows, slices of one projection, keys shared by expansion, one token of one head: same bits as packed."""
    n, nq, nkv = 150, 4, 2
    g = _gen(22)
    q, k, v = (torch.randn(n, h, hd, generator=g).half().to(DEV) for h in (nq, nkv, nkv))
    want = ops.prefill_attention(q, k, v, _cum([n]))
    major = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v)]
    assert major[0].stride() == (hd, n * hd, 1)
    assert torch.equal(ops.prefill_attention(*major, _cum([n])), want)
    qkv = torch.cat([q, k, v], 1)
    assert torch.equal(ops.prefill_attention(qkv[:, :nq], qkv[:, nq : nq + nkv], qkv[:, nq + nkv :], _cum([n])), want)
    one = k[:, :1].expand(n, nkv, hd)
    assert torch.equal(ops.prefill_attention(q, one, one, _cum([n])),
                       ops.prefill_attention(q, one.contiguous(), one.contiguous(), _cum([n])))
    x = torch.randn(3, 5, hd, generator=g).half().to(DEV)
    got = ops.prefill_attention(x[1:2, 2:3], x[0:1, 1:2], x[2:3, 4:5], _cum([1]))  # one key: its value
    assert torch.equal(got, x[2:3, 4:5])


def test_prefill_rows_without_keys():
    """More queries than keys: the first rows see nothing and give zeros; a sequence without keys gives zeros."""
    new, ctx, nq, nkv, hd = [150, 40, 3], [130, 0, 3], 4, 2, 128
    g = _gen(8)
    q = torch.randn(sum(new), nq, hd, generator=g).half().to(DEV)
    k, v = (torch.randn(sum(ctx), nkv, hd, generator=g).half().to(DEV) for _ in range(2))
    got = ops.prefill_attention(q, k, v, _cum(new), cu_seqlens_k=_cum(ctx))
    assert torch.count_nonzero(got[:20]) == 0 and torch.count_nonzero(got[150:190]) == 0
    _check_prefill(got, q, k, v, new, ctx)
    none = ops.prefill_attention(q, k[:0], v[:0], _cum(new), cu_seqlens_k=_cum([0, 0, 0]))
    assert torch.count_nonzero(none) == 0


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_prefill_masked_places_do_not_count(bad):
    """A non-finite key or value reaches the rows that see it and no other (their own tile's earlier rows included)."""
    n, nq, nkv, hd, at = 200, 4, 2, 128, 150
    g = _gen(9)
    q = torch.randn(n, nq, hd, generator=g).half().to(DEV)
    k, v = (torch.randn(n, nkv, hd, generator=g).half().to(DEV) for _ in range(2))
    want = ops.prefill_attention(q, k, v, _cum([n]))
    k2, v2 = k.clone(), v.clone()
    k2[at, 0], v2[at, 1, 3] = bad, bad
    got = ops.prefill_attention(q, k2, v2, _cum([n]))
    # rows before see the same finite keys; the order of sums may differ where a tile is redone
    torch.testing.assert_close(got[:at].float(), want[:at].float(), rtol=4 * 2.0**-11, atol=4 * 2.0**-11)
    assert not torch.isfinite(got[at:, 2:, 3]).any()  # heads of kv head 1, value 3
    assert torch.isfinite(got[at:, 2:, 4:]).all()


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_prefill_non_finite_scores(bad, hd):
    """One non-finite key value or query value, at every place of a tile's columns: the rows that see it are what the
    formula gives (NaN where a score is NaN or +inf, or all are -inf; a score of -inf alone has no weight)."""
    n, count, nq, nkv = 40, 36, 4, 2
    g = _gen(17)
    q = torch.randn(n * count, nq, hd, generator=g).half()
    k, v = (torch.randn(n * count, nkv, hd, generator=g).half() for _ in range(2))
    kb, qb = k.clone(), q.clone()
    for s in range(count):
        kb[n * s + s, 0, s] = bad
        qb[n * s + s, 3, s] = bad
    vb = v.clone()
    vb[n - 1 :: n, :, 7] = float("inf")  # what the last row of each sequence makes of it beside such keys
    got = ops.prefill_attention(qb.to(DEV), kb.to(DEV), vb.to(DEV), _cum([n] * count)).cpu().numpy().astype(np.float64)
    seen = np.tril(np.ones((n, n), bool))
    for s in range(count):
        at = slice(n * s, n * s + n)
        with np.errstate(invalid="ignore"):
            out, _, _ = oracle.attention(*(t[at].numpy().astype(np.float64) for t in (qb, kb, vb)), seen)
        # magnitudes without the bad value: a key with the weight 0 adds nothing to the bound's sums
        _, mag, dot = oracle.attention(*(t[at].numpy().astype(np.float64) for t in (q, k, v)), seen)
        mag = np.maximum(mag, np.abs(v[at].numpy().astype(np.float64)).max())
        fine = np.isfinite(out)
        assert np.array_equal(got[at][~fine], out[~fine], equal_nan=True), s
        err = np.abs(got[at][fine] - out[fine])
        assert np.all(err <= oracle.attention_bound(np.where(fine, out, 0), mag, dot)[fine]), s


def test_prefill_large_scores_and_equal_rows():
    """Scores of thousands (one key takes all) and all-equal keys (the mean of the values seen)."""
    n, hd = 260, 64
    g = _gen(10)
    q, k, v = (torch.randn(n, 1, hd, generator=g).half().to(DEV) for _ in range(3))
    got = ops.prefill_attention(q * 40, k * 40, v, _cum([n]))
    _check_prefill(got, q * 40, k * 40, v, [n], [n])
    got = ops.prefill_attention(q, torch.ones_like(k), v, _cum([n]))
    _check_prefill(got, q, torch.ones_like(k), v, [n], [n])


def test_prefill_captured_and_on_another_stream():
    n, nq, nkv, hd = [100, 300, 50], 16, 8, 128
    g = _gen(12)
    q = torch.randn(sum(n), nq, hd, generator=g).half().to(DEV)
    k, v = (torch.randn(sum(n), nkv, hd, generator=g).half().to(DEV) for _ in range(2))
    cu = _cum(n)
    eager = ops.prefill_attention(q, k, v, cu)
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        out = ops.prefill_attention(q, k, v, cu)
    gr.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, eager)
    cu.copy_(_cum([10, 0, 440]))
    gr.replay()
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        again = ops.prefill_attention(q, k, v, cu)
    torch.cuda.synchronize()
    assert torch.equal(out, again)
    _check_prefill(again, q, k, v, [10, 0, 440], [10, 0, 440])


# ------------------------------------------------------------------ a run of them together
@pytest.mark.parametrize("bits", [16, 4])
def test_prompts_chunks_and_decode_steps_over_one_cache(bits):
    """Prompts of three sequences in two chunks, then decode steps: each step's attention equals the definition on what
    the cache holds, and with fp16 pages the whole run equals attention over the uncut sequences."""
    nq, nkv, hd, page, eps = 8, 2, 128, 16, 1e-6
    chunks, steps = [[40, 7, 65], [30, 50, 1]], 3
    total = [sum(c[b] for c in chunks) + steps for b in range(3)]
    table, pages = _table(total, page, 4)
    table_d = table.to(DEV)
    pools = _pools(pages, nkv, page, hd, bits)
    g = _gen(13)
    x = [torch.randn(n, nq + 2 * nkv, hd, generator=g).half().to(DEV) for n in total]
    cos, sin = ops.precompute_rope_table(hd, 1e6, max(total), DEV)
    qw, kw = ((1 + 0.2 * torch.randn(hd, generator=g)).half().to(DEV) for _ in range(2))
    have = [0, 0, 0]
    outs, rotated = [[] for _ in total], [[] for _ in total]
    for new in chunks + [[1, 1, 1]] * steps:
        rows = torch.cat([x[b][have[b] : have[b] + n] for b, n in enumerate(new)])
        start = torch.tensor(have, dtype=torch.int32, device=DEV)
        decode = new == [1, 1, 1]
        cu = None if decode else _cum(new)
        q, k = ops.paged_kv_append(rows[:, :nq], rows[:, nq : nq + nkv], rows[:, nq + nkv :], *pools, table_d, start, cos,
                                   sin, cu_seqlens=cu, q_norm=qw, k_norm=kw, eps=eps, return_k=True)
        have = [h + n for h, n in zip(have, new)]
        if decode:
            o = ops.paged_decode_attention(q, *pools, table_d, start + 1)
            _check_decode(o, q, pools, bits, table, have, pages)
        else:
            kc, vc = ops.paged_kv_read(*pools, table_d, _cum(have), sum(have))
            o = ops.prefill_attention(q, kc, vc, _cum(new), cu_seqlens_k=_cum(have))
            _check_prefill(o, q, kc, vc, new, have)
        at = 0
        for b, n in enumerate(new):
            outs[b].append(o[at : at + n])
            rotated[b].append((q[at : at + n], k[at : at + n]))
            at += n
    if bits == 16:
        for b, n in enumerate(total):
            q, k = (torch.cat([r[i] for r in rotated[b]]) for i in range(2))
            _check_prefill(torch.cat(outs[b]), q, k, x[b][:, nq + nkv :], [n], [n])


# ------------------------------------------------------------------ refusals
def test_refusals():
    hd, nkv, page = 128, 2, 16
    kp, vp = ops.paged_kv_alloc(2, nkv, page, hd, 16, DEV)
    k4, v4 = ops.paged_kv_alloc(2, nkv, page, hd, 4, DEV)
    t = torch.zeros(1, 2, dtype=torch.int32, device=DEV)
    n = torch.ones(1, dtype=torch.int32, device=DEV)
    cu = torch.tensor([0, 1], dtype=torch.int32, device=DEV)
    q = torch.zeros(1, 4, hd, dtype=torch.float16, device=DEV)
    kv = torch.zeros(1, nkv, hd, dtype=torch.float16, device=DEV)
    cos, sin = ops.precompute_rope_table(hd, 1e6, 8, DEV)

    def refused(match, fn, *a, **kw):
        with pytest.raises(RuntimeError, match=match):
            fn(*a, **kw)

    dec, app, read, pre = ops.paged_decode_attention, ops.paged_kv_append, ops.paged_kv_read, ops.prefill_attention
    refused("float16", dec, q.float(), kp, vp, t, n)
    refused("multiple of num_kv_heads", dec, q[:, :3], kp, vp, t, n)
    refused("both", dec, q, kp, v4, t, n)
    refused("widths", dec, q, k4, k4, t, n)
    refused("disagree", dec, q[..., :64].contiguous(), kp, vp, t, n)
    refused("int32", dec, q, kp, vp, t.long(), n)
    refused("seq_lens", dec, q, kp, vp, t, n.long())
    refused("one row per query", dec, q, kp, vp, t.expand(2, 2).contiguous(), n)
    refused("16-byte", dec, torch.zeros(4 * hd + 1, dtype=torch.float16, device=DEV)[1:].view(1, 4, hd), kp, vp, t, n)
    refused("power of two", dec, q, kp[:, :, :12].contiguous(), vp[:, :, :12].contiguous(), t, n)
    refused("out must be", dec, q, kp, vp, t, n, out=q[:, :2])
    refused("CUDA", dec, q.cpu(), kp, vp, t, n)
    refused("num_kv_heads", app, q, q, q, kp, vp, t, n, cos, sin)
    refused("one token per sequence", app, None, kv.expand(3, nkv, hd).contiguous(), kv.expand(3, nkv, hd).contiguous(), kp,
            vp, t, n, cos, sin)
    refused("head_dim / 2", app, q, kv, kv, kp, vp, t, n, cos[:, :32].contiguous(), sin[:, :32].contiguous())
    refused("q_norm", app, q, kv, kv, kp, vp, t, n, cos, sin, q_norm=cos[0].half())
    refused("eps", app, q, kv, kv, kp, vp, t, n, cos, sin, eps=-1.0)
    refused("cu_seqlens", read, kp, vp, t, n, 1)
    refused("total", read, kp, vp, t, cu, -1)
    refused("same tokens", pre, q, kv[:0], kv[:0], cu)
    refused("64 or 128", pre, q[..., :32].contiguous(), kv[..., :32].contiguous(), kv[..., :32].contiguous(), cu)
    refused("multiple", pre, q[:, :3], kv, kv, cu)
    refused("64 or 128", ops.paged_kv_alloc, 1, 1, 16, 96, 16, DEV)
    refused("power of two", ops.paged_kv_alloc, 1, 1, 24, 64, 16, DEV)
    refused("bits", ops.paged_kv_alloc, 1, 1, 16, 64, 8, DEV)
    # nothing to do is not an error
    empty = q[:0]
    assert dec(empty, kp, vp, t[:0], n[:0]).shape == (0, 4, hd)
    assert pre(empty, kv[:0], kv[:0], torch.zeros(1, dtype=torch.int32, device=DEV)).shape == (0, 4, hd)
    assert app(empty, kv[:0], kv[:0], kp, vp, t[:0], n[:0], cos, sin, return_k=True)[1].shape == (0, nkv, hd)
    assert read(kp, vp, t, torch.zeros(2, dtype=torch.int32, device=DEV), 0)[0].shape == (0, nkv, hd)
    # a table without columns names no page
    got = dec(q, kp, vp, t[:, :0], n)
    assert torch.count_nonzero(got) == 0
