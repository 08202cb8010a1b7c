"""Values and calls at the edge of what the paged-cache and prompt operators take."""
import numpy as np
import pytest
import torch

import soinfer.ops as ops
from tests import paged_oracle as oracle

pytestmark = pytest.mark.gpu
DEV = "cuda"
INF, NAN = float("inf"), float("nan")


def _ints(*x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _gen(seed):
    return torch.Generator().manual_seed(seed)


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("hd", [64, 128])
def test_append_of_non_finite_rows_under_the_head_norm(hd, bits):
    """A head row with an infinity: 1 / sqrt(inf) = 0, so its finite values become 0 and the infinity NaN, with the partner
    of its rotation pair; in 4 bits the groups of these two.  A NaN makes the whole row NaN.  Queries and keys alike."""
    T, nq, nkv, page, eps = 7, 3, 2, 16, 1e-6
    g = _gen(hd + bits)
    x = torch.randn(T, nq + 2 * nkv, hd, generator=g).half()
    for t, (value, d) in enumerate([(INF, 0), (-INF, 5), (NAN, 9), (INF, hd - 1), (-INF, hd // 2 + 3), (INF, 40)]):
        x[t, 1, d] = x[t, nq + t % nkv, d] = value
    x[5, nq + 1, 3] = -INF  # two of them
    cos, sin = (t.cpu() for t in ops.precompute_rope_table(hd, 1e4, 32, "cpu"))
    qw, kw = ((1 + 0.2 * torch.randn(hd, generator=g)).half() for _ in range(2))
    pools = ops.paged_kv_alloc(1, nkv, page, hd, bits, DEV)
    d = x.to(DEV)
    q, k = ops.paged_kv_append(d[:, :nq], d[:, nq : nq + nkv], d[:, nq + nkv :], *pools, _ints([0]), _ints(3), cos.to(DEV),
                               sin.to(DEV), cu_seqlens=_ints(0, T), q_norm=qw.to(DEV), k_norm=kw.to(DEV), eps=eps, return_k=True)
    c, s = cos.numpy()[3 : 3 + T], sin.numpy()[3 : 3 + T]
    want = [t.cpu().numpy() for t in ops.paged_kv_alloc(1, nkv, page, hd, bits, DEV)]
    with np.errstate(all="ignore"):
        for got, rows, w in ((q, x[:, :nq], qw), (k, x[:, nq : nq + nkv], kw)):
            exact = oracle.rotate(rows.numpy(), w.numpy(), eps, c, s)
            got = got.cpu().numpy().astype(np.float64)
            assert np.array_equal(np.isnan(got), np.isnan(exact))
            bad = ~np.isfinite(rows.numpy()).all(-1)
            assert np.all(got[bad][np.isfinite(exact[bad])] == 0)
            # |x^| <= sqrt(hd) |w|: half a step and about twelve fp32 roundings of two such terms
            most = np.nanmax(np.abs(exact))
            fine = np.isfinite(exact)
            assert np.all(np.abs(got - exact)[fine] <= oracle.HALF_ULP16 * np.abs(exact[fine]) + 24 * 2.0**-24 * 2 * most + 2.0**-25)
        kx = oracle.rotate(x[:, nq : nq + nkv].numpy(), kw.numpy(), eps, c, s, np.float32)
        for t in range(T):
            oracle.put(want, bits, page, 0, 3 + t, kx[t], x[t, nq + nkv :].numpy())
        kr, vr = ops.paged_kv_read(*pools, _ints([0]), _ints(0, 3 + T), 3 + T)
        for t in range(T):
            wk, wv = oracle.get(want, bits, page, hd, 0, 3 + t)
            assert np.array_equal(kr[3 + t].cpu().numpy(), wk.astype(np.float16), equal_nan=True), t
            assert np.array_equal(vr[3 + t].cpu().numpy(), wv.astype(np.float16), equal_nan=True), t


@pytest.mark.parametrize("eps,weight", [(0.0, 1.0), (1e-6, INF)])
def test_tokens_without_a_place_are_zeros_whatever_the_norm(eps, weight):
    """Beyond the tables, of no sequence, with a negative start: zeros, where the norm of a zero row would be NaN."""
    hd, nkv = 64, 2
    cos, sin = ops.precompute_rope_table(hd, 1e4, 10, DEV)
    x = torch.randn(6, 3 * nkv, hd, generator=_gen(1)).half().to(DEV)
    w = torch.ones(hd, dtype=torch.float16, device=DEV)
    w[3] = weight
    pools = ops.paged_kv_alloc(2, nkv, 16, hd, 16, DEV)
    args = (x[:, :nkv], x[:, nkv : 2 * nkv], x[:, 2 * nkv :], *pools, _ints([0], [1]), _ints(8, -1), cos, sin)
    q, k = ops.paged_kv_append(*args, cu_seqlens=_ints(0, 3, 4), q_norm=w, k_norm=w, eps=eps, return_k=True)
    for t in (q, k):  # rows 0, 1 stand at 8 and 9; row 2 at 10, row 3 at -1, rows 4 and 5 nowhere
        assert torch.count_nonzero(t[2:]) == 0
        assert torch.all(t[:2].isnan() | (t[:2] != 0) if weight == INF else t[:2].isfinite())
    assert torch.count_nonzero(pools[0][1]) == 0


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("cols", [2, 640])
@pytest.mark.parametrize("route", ["infinity", "scale"])
def test_four_bit_keys_that_read_as_nan_reach_the_output(route, cols, hd):
    """A key group with an infinity, or whose scale is beyond fp16, reads as NaN: so is every head that attends to it."""
    B, n, nq, nkv, page = 96, 20, 4, 2, 16
    g = _gen(hd + cols)
    k, v = (torch.randn(B * n, nkv, hd, generator=g).half() for _ in range(2))
    cos, sin = ops.precompute_rope_table(hd, 1e4, n, DEV)
    table = torch.full((B, cols), -1, dtype=torch.int32)
    table[:, :2] = torch.arange(2 * B, dtype=torch.int32).view(B, 2)
    weight = None
    for b in range(B):  # head 0 of one position of each sequence
        at = b * n + 1 + b % (n - 1)
        if route == "infinity":
            k[at, 0, b * 5 % hd] = INF if b % 2 else -INF
        else:  # normalised to +- sqrt(hd) at one value, times a weight of 65504: beyond 7 times fp16's largest scale, 458528
            k[at, 0] = 0
            k[at, 0, b * 5 % hd] = 1.0 if b % 2 else -1.0
    if route == "scale":
        # 8 * 65504 (hd 64) may fall below 458528 after a rotation; the random rows, at most 4.9 * 65504, stay below it
        grow = 1.3 if hd == 64 else 1.0
        cos, sin = grow * cos, grow * sin
        weight = torch.full((hd,), 65504.0, dtype=torch.float16, device=DEV)
    pools = ops.paged_kv_alloc(2 * B, nkv, page, hd, 4, DEV)
    cu = _ints(*range(0, B * n + 1, n))
    ops.paged_kv_append(None, k.to(DEV), v.to(DEV), *pools, table.to(DEV), torch.zeros(B, dtype=torch.int32, device=DEV), cos,
                        sin, cu_seqlens=cu, k_norm=weight)
    kr, _ = ops.paged_kv_read(*pools, table.to(DEV), cu, B * n)
    assert kr.view(B, n, nkv, hd)[:, :, 0].isnan().any(-1).any(-1).all()
    q = torch.randn(B, nq, hd, generator=g).half().to(DEV)
    if route == "scale":
        q *= 2.0**-10
    lens = torch.full((B,), n, dtype=torch.int32, device=DEV)
    # (values of very different sizes: sums over the codes' offsets that do not come out exactly)
    wide = (q.cpu() * torch.exp2(torch.randint(-10, 1, (B, nq, hd), generator=g))).half().to(DEV)
    for x in (q, wide):
        got = ops.paged_decode_attention(x, *pools, table.to(DEV), lens)
        assert got[:, : nq // nkv].isnan().all()
        assert got[:, nq // nkv :].isfinite().all()


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("cols", [5, 640])
@pytest.mark.parametrize("bits", [16, 4])
def test_decode_scores_of_minus_infinity(bits, cols, hd):
    """exp(-inf) is 0 beside a finite score; where every score is -inf the output is 0 / 0, not that of an empty sequence."""
    page, nq, nkv, n = 16, 4, 1, 70
    lens = [n, n, n, 0, 1]
    B, g = len(lens), _gen(3)
    k, v = (torch.randn(B, n, nkv, hd, generator=g).half() for _ in range(2))
    q = torch.randn(B, nq, hd, generator=g).half()
    channel = 5  # one value of every key that a query of infinity meets
    k[:, :, :, channel] = -1 - k[:, :, :, channel].abs()
    q[0, 1, channel] = INF             # every score -inf: NaN; the other heads are not touched
    q[3, :, channel] = q[4, 2, channel] = INF
    q[1:3, :, channel] = 1 + q[1:3, :, channel].abs()
    if bits == 16:
        k[1, :40, :, channel] = -INF   # whole tiles of -inf, then finite ones
        k[2, :, :, channel] = -INF     # nothing else: every head NaN
    need = -(-n // page)
    table = torch.full((B, cols), -1, dtype=torch.int32)
    table[:, :need] = torch.arange(B * need, dtype=torch.int32).view(B, need)
    pools = ops.paged_kv_alloc(B * need, nkv, page, hd, bits, DEV)
    if bits == 16:
        for pool, rows in zip(pools, (k, v)):
            at = torch.zeros(B, need * page, nkv, hd, dtype=torch.float16)
            at[:, :n] = rows
            pool.copy_(at.view(B * need, page, nkv, hd).transpose(1, 2))
    else:
        one = torch.ones(n, hd // 2, device=DEV)
        ops.paged_kv_append(None, *(t.reshape(B * n, nkv, hd).to(DEV) for t in (k, v)), *pools, table.to(DEV),
                            torch.zeros(B, dtype=torch.int32, device=DEV), one, 0 * one,
                            cu_seqlens=_ints(*range(0, B * n + 1, n)))
    got = ops.paged_decode_attention(q.to(DEV), *pools, table.to(DEV), _ints(*lens)).cpu()
    nan = torch.zeros(B, nq, dtype=torch.bool)
    nan[0, 1] = nan[4, 2] = True
    if bits == 16:
        nan[2] = True
    assert torch.equal(got.isnan().all(-1), nan) and torch.equal(got.isnan().any(-1), nan)
    assert torch.count_nonzero(got[3]) == 0
    if bits == 16:
        out, mag, dot = oracle.attention(q[1:2].numpy(), k[1, 40:].numpy().astype(np.float64), v[1, 40:].numpy().astype(np.float64),
                                         np.ones((1, n - 40), bool))
        assert np.all(np.abs(got[1:2].numpy().astype(np.float64) - out) <= oracle.attention_bound(out, mag, dot))
    none = torch.full_like(table, -1)  # positions, but no page: nothing to attend to, whatever the query
    assert torch.count_nonzero(ops.paged_decode_attention(q.to(DEV), *pools, none.to(DEV), _ints(*lens))) == 0


def test_prefill_of_empty_expanded_rows():
    """Keys shared by expansion, of which there are none: every query gives zeros."""
    q = torch.randn(5, 4, 64, generator=_gen(2)).half().to(DEV)
    none = torch.empty(0, 1, 64, dtype=torch.float16, device=DEV).expand(0, 2, 64)
    got = ops.prefill_attention(q, none, none, _ints(0, 5), cu_seqlens_k=_ints(0, 0))
    assert got.shape == q.shape and torch.count_nonzero(got) == 0
    empty = torch.empty(0, 1, 64, dtype=torch.float16, device=DEV).expand(0, 4, 64)
    assert ops.prefill_attention(empty, none, none, _ints(0, 0)).shape == (0, 4, 64)


def test_read_into_overlapping_outputs_is_refused():
    pools = ops.paged_kv_alloc(2, 2, 16, 64, 16, DEV)
    buf = torch.zeros(2 * 20 * 2 * 64, dtype=torch.float16, device=DEV)
    a, b = buf[: 20 * 128].view(20, 2, 64), buf[20 * 128 :].view(20, 2, 64)
    ops.paged_kv_read(*pools, _ints([0, 1]), _ints(0, 20), 20, out=(a, b))
    shifted = buf[128 : 21 * 128].view(20, 2, 64)
    for out in ((a, a), (a, shifted), (shifted, a)):
        with pytest.raises(RuntimeError, match="overlap"):
            ops.paged_kv_read(*pools, _ints([0, 1]), _ints(0, 20), 20, out=out)


@pytest.mark.parametrize("cols", [20, 640])
@pytest.mark.parametrize("bad", [INF, -INF, NAN])
def test_decode_of_non_finite_values(bad, cols):
    """A value that is not finite reaches that value of its kv head's outputs, as the formula has it where its weight is not
    far below the others', and nothing if it lies behind the sequence."""
    lens, page, nq, nkv, hd = [300, 300, 20], 16, 6, 2, 64
    table = torch.full((3, cols), -1, dtype=torch.int32)
    table[:, :19] = torch.arange(57, dtype=torch.int32).view(3, 19)
    g = _gen(5)
    q = torch.randn(3, nq, hd, generator=g).half().to(DEV)
    k, v = (torch.randn(57, nkv, page, hd, generator=g).half().to(DEV) for _ in range(2))
    lens = _ints(*lens)
    want = ops.paged_decode_attention(q, k, v, table.to(DEV), lens)
    v[19 * 0 + 7, 1, 3, 9] = bad   # position 115 of the first
    v[19 * 1 + 18, 0, 12, 5] = bad  # position 300 of the second: behind it
    v[19 * 2 + 1, 0, 4:] = bad     # position 20 and on of the third
    got = ops.paged_decode_attention(q, k, v, table.to(DEV), lens)
    hit = got[0, 3:, 9]
    assert hit.isnan().all() if bad != bad else torch.all(hit == bad)
    got[0, 3:, 9] = want[0, 3:, 9] = 0
    assert torch.equal(got, want)
