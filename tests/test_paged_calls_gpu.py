"""Calls that the documents of the paged-cache and prompt operators allow, beside the plain ones: layouts, shared and very
large pages, thousands of sequences, rows past 4 GiB, two threads and streams at once."""
import threading

import numpy as np
import pytest
import torch

import soinfer.ops as ops
from soinfer import _C
from tests import paged_oracle as oracle

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _randn(seed, *shape):
    return torch.randn(*shape, generator=_gen(seed), device=DEV).half()


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _cum(lens):
    return _ints([0] + list(np.cumsum(lens)))


def _filled(lens, page, nkv, hd, bits, seed, extra_cols=0):
    """Pools and a table that hold random rows of these lengths, and the rows."""
    cols = -(-max(lens) // page) + extra_cols
    order = np.random.default_rng(seed).permutation(len(lens) * cols).reshape(len(lens), cols)
    pools, table = ops.paged_kv_alloc(order.size, nkv, page, hd, bits, DEV), _ints(order.tolist())
    k, v = _randn(seed, sum(lens), nkv, hd), _randn(seed + 1, sum(lens), nkv, hd)
    one = torch.ones(max(lens), hd // 2, device=DEV)
    ops.paged_kv_append(None, k, v, *pools, table, _ints([0] * len(lens)), one, 0 * one, cu_seqlens=_cum(lens))
    return pools, table, k, v


def _close(got, q, k, v, seen):
    """Against the definition over rows as the cache gives them (fp16 pages)."""
    out, mag, dot = oracle.attention(q.cpu().numpy(), *(t.cpu().numpy().astype(np.float64) for t in (k, v)), seen)
    assert np.all(np.abs(got.cpu().numpy().astype(np.float64) - out) <= oracle.attention_bound(out, mag, dot))


@pytest.mark.parametrize("bits", [16, 4])
def test_layouts_of_append_and_decode_rows(bits):
    """Heads-major and expanded rows, a window of a wider table: the same bits as packed ones."""
    lens, page, nq, nkv, hd = [40, 1, 300], 16, 6, 2, 64
    pools, table, k, v = _filled(lens, page, nkv, hd, bits, 1)
    q, n = _randn(3, 3, nq, hd), _ints(lens)
    want = ops.paged_decode_attention(q, *pools, table, n)
    major = q.transpose(0, 1).contiguous().transpose(0, 1)
    wide = torch.full((3, table.shape[1] + 9), -5, dtype=torch.int32, device=DEV)
    wide[:, 4 : 4 + table.shape[1]] = table
    window = wide[:, 4 : 4 + table.shape[1]]
    assert torch.equal(ops.paged_decode_attention(major, *pools, window, n), want)
    same = q[:1].expand(3, nq, hd)
    assert torch.equal(ops.paged_decode_attention(same, *pools, table, n),
                       ops.paged_decode_attention(same.contiguous(), *pools, table, n))
    cos, sin = ops.precompute_rope_table(hd, 1e4, 300, DEV)
    x = _randn(4, sum(lens), nq, hd)
    shared = v[:, :1].expand(sum(lens), nkv, hd)
    results = []
    for rows, keys, values, tab in ((x, k, shared.contiguous(), table),
                                    (x.transpose(0, 1).contiguous().transpose(0, 1),
                                     k.transpose(0, 1).contiguous().transpose(0, 1), shared, window)):
        into = ops.paged_kv_alloc(pools[0].shape[0], nkv, page, hd, bits, DEV)
        out = ops.paged_kv_append(rows, keys, values, *into, tab, _ints([0] * 3), cos, sin, cu_seqlens=_cum(lens), return_k=True)
        results.append((*out, *into, *ops.paged_kv_read(*into, tab, _cum(lens), sum(lens))))
    for a, b in zip(*results):
        assert torch.equal(a, b)


@pytest.mark.parametrize("cols", [0, 900])
@pytest.mark.parametrize("bits", [16, 4])
def test_sequences_that_share_pages(bits, cols):
    """A common prefix is held once: three tables name its pages, and the same page may stand twice in one table."""
    page, nq, nkv, hd = 16, 8, 2, 128
    pools, table, k, v = _filled([100], page, nkv, hd, bits, 5)
    row = table[0].tolist()
    tables = _ints([row + [-1] * cols, row[:3] + [-1] * (len(row) - 3 + cols), row[:2] + row[:2] + [-1] * (len(row) - 4 + cols)])
    q = _randn(7, 1, nq, hd).expand(3, nq, hd).contiguous()
    lens = [100, 40, 64]
    got = ops.paged_decode_attention(q, *pools, tables, _ints(lens))
    kr, vr = ops.paged_kv_read(*pools, tables, _cum(lens), sum(lens))
    assert torch.equal(kr[100:140], kr[:40]) and torch.equal(kr[140:172], kr[:32]) and torch.equal(vr[172:], vr[:32])
    alone = ops.paged_decode_attention(q[:1], *pools, tables[1:2, :], _ints([40]))
    assert torch.equal(got[1:2], alone) or cols  # (by ranges the cuts may lie elsewhere)
    half = ops.paged_decode_attention(q[:1], *pools, tables[:1], _ints([32]))  # every position twice: the same mean
    torch.testing.assert_close(got[2:].float(), half.float(), rtol=4 * 2.0**-11, atol=4 * 2.0**-11)


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("page", [1024, 65536])
def test_very_large_pages(page, bits):
    lens, nq, nkv, hd = [page + 77, 5, page], 4, 2, 64
    pools, table, k, v = _filled(lens, page, nkv, hd, bits, 8)
    q = _randn(9, 3, nq, hd)
    got = ops.paged_decode_attention(q, *pools, table, _ints(lens))
    kr, vr = ops.paged_kv_read(*pools, table, _cum(lens), sum(lens))
    if bits == 16:
        assert torch.equal(kr, k) and torch.equal(vr, v)
    at = 0
    for b, n in enumerate(lens):
        x = q[b].float().view(nkv, nq // nkv, hd) @ kr[at : at + n].float().permute(1, 2, 0) / 8.0
        want = (torch.softmax(x.double(), -1) @ vr[at : at + n].double().transpose(0, 1)).view(nq, hd)
        # half a step of each probability and of the output; 4-bit rows come back rounded to fp16: as much again of each
        # value, and of each score's terms (|q| |k| / 8 below 12 here)
        size = (torch.softmax(x.double(), -1) @ vr[at : at + n].double().abs().transpose(0, 1)).view(nq, hd)
        bound = size * (2.0**-11 + 2.0**-14 + (2.0**-11 * 25 if bits == 4 else 0)) + 2.0**-11 * want.abs() + 2.0**-24
        assert torch.all((got[b].double() - want).abs() <= bound)
        at += n


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("seqs", [5000, 32768])
def test_thousands_of_sequences(seqs, bits):
    """Each one's few positions and its own result; one of them empty, one long."""
    page, nq, nkv, hd = 16, 2, 1, 64
    lens = [1 + i % 3 for i in range(seqs)]
    lens[seqs // 2], lens[7] = 3000, 0
    start = np.concatenate([[0], np.cumsum([-(-n // page) for n in lens])])
    table = np.full((seqs, 188), -1, np.int32)
    for b, n in enumerate(lens):
        table[b, : start[b + 1] - start[b]] = np.arange(start[b], start[b + 1])
    pools, table = ops.paged_kv_alloc(int(start[-1]), nkv, page, hd, bits, DEV), torch.from_numpy(table).to(DEV)
    v = torch.zeros(sum(lens), nkv, hd, dtype=torch.float16, device=DEV)
    owner = torch.repeat_interleave(torch.arange(seqs, device=DEV), _ints(lens).long())
    v[torch.arange(len(owner), device=DEV), 0, owner % hd] = 7.0
    one = torch.ones(3000, hd // 2, device=DEV)
    q, k = ops.paged_kv_append(_randn(1, sum(lens), nq, hd), _randn(2, sum(lens), nkv, hd), v, *pools, table,
                               _ints([0] * seqs), one, 0 * one, cu_seqlens=_cum(lens), return_k=True)
    got = ops.paged_decode_attention(_randn(3, seqs, nq, hd), *pools, table, _ints(lens)).float()
    want = torch.zeros(seqs, hd, device=DEV)
    want[torch.arange(seqs), torch.arange(seqs) % hd] = 7.0  # all values of a sequence are alike: their mean
    want[7] = 0
    assert torch.all((got - want[:, None]).abs() <= 7 * 2 * 2.0**-11)
    kr, vr = ops.paged_kv_read(*pools, table, _cum(lens), sum(lens))
    assert torch.equal(vr, v) and (bits == 4 or torch.equal(kr, k))


def test_prompt_rows_past_four_gigabytes():
    """Queries, outputs, keys and values whose byte offsets pass 32 bits: the last sequences equal the same ones alone."""
    hd, nkv, nq = 128, 4, 8
    ctx = (1 << 32) // (nkv * hd * 2) + 5000
    k, v = (torch.zeros(ctx, nkv, hd, dtype=torch.float16, device=DEV) for _ in range(2))
    for t, seed in ((k, 1), (v, 2)):
        t[-2000:] = _randn(seed, 2000, nkv, hd)
    q = _randn(3, 300, nq, hd)
    got = ops.prefill_attention(q, k, v, _ints([0, 0, 300]), cu_seqlens_k=_ints([0, ctx - 2000, ctx]))
    want = ops.prefill_attention(q, k[-2000:].clone(), v[-2000:].clone(), _ints([0, 0, 300]), cu_seqlens_k=_ints([0, 0, 2000]))
    bound = 4 * 2.0**-11
    torch.testing.assert_close(got.float(), want.float(), rtol=bound, atol=bound)  # (the keys may be shared otherwise)
    del k, v
    T = (1 << 32) // (nq * hd * 2) + 3000
    q = torch.zeros(T, nq, hd, dtype=torch.float16, device=DEV)
    q[-300:] = _randn(4, 300, nq, hd)
    k, v = _randn(5, 2000, nkv, hd), _randn(6, 2000, nkv, hd)
    out = torch.full_like(q, 3.0)
    ops.prefill_attention(q, k, v, _ints([T - 300, T]), cu_seqlens_k=_ints([0, 2000]), out=out)
    want = ops.prefill_attention(q[-300:].clone(), k, v, _ints([0, 300]), cu_seqlens_k=_ints([0, 2000]))
    torch.testing.assert_close(out[-300:].float(), want.float(), rtol=bound, atol=bound)
    assert torch.all(out[:-300] == 3.0)


def test_many_empty_prompts_and_many_heads():
    q, k, v = _randn(1, 3, 1024, 64), _randn(2, 3, 1, 64), _randn(3, 3, 1, 64)
    cu = _ints([0] * 500 + [1] * 500 + [3] * 500)
    got = ops.prefill_attention(q, k, v, cu)
    _close(got[:1], q[:1], k[:1], v[:1], np.ones((1, 1), bool))
    _close(got[1:], q[1:], k[1:], v[1:], np.tril(np.ones((2, 2), bool)))
    pools, table, k, v = _filled([30, 200], 32, 1, 64, 16, 4)
    for extra in (0, 300):
        wide = torch.cat([table, torch.full((2, extra), -1, dtype=torch.int32, device=DEV)], 1)
        got = ops.paged_decode_attention(q[:2], *pools, wide, _ints([30, 200]))
        _close(got[:1], q[:1], k[:30], v[:30], np.ones((1, 30), bool))
        _close(got[1:], q[1:2], k[30:], v[30:], np.ones((1, 200), bool))


def test_two_threads_at_once():
    """Each thread its own stream and inputs, all four operators: what one alone gives."""
    nq, nkv, hd, page = 8, 2, 128, 16
    cos, sin = ops.precompute_rope_table(hd, 1e4, 700, DEV)

    def work(seed, bits):
        lens = [300 + seed, 40, 600]
        pools, table, k, v = _filled(lens, page, nkv, hd, bits, seed)
        x = _randn(seed + 9, 3, nq + 2 * nkv, hd)
        q, _ = ops.paged_kv_append(x[:, :nq], x[:, nq : nq + nkv], x[:, nq + nkv :], *pools, table, _ints([n - 1 for n in lens]), cos, sin)
        kr, vr = ops.paged_kv_read(*pools, table, _cum(lens), sum(lens))
        y = _randn(seed + 5, sum(lens), nq, hd)
        wide = torch.cat([table, torch.full((3, 600), -1, dtype=torch.int32, device=DEV)], 1)
        return [ops.paged_decode_attention(q, *pools, table, _ints(lens)), ops.paged_decode_attention(q, *pools, wide, _ints(lens)),
                kr, vr, ops.prefill_attention(y, kr, vr, _cum(lens))]

    want = [work(i, bits) for i, bits in enumerate((16, 4))]
    torch.cuda.synchronize()
    wrong = []

    def thread(i, bits):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(10):
                    got = work(i, bits)
                    torch.cuda.current_stream().synchronize()
                    if not all(torch.equal(a, b) for a, b in zip(got, want[i])):
                        wrong.append(i)
        except Exception as e:  # (an assertion in a thread would be lost)
            wrong.append(e)

    threads = [threading.Thread(target=thread, args=(i, bits)) for i, bits in enumerate((16, 4))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("bits", [16, 4])
def test_chains_without_other_kernels_between(bits, wide):
    """Each operator's kernel may be scheduled before the one in front of it has ended: appended rows, queries, outputs and
    lengths are what the calls before have written, eager and replayed, as when each call is waited for."""
    B, nq, nkv, hd, page, steps = 3, 8, 2, 128, 16, 40
    have = [30, 1, 555]
    pools, table, _, _ = _filled([h + steps for h in have], page, nkv, hd, bits, 1, 300 if wide else 0)
    first = [t.clone() for t in pools]
    cos, sin = ops.precompute_rope_table(hd, 1e4, 700, DEV)
    w = 1 + _randn(2, hd) / 8
    starts = [_ints([h + i for h in have]) for i in range(steps)]
    lens = [_ints([h + i + 1 for h in have]) for i in range(steps)]
    ctx = [_cum([h + i + 1 for h in have]) for i in range(steps)]
    totals = [sum(h + i + 1 for h in have) for i in range(steps)]
    cu = _cum([1] * B)
    x0 = _randn(3, B, nq, hd)
    outs = [torch.empty_like(x0) for _ in range(2 * steps)]
    rows = [tuple(torch.empty(totals[-1], nkv, hd, dtype=torch.float16, device=DEV) for _ in range(2)) for _ in range(2)]

    def run(wait):
        x = x0
        for i in range(steps):
            # the outputs of one step are the queries, keys and values of the next
            q, _ = ops.paged_kv_append(x, x[:, :nkv], x[:, nkv : 2 * nkv], *pools, table, starts[i], cos, sin, q_norm=w, k_norm=w)
            wait()
            ops.paged_decode_attention(q, *pools, table, lens[i], out=outs[2 * i])
            wait()
            k, v = (t[: totals[i]] for t in rows[i % 2])
            ops.paged_kv_read(*pools, table, ctx[i], totals[i], out=(k, v))
            wait()
            x = ops.prefill_attention(q, k, v, cu, cu_seqlens_k=ctx[i], out=outs[2 * i + 1])
            wait()

    def reset():
        for t, f in zip(pools, first):
            t.copy_(f)
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()

    reset()
    run(torch.cuda.synchronize)
    want, held = [o.clone() for o in outs], [t.clone() for t in pools]
    assert all(o.isfinite().all() and o.abs().sum() > 0 for o in want)
    graph = torch.cuda.CUDAGraph()
    reset()
    with torch.cuda.graph(graph):
        run(lambda: None)
    for again in (lambda: run(lambda: None), graph.replay) * 4:
        reset()
        again()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))
        assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(pools, held))


@pytest.mark.parametrize("bits", [16, 4])
def test_position_advanced_in_the_chain(bits):
    """A decode loop whose position and length the framework's own step kernel advances, nothing else between."""
    nq, nkv, hd, page, have, steps = 8, 2, 64, 16, 14, 120
    pools, table, _, _ = _filled([have + steps + 1], page, nkv, hd, bits, 1)
    first = [t.clone() for t in pools]
    cos, sin = ops.precompute_rope_table(hd, 1e4, 200, DEV)
    start, length, zero = _ints([have]), _ints([have + 1]), _ints([0])
    ids = torch.zeros(500, dtype=torch.int32, device=DEV)
    x0 = _randn(2, 1, nq, hd)
    outs = [torch.empty_like(x0) for _ in range(steps)]

    def run(wait):
        x = x0
        for out in outs:
            q, _ = ops.paged_kv_append(x, x[:, :nkv], x[:, nkv : 2 * nkv], *pools, table, start, cos, sin)
            wait()
            x = ops.paged_decode_attention(q, *pools, table, length, out=out)
            wait()
            for t in (start, length):
                _C.decode_step_advance(ids, t, zero, zero)
                wait()

    def reset():
        for t, f in zip((*pools, start, length), (*first, _ints([have]), _ints([have + 1]))):
            t.copy_(f)
        torch.cuda.synchronize()

    reset()
    run(torch.cuda.synchronize)
    assert start.item() == have + steps and length.item() == have + steps + 1
    want = [o.clone() for o in outs]
    assert not torch.equal(want[-1], want[-2])
    graph = torch.cuda.CUDAGraph()
    reset()
    with torch.cuda.graph(graph):
        run(lambda: None)
    for again in (lambda: run(lambda: None), graph.replay) * 4:
        reset()
        again()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))
