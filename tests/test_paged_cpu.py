"""The paged-cache and prompt-attention entry points without a GPU: argument
errors come back as status codes before anything is launched, sizes of the
workspace, and the Python front end's checks on CPU tensors."""
import pytest
import torch

import soinfer.ops as ops
from soinfer import _C

P = 0x10000


def _cache(**kw):
    f = dict(k_pages=P, v_pages=P, block_table=P, table_stride=4, table_cols=4, num_pages=8, num_kv_heads=2, page_size=16,
             head_dim=128, bits=16)
    f.update(kw)
    order = ("k_pages", "v_pages", "block_table", "table_stride", "table_cols", "num_pages", "num_kv_heads", "page_size",
             "head_dim", "bits")
    return _C._PAGED_CACHE.pack(*(f[n] or 0 for n in order))


def _rows(data=P, token=1024, head=128):
    return _C._ROWS.pack(data or 0, token, head)


def _err():
    return _C.lib().soinfer_last_error().decode()


@pytest.mark.parametrize("bad,msg", [(dict(head_dim=96), "head_dim"), (dict(page_size=24), "power of two"),
                                     (dict(page_size=8), "power of two"), (dict(bits=8), "bits"),
                                     (dict(num_kv_heads=0), "num_kv_heads"), (dict(table_stride=3), "table_stride"),
                                     (dict(num_pages=-1), "num_pages"), (dict(k_pages=None), "null pages"),
                                     (dict(block_table=None), "null block_table"), (dict(v_pages=P + 2), "16-byte")])
def test_bad_caches_are_refused_by_every_entry(bad, msg):
    lib, c = _C.lib(), _cache(**bad)
    assert lib.soinfer_paged_kv_append(c, _rows(), _rows(), _rows(), P, P, 1, 4, 1, P, P, P, P, 8, None, None, 1e-6, None) == 1
    assert msg in _err()
    assert lib.soinfer_paged_kv_read(c, P, 1, 1, P, P, None) == 1 and msg in _err()
    assert lib.soinfer_paged_decode_attention(c, _rows(), P, 1, 4, P, P, 1 << 30, None) == 1 and msg in _err()


def test_append_arguments():
    f = _C.lib().soinfer_paged_kv_append
    ok = [_cache(), _rows(), _rows(), _rows(), P, P, 1, 4, 1, P, P, P, P, 8, None, None, 1e-6, None]

    def refused(msg, **kw):
        a = list(ok)
        for i, v in kw.items():
            a[int(i[1:])] = v
        assert f(*a) == 1 and msg in _err(), _err()

    refused("null cache", _0=None)
    refused("null q", _1=None)
    refused("null k", _2=_rows(data=None))
    refused("multiples of 8", _3=_rows(head=130))
    refused("multiples of 8", _2=_rows(token=-128))
    refused("16-byte", _1=_rows(data=P + 2))
    refused("q_out", _4=None)
    refused("k_out", _5=P + 2)
    refused("tokens", _6=-1)
    refused("num_q_heads", _7=-1)
    refused("null start", _10=None)
    refused("null start", _11=None)
    refused("table_rows", _13=0)
    refused("16-byte", _14=P + 2)
    refused("eps", _16=-1.0)
    a = list(ok)
    a[6] = 0
    assert f(*a) == 0  # no tokens: nothing to do


def test_read_decode_and_prefill_arguments():
    lib = _C.lib()
    assert lib.soinfer_paged_kv_read(_cache(), None, 1, 1, P, P, None) == 1 and "null" in _err()
    assert lib.soinfer_paged_kv_read(_cache(), P, 1, 1, P + 2, P, None) == 1 and "16-byte" in _err()
    assert lib.soinfer_paged_kv_read(_cache(), P, 1, 0, None, None, None) == 0
    need = lib.soinfer_paged_decode_workspace_bytes(3, 8, 2, 128, 100_000)
    assert need >= 3 * 8 * 130 * 4 and lib.soinfer_paged_decode_workspace_bytes(3, 7, 2, 128, 100_000) == 0
    # the front end asks for a workspace exactly where one is needed
    assert lib.soinfer_paged_decode_workspace_bytes(3, 8, 2, 128, _C.PAGED_CLUSTER_POSITIONS) == 0
    assert lib.soinfer_paged_decode_workspace_bytes(3, 8, 2, 128, _C.PAGED_CLUSTER_POSITIONS + 16) > 0
    most = _C.PAGED_CLUSTER_UNITS  # sequences x kv heads (x groups of 8 query heads of a kv head)
    for seqs, nq, nkv in ((most, 8, 1), (most // 2, 2, 2), (most // 3, 17, 1)):
        assert lib.soinfer_paged_decode_workspace_bytes(seqs, nq, nkv, 64, 64) == 0
    for seqs, nq, nkv in ((most + 1, 8, 1), (most // 2 + 1, 2, 2), (most // 3 + 1, 17, 1)):
        assert lib.soinfer_paged_decode_workspace_bytes(seqs, nq, nkv, 64, 64) > 0
    d = lib.soinfer_paged_decode_attention
    long = dict(table_cols=10_000, table_stride=10_000)
    assert d(_cache(**long), _rows(), P, 3, 8, P, P, need - 1, None) == 1 and "workspace" in _err()
    assert d(_cache(**long), _rows(), P, 3, 8, P, None, need, None) == 1 and "workspace" in _err()
    assert d(_cache(), _rows(), P, 3, 7, P, P, need, None) == 1 and "multiple of num_kv_heads" in _err()
    assert d(_cache(), _rows(), P, 40000, 8, P, P, 1 << 40, None) == 1 and "num_seqs" in _err()
    assert d(_cache(), _rows(), None, 3, 8, P, P, need, None) == 1 and "null" in _err()
    assert d(_cache(), None, None, 0, 8, None, None, 0, None) == 0
    p = lib.soinfer_prefill_attention
    assert p(_rows(), _rows(), _rows(), P, 4, 4, 1, P, P, 8, 2, 96, None) == 1 and "head_dim" in _err()
    assert p(_rows(), _rows(), _rows(), P, 4, 4, 1, P, P, 8, 3, 64, None) == 1 and "multiple" in _err()
    assert p(_rows(), _rows(), None, P, 4, 4, 1, P, P, 8, 2, 64, None) == 1 and "null v" in _err()
    assert p(_rows(head=4), _rows(), _rows(), P, 4, 4, 1, P, P, 8, 2, 64, None) == 1 and "multiples of 8" in _err()
    assert p(_rows(), _rows(), _rows(), P, 4, 4, 1, None, P, 8, 2, 64, None) == 1 and "null" in _err()
    assert p(_rows(), _rows(), _rows(), P, -1, 4, 1, P, P, 8, 2, 64, None) == 1 and "tokens" in _err()
    assert p(None, None, None, None, 0, 0, 0, None, None, 8, 2, 64, None) == 0


def test_front_end_refuses_cpu_tensors_and_knows_its_layouts():
    k, v = ops.paged_kv_alloc(3, 2, 32, 128, 4, "cpu")
    assert k.shape == (3, 2, 32, 72) and v.shape == (3, 2, 32, 66) and k.dtype == torch.uint8
    k, v = ops.paged_kv_alloc(3, 2, 32, 64, 16, "cpu")
    assert k.shape == v.shape == (3, 2, 32, 64) and k.dtype == torch.float16
    q = torch.zeros(1, 2, 64, dtype=torch.float16)
    t, n = torch.zeros(1, 1, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    for call in (lambda: ops.paged_decode_attention(q, k, v, t, n), lambda: ops.prefill_attention(q, q, q, torch.zeros(2)),
                 lambda: ops.paged_kv_read(k, v, t, n, 1)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()
    with pytest.raises(RuntimeError, match="64 or 128"):
        ops.paged_kv_alloc(1, 1, 16, 256, 16, "cpu")
