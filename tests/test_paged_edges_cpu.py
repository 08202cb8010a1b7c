"""Sizes of the decode workspace at the borders of the split, which the Python front end knows too."""
from soinfer import _C


def test_front_end_asks_for_a_workspace_exactly_where_one_is_needed():
    need = _C.lib().soinfer_paged_decode_workspace_bytes
    for hd, most in ((64, _C.PAGED_CLUSTER_UNITS), (128, _C.PAGED_CLUSTER_UNITS_128)):
        for nq, nkv, units in ((8, 1, 1), (2, 2, 2), (17, 1, 3), (40, 8, 8), (18, 2, 4)):
            seqs = most // units
            assert need(seqs, nq, nkv, hd, _C.PAGED_CLUSTER_POSITIONS) == 0
            assert need(seqs + 1, nq, nkv, hd, 64) > 0
            assert need(seqs, nq, nkv, hd, _C.PAGED_CLUSTER_POSITIONS + 16) > 0
