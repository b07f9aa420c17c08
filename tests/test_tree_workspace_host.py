"""CPU checks of the bytes that a call of tree decoding asks for: one partial sum for each group of 2048 keys in large calls,
four where a group's strands have workgroups of their own, one for each chunk where requests may have many rows."""
import ctypes

import pytest

from vllm_exact import _native as nx


def call_workspace(n, tokens, H, KV, D, max_nodes, max_len):
    out = ctypes.c_size_t()
    rc = nx.lib().vxa_tree_decode_call_workspace(n, tokens, H, KV, D, max_nodes, max_len, ctypes.byref(out))
    return rc, out.value


def parts(n, KV, G, D, max_nodes, max_len):
    tokens = n * max_nodes
    rc, size = call_workspace(n, tokens, KV * G, KV, D, max_nodes, max_len)
    assert rc == nx.VXA_OK and size <= nx.tree_workspace(tokens, KV * G, D, max_len)
    unit = tokens * KV * G * (D + 2) * 4
    assert size % unit == 0
    return size // unit


def test_sizes_on_both_sides_of_each_switch():
    # up to four segments of 512 keys: one group, its segments counted
    assert [parts(1, 8, 4, 128, 1, x) for x in (512, 513, 1025, 2048)] == [0, 2, 3, 4]
    # a group for each 2048 keys and fewer than 256 workgroups: a workgroup for each strand
    assert [parts(1, 8, 4, 128, 1, x) for x in (2049, 16384, 131072 // 2 - 2048)] == [8, 32, 124]
    # from 256 workgroups of whole groups on
    assert parts(3, 8, 4, 128, 1, 10 * 2048) == 40 and parts(4, 8, 4, 128, 1, 8 * 2048) == 8
    # 16 rows a workgroup up to 16 rows, 32 beyond: 1, 1, 2 and 3 row blocks of 120 groups
    assert [parts(3, 4, 4, 128, x, 10 * 2048) for x in (4, 8, 16, 24)] == [40, 40, 40, 10]
    # requests of more than 96 rows (32 at 256 dims): a partial sum for each chunk of 512 keys, 1024 past 4096
    assert [parts(64, 8, 4, 128, x, 8192) for x in (24, 25)] == [4, 8]
    assert [parts(64, 8, 4, 256, x, 8192) for x in (8, 9)] == [4, 8]
    assert [parts(64, 8, 4, 128, 64, x) for x in (2049, 4096, 4097, 9000, 131072)] == [5, 8, 8, 9, 128]


def test_a_large_call():
    """4096 nodes of 512 requests, 32 heads of 128 dims, lengths up to 131072: a quarter of what any call may need."""
    assert call_workspace(512, 4096, 32, 8, 128, 8, 131072) == (nx.VXA_OK, 4096 * 32 * 64 * 130 * 4)
    assert nx.tree_workspace(4096, 32, 128, 131072) == 4 * 4096 * 32 * 64 * 130 * 4


def test_refusals():
    good = dict(n=2, tokens=10, H=8, KV=2, D=128, max_nodes=5, max_len=5000)
    for bad in (dict(n=-1), dict(tokens=-1), dict(H=0), dict(KV=0), dict(H=7), dict(D=0), dict(max_nodes=-1), dict(max_len=-1)):
        assert call_workspace(**{**good, **bad})[0] == nx.VXA_ERR_ARG, bad
    for bad in (dict(n=1 << 40), dict(tokens=1 << 40), dict(H=1 << 17), dict(D=96), dict(max_nodes=65), dict(max_len=1 << 31)):
        assert call_workspace(**{**good, **bad})[0] == nx.VXA_ERR_UNSUPPORTED, bad
    with pytest.raises(NotImplementedError):  # more bytes than there are numbers for
        nx.tree_workspace(1 << 50, 64, 128, 1 << 30)
    assert nx.lib().vxa_tree_decode_call_workspace(2, 10, 8, 2, 128, 5, 5000, None) == nx.VXA_ERR_ARG
