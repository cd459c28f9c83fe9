"""Lists of the operators whose addresses are not multiples of their entries' size are refused by
the host, before any launch could read them (none of the made-up addresses is ever used)."""
import ctypes

import pytest

from test_ops_refusals import A, APPEND, PACKED, PACKED_OK, TREE, append_ok, pool, refused, tree_ok, with_

COPY = ["pool", "src", "dst", "count", "n", "status", "stream"]
GATHER = ["pool", "src_table", "src_pages", "dst_table", "dst_pages", "begin", "cu", "keep", "seqs", "total", "status", "stream"]


def test_packed():
    for off in (1, 2, 3):
        refused("yue2_attention_packed", with_(PACKED_OK, PACKED, dict(cu=A + off)), "aligned")


@pytest.mark.parametrize("name,size", [("table", 4), ("context", 4), ("cu", 4), ("mask", 8)])
def test_tree(name, size):
    p = pool()
    for off in range(1, size):
        refused("yue2_attention_tree", with_(tree_ok(p), TREE, {name: A + off}), "aligned")


@pytest.mark.parametrize("name,size", [("positions", 4), ("slots", 8)])
def test_append(name, size):
    p = pool()
    for off in range(1, size):
        refused("yue2_qk_rope_append", with_(append_ok(p), APPEND, {name: A + off}), "aligned")


@pytest.mark.parametrize("name", ["src", "dst", "count"])
def test_copy(name):
    p = pool()
    ok = [ctypes.addressof(p), A, A, A, 4, A, None]
    for off in (1, 2, 3):
        refused("yue2_kv_copy", with_(ok, COPY, {name: A + off}), "aligned")


@pytest.mark.parametrize("name", ["src_table", "dst_table", "begin", "cu", "keep"])
def test_gather(name):
    p = pool()
    ok = [ctypes.addressof(p), A, 4, A, 4, A, A, A, 2, 8, A, None]
    for off in (1, 2, 3):
        refused("yue2_kv_gather", with_(ok, GATHER, {name: A + off}), "aligned")
