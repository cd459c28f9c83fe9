"""The host checks of the operators over caller-owned buffers: every call below is refused with
YUE2_ERR_INVALID before any launch, so none of the (made-up) addresses is ever used."""
import ctypes

import pytest

from yue2_rs_b200 import _lib

A = 1 << 20  # a 16-byte aligned address that nothing reads


def pool(**over):
    f = dict(base=A, pages=8, layers=2, kv=2, dim=64, dtype=0)
    f.update(over)
    return _lib.KvPool(f["base"], f["pages"], f["layers"], f["kv"], f["dim"], f["dtype"])


def refused(name, args, message):
    rc = getattr(_lib.lib(), name)(*args)
    assert rc == -1, (name, rc)
    assert message in _lib.last_error(), _lib.last_error()


BAD_POOLS = [(dict(base=0), "null KV pool"), (dict(base=A + 8), "16-byte aligned"), (dict(dtype=1), "bf16 or f16"),
             (dict(dim=80), "head dim"), (dict(pages=0), "out of range"), (dict(layers=0), "out of range"),
             (dict(kv=0), "out of range"), (dict(kv=1025), "out of range"), (dict(pages=(1 << 30) + 1), "out of range")]


def with_(args, names, over):
    a = list(args)
    for k, v in over.items():
        a[names.index(k)] = v
    return a


PACKED = ["q", "k", "v", "out", "cu", "seqs", "tokens", "heads", "kv", "dim", "qs", "ks", "vs", "os", "dtype", "causal", "scale",
          "status", "stream"]
PACKED_OK = [A, A, A, A, A, 2, 100, 4, 2, 64, 256, 128, 128, 256, 0, 1, 0.125, A, None]


@pytest.mark.parametrize("over,message", [
    (dict(q=0), "q must be"), (dict(k=A + 2), "k must be"), (dict(v=A + 8), "v must be"), (dict(out=0), "out must be"),
    (dict(cu=0), "null sequence offsets"), (dict(seqs=1025), "1,024 sequences"), (dict(tokens=(1 << 18) + 1), "262,144"),
    (dict(heads=3), "multiple of kv"), (dict(heads=0), "multiple of kv"), (dict(kv=0), "multiple of kv"),
    (dict(dim=256), "head dim"), (dict(dim=80), "head dim"), (dict(qs=252), "row stride"), (dict(qs=248), "row stride"),
    (dict(ks=0), "row stride"), (dict(vs=1 << 40), "row stride"), (dict(dtype=1), "bf16 or f16"),
    (dict(scale=float("nan")), "finite"), (dict(scale=float("inf")), "finite"), (dict(status=0), "status"),
    (dict(status=A + 1), "status")])
def test_packed(over, message):
    refused("yue2_attention_packed", with_(PACKED_OK, PACKED, over), message)


TREE = ["q", "rows", "heads", "qs", "pool", "layer", "table", "seqs", "pages", "context", "cu", "mask", "scale", "out", "os", "work",
        "bytes", "status", "stream"]


def tree_ok(p):
    return [A, 10, 4, 256, ctypes.addressof(p), 1, A, 3, 4, A, A, None, 0.125, A, 256, A, 1 << 40, A, None]


@pytest.mark.parametrize("over,message", [
    (dict(q=0), "q must be"), (dict(out=A + 4), "out must be"), (dict(heads=3), "multiple of kv"), (dict(layer=2), "layer outside"),
    (dict(table=0), "null page table"), (dict(context=0), "null page table"), (dict(cu=0), "null page table"),
    (dict(seqs=1025), "1,024 sequences"), (dict(pages=(1 << 24) + 1), "2^24 pages"), (dict(rows=65537), "64 drafted rows"),
    (dict(qs=100), "row stride"), (dict(scale=float("inf")), "finite"), (dict(status=0), "status")])
def test_tree(over, message):
    p = pool()
    refused("yue2_attention_tree", with_(tree_ok(p), TREE, over), message)


@pytest.mark.parametrize("over,message", BAD_POOLS + [(dict(dim=256), "head dim")])
def test_tree_pool(over, message):
    p = pool(**over)
    refused("yue2_attention_tree", tree_ok(p), message)
    refused("yue2_attention_tree", with_(tree_ok(p), TREE, dict(pool=None)), "null KV pool")


APPEND = ["qkv", "rows", "heads", "stride", "q_norm", "k_norm", "eps", "cos", "sin", "table_rows", "positions", "pool", "layer",
          "slots", "q_out", "qs", "k_out", "ks", "status", "stream"]


def append_ok(p):
    return [A, 10, 4, 512, A, A, 1e-6, A, A, 100, A, ctypes.addressof(p), 1, A, A, 256, A, 128, A, None]


@pytest.mark.parametrize("over,message", [
    (dict(qkv=0), "qkv must be"), (dict(stride=504), "row stride"), (dict(q_out=0), "q_out must be"), (dict(qs=8), "row stride"),
    (dict(k_out=A + 2), "k_out must be"), (dict(ks=120), "row stride"), (dict(q_norm=0), "go together"), (dict(k_norm=0), "go together"),
    (dict(positions=0), "positions, slots"), (dict(slots=0), "positions, slots"), (dict(cos=A + 4), "16-byte aligned cos"),
    (dict(heads=0), "heads must"), (dict(layer=2), "layer outside"), (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"),
    (dict(status=0), "status"), (dict(rows=1 << 31), "below 2^31")])
def test_append(over, message):
    p = pool()
    refused("yue2_qk_rope_append", with_(append_ok(p), APPEND, over), message)


@pytest.mark.parametrize("over,message", BAD_POOLS)
def test_pools(over, message):
    p = pool(**over)
    ref = ctypes.addressof(p)
    refused("yue2_qk_rope_append", append_ok(p), message)
    refused("yue2_kv_copy", [ref, A, A, None, 4, A, None], message)
    refused("yue2_kv_gather", [ref, A, 4, A, 4, A, A, A, 2, 8, A, None], message)


def test_copy_and_gather():
    p = pool()
    ref = ctypes.addressof(p)
    refused("yue2_kv_copy", [ref, 0, A, None, 4, A, None], "null page list")
    refused("yue2_kv_copy", [ref, A, 0, None, 4, A, None], "null page list")
    refused("yue2_kv_copy", [ref, A, A, None, 65536, A, None], "65,535")
    refused("yue2_kv_copy", [ref, A, A, None, 4, 0, None], "status")
    for i, what in ((1, 0), (5, 0), (6, 0), (7, 0)):
        args = [ref, A, 4, A, 4, A, A, A, 2, 8, A, None]
        args[i] = what
        refused("yue2_kv_gather", args, "null table or list")
    refused("yue2_kv_gather", [ref, A, 4, A, 4, A, A, A, 65536, 8, A, None], "65,535")
    refused("yue2_kv_gather", [ref, A, 4, A, 4, A, A, A, 2, 1 << 31, A, None], "2^31")
    refused("yue2_kv_gather", [ref, A, 1 << 27, A, 4, A, A, A, 2, 8, A, None], "2^26")
    refused("yue2_kv_gather", [ref, A, 4, A, 4, A, A, A, 2, 8, A + 2, None], "status")


def test_empty_calls_are_done_without_a_launch():
    p = pool()
    ref = ctypes.addressof(p)
    L = _lib.lib()
    assert L.yue2_kv_copy(ref, 0, 0, None, 0, A, None) == 0
    assert L.yue2_kv_gather(ref, 0, 0, 0, 0, 0, 0, 0, 0, 0, A, None) == 0
    assert L.yue2_attention_packed(*with_(PACKED_OK, PACKED, dict(tokens=0, q=0, k=0, v=0, out=0))) == 0
    assert L.yue2_attention_packed(*with_(PACKED_OK, PACKED, dict(seqs=0))) == 0
    assert L.yue2_attention_tree(*with_(tree_ok(p), TREE, dict(rows=0, q=0, out=0))) == 0
    assert L.yue2_qk_rope_append(*with_(append_ok(p), APPEND, dict(rows=0, qkv=0, q_out=0))) == 0
