"""What the torch wrappers of the operators owe autograd and the status word."""
import pytest
import torch

from test_gpu_ops import DEV, ints, offsets, ops, randn  # noqa: F401 (ops is a fixture)
from yue2_rs_b200 import Yue2Error

pytestmark = pytest.mark.gpu


def append_args(dtype=torch.bfloat16):
    qkv, cos = randn((10, 8, 64), dtype, 1), torch.ones(16, 32, device=DEV)
    return qkv, cos, cos.clone(), ints(range(10)), ints(range(10), torch.int64)


def calls(ops, data, cos=None, sin=None):
    """One call of every operator that takes the pool, by name."""
    qkv, c, s, pos, slots = append_args()
    c, s = c if cos is None else cos, s if sin is None else sin
    pool, table = ops.KvPool(data), ints([[0, 1]])
    return {"append": lambda: ops.qk_rope_append(qkv, None, None, 0.0, c, s, pos, pool, 0, slots),
            "tree": lambda: ops.attention_tree(qkv[:, :4], pool, 0, table, ints([20]), offsets([10])),
            "copy": lambda: ops.kv_copy(pool, ints([0]), ints([1])),
            "gather": lambda: ops.kv_gather(pool, table, None, ints([0]), offsets([1]), ints([5]))}


@pytest.mark.parametrize("name", ["append", "tree", "copy", "gather"])
def test_a_pool_that_asks_for_a_gradient_is_refused(ops, name):
    data = randn((2, 1, 2, 2, 64, 64), torch.bfloat16, 1).requires_grad_()
    call = calls(ops, data)[name]
    with pytest.raises(Yue2Error, match="gradient"):
        call()
    with torch.no_grad():
        call()
    ops.check_status()


@pytest.mark.parametrize("which", ["cos", "sin"])
def test_tables_that_ask_for_a_gradient_are_refused(ops, which):
    table = torch.ones(16, 32, device=DEV, requires_grad=True)
    call = calls(ops, randn((2, 1, 2, 2, 64, 64), torch.bfloat16, 1), **{which: table})["append"]
    with pytest.raises(Yue2Error, match="gradient"):
        call()
    with torch.no_grad():
        call()
    ops.check_status()


@pytest.mark.parametrize("which", ["q", "k", "v", "pool", "qkv", "gain", "cos"])
def test_tangents_are_refused(ops, which):
    import torch.autograd.forward_ad as fwd
    q, k = randn((10, 4, 64), torch.bfloat16, 1), randn((10, 2, 64), torch.bfloat16, 2)
    data, gain = randn((2, 1, 2, 2, 64, 64), torch.bfloat16, 3), torch.ones(64, device=DEV)
    qkv, cos, sin, pos, slots = append_args()
    cu = offsets([10])

    def dual(t, name):
        return fwd.make_dual(t, torch.ones_like(t)) if name == which else t

    with torch.no_grad(), fwd.dual_level():
        with pytest.raises(Yue2Error, match="gradient"):
            if which in ("q", "k", "v"):
                ops.attention_packed(dual(q, "q"), dual(k, "k"), dual(k, "v"), cu)
            elif which == "pool":
                ops.attention_tree(q, ops.KvPool(dual(data, "pool")), 0, ints([[0, 1]]), ints([0]), cu)
            else:
                ops.qk_rope_append(dual(qkv, "qkv"), dual(gain, "gain"), gain, 1e-6, dual(cos, "cos"), sin, pos, ops.KvPool(data), 0, slots)
        ops.attention_packed(q, k, k, cu)  # tensors without a tangent are taken at this level too
    ops.check_status()


def test_what_is_written_counts_as_modified(ops):
    # a product that saved the buffer for its backward pass must not use what is there later
    q, k = randn((10, 4, 64), torch.bfloat16, 1), randn((10, 2, 64), torch.bfloat16, 2)
    cu, table = offsets([10]), ints([[0, 1]])
    qkv, cos, sin, pos, slots = append_args()
    writes = {
        "packed": lambda b, p: ops.attention_packed(q, k, k, cu, out=b),
        "tree": lambda b, p: ops.attention_tree(q, p, 0, table, ints([0]), cu, out=b),
        "q_out": lambda b, p: ops.qk_rope_append(qkv, None, None, 0.0, cos, sin, pos, p, 0, slots, q_out=b),
        "k_out": lambda b, p: ops.qk_rope_append(qkv, None, None, 0.0, cos, sin, pos, p, 0, slots, k_out=b[:, :2])}
    for name, write in writes.items():
        b = randn((10, 4, 64), torch.bfloat16, 5)
        w = torch.ones_like(b, requires_grad=True)
        y = (w * b).sum()
        write(b, ops.KvPool(randn((2, 1, 2, 2, 64, 64), torch.bfloat16, 3)))
        with pytest.raises(RuntimeError, match="modified by an inplace"):
            y.backward()
            pytest.fail(f"{name} went unnoticed")
    for name in ("append", "copy", "gather"):
        data = randn((2, 1, 2, 2, 64, 64), torch.bfloat16, 3)
        w = torch.ones_like(data, requires_grad=True)
        y = (w * data).sum()
        calls(ops, data)[name]()
        with pytest.raises(RuntimeError, match="modified by an inplace"):
            y.backward()
            pytest.fail(f"{name} went unnoticed")
    ops.check_status()


def test_a_first_call_in_inference_mode_reports_as_any(ops, monkeypatch):
    monkeypatch.setattr(ops, "_status", {})
    data = randn((2, 1, 2, 1, 64, 64), torch.bfloat16, 1)
    with torch.inference_mode():
        ops.kv_copy(ops.KvPool(data), ints([0]), ints([7]))
    with pytest.raises(Yue2Error, match="page index"):
        ops.check_status()
    ops.check_status()  # cleared
    with torch.inference_mode():
        ops.kv_copy(ops.KvPool(torch.zeros_like(data)), ints([-1]), ints([1]))
        with pytest.raises(Yue2Error, match="page index"):
            ops.check_status()
        ops.check_status()


def test_a_check_inside_a_capture_is_refused_and_the_capture_lives(ops):
    data = randn((2, 1, 2, 1, 64, 64), torch.bfloat16, 1)
    pool, src, dst = ops.KvPool(data), ints([0]), ints([1])
    ops.kv_copy(pool, src, dst)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(Yue2Error, match="capture"):
            ops.check_status()
        ops.kv_copy(pool, src, dst)
    data[0] = 3
    graph.replay()
    ops.check_status()
    assert (data[1] == 3).all()


def test_odd_arguments_raise_the_wrappers_error(ops):
    pool = ops.KvPool(randn((2, 1, 2, 2, 64, 64), torch.bfloat16, 3))
    empty = torch.empty((4, 2, 0), dtype=torch.bfloat16, device=DEV)
    for f in (lambda: ops.attention_packed(empty, empty, empty, offsets([4])),
              lambda: ops.kv_copy(pool, torch.tensor(0, dtype=torch.int32, device=DEV), torch.tensor(1, dtype=torch.int32, device=DEV))):
        with pytest.raises(Yue2Error):
            f()
