"""The operators over caller-owned buffers (yue2_rs_b200.ops) against plain 64-bit forms.

Tolerances, derived before the first run. With u = eps / 2 of the type (bf16 2^-8, f16 2^-11):
an attention output is rounded once (u |out|), each probability at most once more (u A with
A = sum_j p_j |v_j|), and a score carries the f32 error of a dim-term dot product,
delta = (dim + 4) 2^-24 scale max_j sum_d |q_d k_jd|, which moves every weight by at most
2 delta, plus 2^-20 for exp and the f32 sums; f16 probabilities below the normal range are off
by up to 2^-25 of the largest one each: 2^-25 sum_j |v_j|. An appended head is rounded once; its
f32 steps (norm, two products, one sum) stay below 2^-18 (|a| + |b|)."""
import math
import random

import numpy as np
import pytest
import torch

from yue2_rs_b200 import Yue2Error

pytestmark = pytest.mark.gpu

DEV = "cuda"
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


@pytest.fixture(scope="module")
def ops():
    from yue2_rs_b200 import ops as o
    o.check_status()
    return o


def randn(shape, dtype, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randn(shape, generator=g, device=DEV).to(dtype)


def ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype).to(DEV)


def offsets(lens, first=0):
    return ints(np.concatenate([[0], np.cumsum(lens)]) + first)


def attend(q, k, v, see, scale):
    """Rows q [n, D] over keys k, v [m, D] (f64) with the visible set see [n, m]: the output
    and the tolerance of the head. Masked places are never touched."""
    n, dim = q.shape
    q64, k64, v64 = q.double(), k.double(), v.double()
    live = see.any(0)
    k64 = torch.where(live[:, None], k64, 0.0)
    v64 = torch.where(live[:, None], v64, 0.0)
    s = q64 @ k64.T * scale
    s = torch.where(see, s, -math.inf)
    m = s.amax(1, keepdim=True)
    p = torch.exp(s - torch.where(torch.isinf(m), 0.0, m))
    p = torch.where(see, p, 0.0)
    tot = p.sum(1, keepdim=True)
    p = p / torch.where(tot > 0, tot, 1.0)
    out = p @ v64
    u = U[q.dtype]
    delta = (dim + 4) * 2.0 ** -24 * abs(scale) * (q64.abs() @ k64.abs().T).where(see, torch.zeros((), device=q.device, dtype=torch.float64)).amax(1, keepdim=True)
    tol = u * out.abs() + (u + 2 * delta + 2.0 ** -20) * (p @ v64.abs())
    if q.dtype == torch.float16:
        tol = tol + 2.0 ** -25 * (see.double() @ v64.abs())
    return out, tol + 1e-30


def close(got, want, tol, what=""):
    bad = ~((got.double() - want).abs() <= tol)
    assert not bad.any(), (what, int(bad.sum()), float((got.double() - want).abs().max()), bad.nonzero()[:4].tolist())


# ------------------------------------------------------------------ packed prompts
def packed_reference(q, k, v, lens, first, causal, scale):
    heads, kv = q.shape[1], k.shape[1]
    want = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(want)
    at = first
    for n in lens:
        i = torch.arange(n, device=q.device)
        see = i[None] <= i[:, None] if causal else torch.ones((n, n), dtype=torch.bool, device=q.device)
        for h in range(heads if n else 0):
            g = h // (heads // kv)
            want[at:at + n, h], tol[at:at + n, h] = attend(q[at:at + n, h], k[at:at + n, g], v[at:at + n, g], see, scale)
        at += n
    return want, tol


def check_packed(ops, lens, heads, kv, dim, dtype, causal, first=0, behind=0, seed=1, scale=None, mag=1.0):
    total = first + sum(lens) + behind
    qkv = randn((total, heads + 2 * kv, dim), dtype, seed) * mag
    q, k, v = qkv[:, :heads], qkv[:, heads:heads + kv], qkv[:, heads + kv:]
    if behind:
        qkv[first + sum(lens):] = float("nan")
    if first:
        qkv[:first] = float("inf")
    out = torch.full((total, heads, dim), 7.0, dtype=dtype, device=DEV)
    got = ops.attention_packed(q, k, v, offsets(lens, first), causal=causal, scale=scale, out=out)
    assert got is out
    ops.check_status()
    want, tol = packed_reference(q, k, v, lens, first, causal, 1 / math.sqrt(dim) if scale is None else scale)
    a, b = first, first + sum(lens)
    close(out[a:b], want[a:b], tol[a:b])
    assert (out[:a] == 7).all() and (out[b:] == 7).all()


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lens", [[1], [2], [63], [127], [128], [129], [255, 1, 0, 257], [1] * 37, [384, 511], [513, 3, 640]])
def test_packed_lengths(ops, lens, causal):
    check_packed(ops, lens, 4, 2, 64, torch.bfloat16, causal)
    check_packed(ops, lens, 3, 1, 128, torch.bfloat16, causal, seed=2)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads,kv,dim", [(24, 8, 128), (8, 2, 128), (4, 2, 64), (3, 3, 64), (8, 1, 128), (1, 1, 64), (10, 2, 64)])
def test_packed_layouts(ops, heads, kv, dim, dtype):
    check_packed(ops, [130, 1, 259], heads, kv, dim, dtype, True, first=3, behind=5)
    check_packed(ops, [70, 301], heads, kv, dim, dtype, False, first=1, behind=130)


@pytest.mark.parametrize("causal", [True, False])
def test_packed_longer(ops, causal):
    check_packed(ops, [1500, 17, 2300], 6, 2, 128, torch.bfloat16, causal, behind=40)


def test_packed_many_sequences(ops):
    rng = random.Random(3)
    check_packed(ops, [rng.choice([0, 1, 2, 5, 64, 130]) for _ in range(300)], 2, 1, 64, torch.float16, True)


@pytest.mark.parametrize("scale", [0.0, -0.25, 3.0])
def test_packed_scales(ops, scale):
    check_packed(ops, [200, 333], 4, 2, 64, torch.bfloat16, True, scale=scale)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_packed_peaked_scores(ops, dtype):
    # scores of several hundred: the running maximum moves far and most weights vanish
    check_packed(ops, [300, 520], 4, 2, 128, dtype, True, mag=8.0)
    check_packed(ops, [300, 520], 4, 2, 128, dtype, False, mag=8.0)


def test_packed_growing_scores(ops):
    # every next key scores higher, so each tile raises the running maximum
    n, dim = 700, 64
    k = torch.zeros((n, 1, dim), dtype=torch.bfloat16, device=DEV)
    k[:, 0, 0] = torch.arange(n, device=DEV) / 4
    q = torch.zeros_like(k)
    q[:, 0, 0] = 8
    v = randn((n, 1, dim), torch.bfloat16, 5)
    got = ops.attention_packed(q, k, v, offsets([n]))
    want, tol = packed_reference(q, k, v, [n], 0, True, 1 / 8)
    close(got, want, tol)


@pytest.mark.parametrize("value", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("dim", [64, 128])
def test_packed_nonfinite_values_stay_with_the_rows_that_see_them(ops, value, dim):
    n, at = 400, 137
    q, k, v = randn((n, 4, dim), torch.bfloat16, 1), randn((n, 2, dim), torch.bfloat16, 2), randn((n, 2, dim), torch.bfloat16, 3)
    clean = ops.attention_packed(q, k, v, offsets([150, 250]))
    v[at, 1, 5] = value
    got = ops.attention_packed(q, k, v, offsets([150, 250]))
    ops.check_status()
    sees = torch.zeros((n, 4, dim), dtype=torch.bool, device=DEV)
    sees[at:150, 2:, 5] = True
    assert torch.equal(got[~sees], clean[~sees])
    assert torch.equal(torch.isnan(got[sees]), torch.full_like(got[sees], math.isnan(value), dtype=torch.bool))
    if not math.isnan(value):
        assert (got[sees] == value).all()


@pytest.mark.parametrize("value", [float("inf"), float("nan")])
def test_packed_nonfinite_keys_are_masked(ops, value):
    n, at = 300, 201
    q, k, v = randn((n, 2, 128), torch.bfloat16, 1), randn((n, 1, 128), torch.bfloat16, 2), randn((n, 1, 128), torch.bfloat16, 3)
    clean = ops.attention_packed(q, k, v, offsets([n]))
    k[at] = value
    got = ops.attention_packed(q, k, v, offsets([n]))
    assert torch.equal(got[:at], clean[:at])
    assert torch.isnan(got[at]).all()  # inf - inf or NaN in its own score


@pytest.mark.parametrize("value", [float("inf"), float("nan")])
@pytest.mark.parametrize("at", [0, 6, 7, 13, 14, 15, 31, 64, 127, 128, 255, 511])
def test_packed_nonfinite_scores_make_their_rows_nan(ops, at, value):
    # in tiles that every row sees and in the last, at places of either way of exponentials
    n = 700
    q, k, v = randn((n, 1, 128), torch.bfloat16, 1), randn((n, 1, 128), torch.bfloat16, 2), randn((n, 1, 128), torch.bfloat16, 3)
    clean = ops.attention_packed(q, k, v, offsets([n]))
    k[at] = value
    got = ops.attention_packed(q, k, v, offsets([n]))
    assert torch.equal(got[:at], clean[:at])
    assert torch.isnan(got[at:]).all()


@pytest.mark.parametrize("dtype,huge", [(torch.bfloat16, 3.0e38), (torch.float16, 65504.0)])
def test_packed_huge_values_in_masked_places(ops, dtype, huge):
    q, k, v = randn((500, 2, 64), dtype, 1), randn((500, 1, 64), dtype, 2), randn((500, 1, 64), dtype, 3)
    clean = ops.attention_packed(q, k, v, offsets([300, 150]))[:450].clone()
    v[100:300] = huge
    k[100:300] = huge / 2 if dtype == torch.bfloat16 else 100.0
    v[450:], k[450:] = -huge, huge
    got = ops.attention_packed(q, k, v, offsets([300, 150]))
    assert torch.equal(got[:100], clean[:100]) and torch.equal(got[300:450], clean[300:450])


def test_packed_at_the_limits(ops):
    rng = random.Random(8)
    lens = [rng.choice([0, 1, 2, 3, 7]) for _ in range(1024)]
    check_packed(ops, lens, 1, 1, 64, torch.bfloat16, True, behind=2)
    # 262,144 tokens, most of them behind the last sequence
    n = 1 << 18
    q = randn((n, 1, 64), torch.bfloat16, 1)
    lens = [500, 0, 77]
    out = torch.full_like(q, 2.0)
    ops.attention_packed(q, q, q, offsets(lens, n - 600), out=out)
    want, tol = packed_reference(q[n - 600:], q[n - 600:], q[n - 600:], lens, 0, True, 1 / 8)
    close(out[n - 600:n - 23], want[:577], tol[:577])
    assert (out[:n - 600] == 2).all() and (out[n - 23:] == 2).all()
    big = torch.empty((n + 1, 1, 64), dtype=torch.bfloat16, device=DEV)
    with pytest.raises(Yue2Error, match="262,144"):
        ops.attention_packed(big, big, big, offsets([5]))
    with pytest.raises(Yue2Error, match="1,024"):
        ops.attention_packed(q, q, q, offsets([1] * 1025))


def test_packed_output_over_its_queries(ops):
    # every unit has its queries before it writes, and no other reads them
    qkv = randn((700, 8, 128), torch.bfloat16, 1)
    q, k, v = qkv[:, :4], qkv[:, 4:6], qkv[:, 6:]
    want = ops.attention_packed(q, k, v, offsets([400, 300]))
    ops.attention_packed(q, k, v, offsets([400, 300]), out=q)
    assert torch.equal(q, want)


def test_packed_repeats_bit_for_bit_and_on_another_stream(ops):
    q, k, v = randn((900, 8, 128), torch.bfloat16, 1), randn((900, 2, 128), torch.bfloat16, 2), randn((900, 2, 128), torch.bfloat16, 3)
    cu = offsets([300, 1, 599])
    a = ops.attention_packed(q, k, v, cu)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        b = ops.attention_packed(q, k, v, cu)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(a, b)


def test_packed_captured_with_lengths_that_change(ops):
    q, k, v = randn((700, 4, 64), torch.float16, 1), randn((700, 2, 64), torch.float16, 2), randn((700, 2, 64), torch.float16, 3)
    cu = offsets([350, 350])
    out = torch.zeros_like(q)
    ops.attention_packed(q, k, v, cu, out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.attention_packed(q, k, v, cu, out=out)
    for lens in ([350, 350], [1, 699], [640, 0], [0, 0]):
        cu.copy_(offsets(lens))
        out.fill_(9)
        graph.replay()
        want, tol = packed_reference(q, k, v, lens, 0, True, 1 / 8)
        n = sum(lens)
        close(out[:n], want[:n], tol[:n])
        assert (out[n:] == 9).all()
    ops.check_status()


@pytest.mark.parametrize("cu", [[0, 50, 40, 90], [0, 50, 101, 101], [-1, 50, 60, 70], [0, 1 << 30, 60, 70]])
def test_packed_bad_offsets_are_reported(ops, cu):
    q, k, v = randn((100, 2, 64), torch.bfloat16, 1), randn((100, 1, 64), torch.bfloat16, 2), randn((100, 1, 64), torch.bfloat16, 3)
    ops.attention_packed(q, k, v, ints(cu))
    with pytest.raises(Yue2Error, match="out of range"):
        ops.check_status()
    ops.check_status()


def test_packed_offsets_that_go_back_and_forth_do_nothing(ops):
    # each second sequence is valid by itself, together they are more rows than there are
    q, k = randn((300, 2, 64), torch.bfloat16, 1), randn((300, 1, 64), torch.bfloat16, 2)
    out = torch.full_like(q, 7.0)
    ops.attention_packed(q, k, k, ints([0, 300] * 8), out=out)
    with pytest.raises(Yue2Error, match="out of range"):
        ops.check_status()
    assert bool((out == 7.0).all())


# ------------------------------------------------------------------ drafted tokens over pages
def make_pages(rng, need, extra=3):
    """Shuffled page tables for sequences of need[s] positions; unused entries point far away."""
    counts = [-(-n // 64) for n in need]
    total = sum(counts) + extra
    order = list(range(total))
    rng.shuffle(order)
    table = np.full((len(need), max(1, max(counts)) + 1), -1, dtype=np.int32)
    at = 0
    for s, c in enumerate(counts):
        table[s, :c] = order[at:at + c]
        at += c
    return total, table


def tree_masks(rng, nodes):
    out = []
    for n in nodes:
        bits = []
        for j in range(n):
            parent = rng.randint(max(-1, j - 5), j - 1)
            bits.append((bits[parent] if parent >= 0 else 0) | (1 << j))
        out += bits
    return np.array(out, dtype=np.uint64)


def tree_reference(q, data, layer, table, ctx, nodes, mask, scale, first=0):
    heads, kv = q.shape[1], data.shape[3]
    want = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(want)
    at = first
    for s, (c, t) in enumerate(zip(ctx, nodes)):
        n = c + t
        pos = torch.arange(n, device=q.device)
        page = torch.tensor(table[s], device=q.device).long()[pos // 64]
        see = torch.ones((t, n), dtype=torch.bool, device=q.device)
        for i in range(t):
            for j in range(t):
                see[i, c + j] = j <= i if mask is None else bool(int(mask[at + i]) >> j & 1)
        for h in range(heads if t else 0):
            g = h // (heads // kv)
            want[at:at + t, h], tol[at:at + t, h] = attend(q[at:at + t, h], data[page, layer, 0, g, pos % 64],
                                                          data[page, layer, 1, g, pos % 64], see, scale)
        at += t
    return want, tol


def check_tree(ops, ctx, nodes, heads, kv, dim, dtype, masks="tree", layers=2, layer=1, seed=1, first=0, behind=0, empty=False):
    rng = random.Random(seed)
    pages, table = make_pages(rng, [c + t for c, t in zip(ctx, nodes)])
    data = randn((pages, layers, 2, kv, 64, dim), dtype, seed)
    # what lies behind each sequence's last position, and in the pages of nobody, is NaN
    used = torch.zeros((pages, 64), dtype=torch.bool)
    for s, (c, t) in enumerate(zip(ctx, nodes)):
        for p in range(c + t):
            used[table[s, p // 64], p % 64] = True
    data.permute(0, 4, 1, 2, 3, 5)[~used.to(DEV)] = float("nan")
    rows = first + sum(nodes) + behind
    q = randn((rows, heads, dim), dtype, seed + 1)
    mask = tree_masks(rng, nodes) if masks == "tree" else None
    if mask is not None:
        if empty and len(mask) > 1:
            mask[1::3] = 0
        mask = np.concatenate([np.zeros(first, np.uint64), mask, np.zeros(behind, np.uint64)])
    out = torch.full((rows, heads, dim), 7.0, dtype=dtype, device=DEV)
    dmask = None
    if mask is not None:
        beyond = mask.copy()  # bits past the sequence's nodes mean nothing
        at = first
        for t in nodes:
            if t < 64:
                beyond[at:at + t] |= np.uint64(((1 << 64) - 1) ^ ((1 << t) - 1))
            at += t
        dmask = ints(beyond.view(np.int64), torch.int64)
    ops.attention_tree(q, ops.KvPool(data), layer, ints(table), ints(ctx), offsets(nodes, first), mask=dmask, out=out)
    ops.check_status()
    want, tol = tree_reference(q, data, layer, table, ctx, nodes, mask, 1 / math.sqrt(dim), first)
    a, b = first, first + sum(nodes)
    close(out[a:b], want[a:b], tol[a:b])
    assert (out[:a] == 7).all() and (out[b:] == 7).all()


@pytest.mark.parametrize("masks", ["tree", None])
@pytest.mark.parametrize("ctx", [0, 1, 31, 63, 64, 65, 127, 128, 129, 300, 1000])
@pytest.mark.parametrize("nodes", [1, 2, 17, 64])
def test_tree_lengths(ops, ctx, nodes, masks):
    check_tree(ops, [ctx], [nodes], 6, 2, 128, torch.bfloat16, masks)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads,kv,dim", [(24, 8, 128), (8, 2, 128), (4, 2, 64), (2, 2, 64), (8, 1, 128), (16, 1, 64), (5, 1, 64),
                                          (96, 1, 128), (128, 1, 64)])
def test_tree_layouts(ops, heads, kv, dim, dtype):
    check_tree(ops, [130, 0, 700, 64, 5], [9, 3, 1, 0, 33], heads, kv, dim, dtype, first=2, behind=3)
    check_tree(ops, [77, 2000], [64, 1], heads, kv, dim, dtype, None, layers=1, layer=0)


def test_tree_rows_that_see_nothing_are_zero(ops):
    check_tree(ops, [0, 0, 70], [16, 1, 16], 4, 2, 64, torch.bfloat16, empty=True)
    check_tree(ops, [0, 0, 70], [40, 2, 64], 8, 2, 128, torch.float16, empty=True)


@pytest.mark.parametrize("ctx,nodes", [([4096, 3, 1030], [8, 1, 20]), ([5000], [1]), ([3000] * 9, [4] * 9), ([8191, 0], [64, 64])])
def test_tree_split_contexts(ops, ctx, nodes):
    check_tree(ops, ctx, nodes, 6, 2, 128, torch.bfloat16)
    check_tree(ops, ctx, nodes, 4, 1, 64, torch.float16, None)


def test_tree_many_sequences(ops):
    rng = random.Random(2)
    check_tree(ops, [rng.choice([0, 3, 64, 200]) for _ in range(150)], [rng.choice([0, 1, 1, 5]) for _ in range(150)], 4, 2, 64, torch.bfloat16, None)


def test_tree_chain_equals_its_mask_bit_for_bit(ops):
    rng = random.Random(1)
    nodes, ctx = [40, 3], [777, 64]
    pages, table = make_pages(rng, [c + t for c, t in zip(ctx, nodes)])
    pool = ops.KvPool(randn((pages, 1, 2, 2, 64, 128), torch.bfloat16, 4))
    q = randn((43, 4, 128), torch.bfloat16, 5)
    chain = ints([(2 << i) - 1 for t in nodes for i in range(t)], torch.int64)
    args = (q, pool, 0, ints(table), ints(ctx), offsets(nodes))
    a, b, c = ops.attention_tree(*args), ops.attention_tree(*args, mask=chain), ops.attention_tree(*args)
    assert torch.equal(a, b) and torch.equal(a, c)


@pytest.mark.parametrize("value", [float("inf"), float("-inf"), float("nan")])
def test_tree_nonfinite_drafts_stay_with_the_rows_that_see_them(ops, value):
    rng = random.Random(1)
    ctx, nodes = 100, 20
    pages, table = make_pages(rng, [ctx + nodes])
    data = randn((pages, 1, 2, 2, 64, 128), torch.bfloat16, 4)
    q = randn((nodes, 6, 128), torch.bfloat16, 5)
    mask = tree_masks(rng, [nodes])
    args = (q, ops.KvPool(data), 0, ints(table), ints([ctx]), offsets([nodes]), ints(mask.view(np.int64), torch.int64))
    clean = ops.attention_tree(*args)
    j = 7
    data[table[0, (ctx + j) // 64], 0, 1, 1, (ctx + j) % 64, 9] = value
    got = ops.attention_tree(*args)
    ops.check_status()
    sees = torch.zeros((nodes, 6, 128), dtype=torch.bool, device=DEV)
    for i in range(nodes):
        if int(mask[i]) >> j & 1:
            sees[i, 3:, 9] = True
    assert torch.equal(got[~sees], clean[~sees])
    hit = got[sees]
    assert torch.isnan(hit).all() if math.isnan(value) else (hit == value).all()


@pytest.mark.parametrize("value", [float("inf"), float("nan")])
@pytest.mark.parametrize("at", [0, 7, 14, 15, 127, 128, 299, 300, 305])
def test_tree_nonfinite_scores_make_their_rows_nan(ops, at, value):
    ctx, nodes = 300, 12
    rng = random.Random(2)
    pages, table = make_pages(rng, [ctx + nodes])
    data = randn((pages, 1, 2, 1, 64, 64), torch.bfloat16, 4)
    q = randn((nodes, 3, 64), torch.bfloat16, 5)
    mask = tree_masks(rng, [nodes])
    args = (q, ops.KvPool(data), 0, ints(table), ints([ctx]), offsets([nodes]), ints(mask.view(np.int64), torch.int64))
    clean = ops.attention_tree(*args)
    data[table[0, at // 64], 0, 0, 0, at % 64] = value
    got = ops.attention_tree(*args)
    for i in range(nodes):
        if at < ctx or int(mask[i]) >> (at - ctx) & 1:
            assert torch.isnan(got[i]).all()
        else:
            assert torch.equal(got[i], clean[i])


def test_tree_huge_values_in_masked_places(ops):
    rng = random.Random(2)
    ctx, nodes = 60, 40
    pages, table = make_pages(rng, [ctx + nodes])
    data = randn((pages, 1, 2, 1, 64, 128), torch.bfloat16, 4)
    q = randn((nodes, 4, 128), torch.bfloat16, 5)
    args = (q, ops.KvPool(data), 0, ints(table), ints([ctx]), offsets([nodes]))
    clean = ops.attention_tree(*args)
    for p in range(ctx + 20, ctx + nodes):
        data[table[0, p // 64], 0, :, 0, p % 64] = 3.0e38
    got = ops.attention_tree(*args)
    assert torch.equal(got[:20], clean[:20])


def test_tree_at_the_limits(ops):
    rng = random.Random(9)
    n = 1024
    check_tree(ops, [rng.choice([0, 1, 63, 64, 70]) for _ in range(n)], [rng.choice([0, 1, 1, 2]) for _ in range(n)], 2, 1, 64, torch.bfloat16, None,
               layers=1, layer=0)
    check_tree(ops, [0] * 20, [64] * 20, 8, 1, 64, torch.float16, layers=1, layer=0)
    pool = ops.KvPool(randn((2, 1, 2, 1, 64, 64), torch.bfloat16, 1))
    q = randn((1025, 1, 64), torch.bfloat16, 2)
    with pytest.raises(Yue2Error, match="1,024"):
        ops.attention_tree(q, pool, 0, ints([[0]] * 1025), ints([0] * 1025), offsets([1] * 1025))
    wide = ops.KvPool(randn((2, 1, 2, 1, 64, 64), torch.bfloat16, 1))
    with pytest.raises(Yue2Error, match="128 query heads"):
        ops.attention_tree(randn((1, 129, 64), torch.bfloat16, 2), wide, 0, ints([[0]]), ints([0]), offsets([1]))


def test_tree_shared_pages_and_strided_rows(ops):
    # two takes of one prompt: full pages shared, their own tails
    data = randn((6, 1, 2, 2, 64, 64), torch.float16, 1)
    table = np.array([[0, 1, 2], [0, 1, 3]], dtype=np.int32)
    wide = randn((7, 10, 64), torch.float16, 2)
    q = wide[:, 2:6]
    got = torch.full((7, 8, 64), 3.0, dtype=torch.float16, device=DEV)
    ops.attention_tree(q, ops.KvPool(data), 0, ints(table), ints([150, 140]), offsets([4, 3]), out=got[:, 4:])
    ops.check_status()
    want, tol = tree_reference(q, data, 0, table, [150, 140], [4, 3], None, 1 / 8)
    close(got[:, 4:], want, tol)
    assert (got[:, :4] == 3).all()


def test_tree_offsets_past_32_bits(ops):
    # a pool of 3.3e9 values: the last pages lie past 2^32 bytes and past 2^31 values
    pages, layers = 900, 28
    data = torch.zeros((pages, layers, 2, 8, 64, 128), dtype=torch.bfloat16, device=DEV)
    assert data.numel() > 1 << 31
    table = np.array([[899, 5, 898, 897]], dtype=np.int32)
    for i, p in enumerate(table[0]):
        data[p, 27] = randn((2, 8, 64, 128), torch.bfloat16, 10 + i)
    q = randn((5, 24, 128), torch.bfloat16, 3)
    pool = ops.KvPool(data)
    got = ops.attention_tree(q, pool, 27, ints(table), ints([250]), offsets([5]))
    want, tol = tree_reference(q, data, 27, table, [250], [5], None, 1 / math.sqrt(128))
    close(got, want, tol)
    ops.kv_copy(pool, ints([899]), ints([890]), ints([33]))
    assert torch.equal(data[890, 27, :, :, :33], data[899, 27, :, :, :33]) and (data[890, 27, :, :, 33:] == 0).all()
    before = data[897, 27, :, :, 7].clone()
    ops.kv_gather(pool, ints(table), None, ints([64]), offsets([1]), ints([199]))
    assert torch.equal(data[5, 27, :, :, 0], before)
    ops.check_status()


@pytest.mark.parametrize("case,message", [("page", "page index"), ("negative page", "page index"), ("context", "out of range"),
                                          ("negative context", "out of range"), ("nodes", "out of range"), ("offsets", "out of range")])
def test_tree_bad_entries_are_reported(ops, case, message):
    data = randn((6, 1, 2, 2, 64, 64), torch.bfloat16, 1)
    table, ctx, cu = [[0, 1], [2, 3]], [100, 60], [0, 2, 5]
    rows = 100
    if case == "page":
        table[1][0] = 6
    elif case == "negative page":
        table[1][1] = -7
        ctx[1] = 64
    elif case == "context":
        ctx[1] = 126
    elif case == "negative context":
        ctx[1] = -1
    elif case == "nodes":
        cu[2] = 2 + 65
        ctx[1] = 0
    else:
        cu[2] = 101
    q = randn((rows, 4, 64), torch.bfloat16, 2)
    got = ops.attention_tree(q, ops.KvPool(data), 0, ints(table), ints(ctx), ints(cu))
    with pytest.raises(Yue2Error, match=message):
        ops.check_status()
    ops.check_status()
    want, tol = tree_reference(q, data, 0, np.array(table), [ctx[0]], [2], None, 1 / 8)
    close(got[:2], want[:2], tol[:2])  # the sound sequence of the same call


def test_tree_captured_while_the_context_grows(ops):
    rng = random.Random(1)
    pages, table = make_pages(rng, [400, 400])
    data = randn((pages, 1, 2, 2, 64, 128), torch.bfloat16, 4)
    pool, q = ops.KvPool(data), randn((2, 6, 128), torch.bfloat16, 5)
    ctx, cu, tab = ints([0, 0]), offsets([1, 1]), ints(table)
    ops.attention_tree(q, pool, 0, tab, ctx, cu)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for _ in range(2):  # two graphs replayed one after the other
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(ops.attention_tree(q, pool, 0, tab, ctx, cu))
        graphs.append(g)
    for c in ([0, 5], [64, 63], [399, 128], [200, 0]):
        ctx.copy_(ints(c))
        for g in graphs:
            g.replay()
        want, tol = tree_reference(q, data, 0, table, c, [1, 1], None, 1 / math.sqrt(128))
        for o in outs:
            close(o, want, tol)
    ops.check_status()


def test_two_calls_at_once_on_two_streams(ops):
    rng = random.Random(1)
    ctx, nodes = [6000, 3000], [16, 3]
    pages, table = make_pages(rng, [c + t for c, t in zip(ctx, nodes)])
    pool = ops.KvPool(randn((pages, 1, 2, 2, 64, 128), torch.bfloat16, 4))
    q = randn((19, 8, 128), torch.bfloat16, 5)
    args = (q, pool, 0, ints(table), ints(ctx), offsets(nodes))
    want = ops.attention_tree(*args)
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(3)], []
    for _ in range(4):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(ops.attention_tree(*args))
    torch.cuda.synchronize()
    assert all(torch.equal(want, g) for g in got)


# ------------------------------------------------------------------ norm, rotation, append
def tables(rows, dim):
    angle = np.arange(rows)[:, None] * 10000.0 ** (-np.arange(dim // 2) / (dim // 2))[None]
    return torch.tensor(np.cos(angle), dtype=torch.float32).to(DEV), torch.tensor(np.sin(angle), dtype=torch.float32).to(DEV)


def append_reference(x, gain, cos, sin, pos, eps):
    x = x.double()
    half = x.shape[-1] // 2
    if gain is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * gain.double()
    c, s = cos.double()[pos.long()][:, None], sin.double()[pos.long()][:, None]
    a, b = x[..., :half], x[..., half:]
    size = (a.abs() + b.abs()).repeat(1, 1, 2)
    return torch.cat([a * c - b * s, b * c + a * s], -1), size


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,heads,kv,dim", [(1, 4, 2, 64), (2, 24, 8, 128), (77, 8, 2, 128), (130, 3, 1, 64), (40, 4, 4, 256), (9, 1, 1, 256)])
@pytest.mark.parametrize("norm", [True, False])
def test_append(ops, rows, heads, kv, dim, dtype, norm):
    rng = random.Random(rows)
    qkv = randn((rows, heads + 2 * kv, dim), dtype, 1) * 3
    data = randn((4, 3, 2, kv, 64, dim), dtype, 2)
    before = data.clone()
    gains = (1 + 0.2 * randn((dim,), torch.float32, 3), 1 + 0.2 * randn((dim,), torch.float32, 4)) if norm else (None, None)
    cos, sin = tables(500, dim)
    pos = ints([rng.randrange(500) for _ in range(rows)])
    slots = rng.sample(range(256), rows)
    slots = [-1 if i % 5 == 3 else s for i, s in enumerate(slots)]
    k_out = torch.zeros((rows, kv, dim), dtype=dtype, device=DEV)
    q = ops.qk_rope_append(qkv, *gains, 1e-6, cos, sin, pos, ops.KvPool(data), 1, ints(slots, torch.int64), k_out=k_out)
    ops.check_status()
    u = U[dtype]
    for got, part, gain in ((q, qkv[:, :heads], gains[0]), (k_out, qkv[:, heads:heads + kv], gains[1])):
        want, size = append_reference(part, gain, cos, sin, pos, 1e-6)
        close(got, want, u * want.abs() + 2.0 ** -18 * size + (2.0 ** -25 if dtype == torch.float16 else 0))
    for i, s in enumerate(slots):
        if s >= 0:
            assert torch.equal(data[s // 64, 1, 0, :, s % 64], k_out[i])
            assert torch.equal(data[s // 64, 1, 1, :, s % 64], qkv[i, heads + kv:])
            before[s // 64, 1, :, :, s % 64] = data[s // 64, 1, :, :, s % 64]
    assert torch.equal(data, before)  # nothing else moved


def test_append_in_place_and_strided(ops):
    rows, heads, kv, dim = 33, 6, 2, 128
    wide = randn((rows, 14, dim), torch.bfloat16, 1)
    keep = wide.clone()
    qkv = wide[:, 3:13]
    data = torch.zeros((2, 1, 2, kv, 64, dim), dtype=torch.bfloat16, device=DEV)
    cos, sin = tables(64, dim)
    pos, slots = ints(list(range(rows))), ints(list(range(rows)), torch.int64)
    apart = ops.qk_rope_append(qkv.clone(), None, None, 0.0, cos, sin, pos, ops.KvPool(data.clone()), 0, slots)
    ops.qk_rope_append(qkv, None, None, 0.0, cos, sin, pos, ops.KvPool(data), 0, slots, q_out=qkv[:, :heads], k_out=qkv[:, heads:heads + kv])
    ops.check_status()
    assert torch.equal(qkv[:, :heads], apart)
    assert torch.equal(qkv[:, heads:heads + kv], data[0, 0, 0].permute(1, 0, 2)[:rows])
    assert torch.equal(wide[:, :3], keep[:, :3]) and torch.equal(wide[:, 11:], keep[:, 11:])


@pytest.mark.parametrize("pos,slot,message", [(64, 0, "out of range"), (-1, 0, "out of range"), (3, 128, "page index"), (3, 1 << 40, "page index")])
def test_append_bad_rows_are_reported(ops, pos, slot, message):
    data = torch.zeros((2, 1, 2, 1, 64, 64), dtype=torch.bfloat16, device=DEV)
    cos, sin = tables(64, 64)
    qkv = randn((3, 4, 64), torch.bfloat16, 1)
    ops.qk_rope_append(qkv, None, None, 0.0, cos, sin, ints([1, pos, 2]), ops.KvPool(data), 0, ints([5, slot, 6], torch.int64))
    with pytest.raises(Yue2Error, match=message):
        ops.check_status()
    assert (data[0, 0, 1, 0, 5] == qkv[0, 3]).all() and (data[0, 0, 1, 0, 6] == qkv[2, 3]).all()
    assert (data != 0).sum() <= 4 * 64  # the two sound rows


# ------------------------------------------------------------------ page moves
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("layers,kv,dim", [(1, 1, 64), (3, 2, 128), (2, 1, 256), (28, 8, 128)])
def test_copy(ops, layers, kv, dim, dtype):
    data = randn((20, layers, 2, kv, 64, dim), dtype, 1)
    want = data.clone()
    src, dst, count = [3, 7, 3, 0, 11], [19, 1, 2, 5, 6], [64, 0, 1, 63, 17]
    for a, b, n in zip(src, dst, count):
        want[b, :, :, :, :n] = data[a, :, :, :, :n]
    ops.kv_copy(ops.KvPool(data), ints(src), ints(dst), ints(count))
    assert torch.equal(data, want)
    want[dst] = data[src]
    ops.kv_copy(ops.KvPool(data), ints(src), ints(dst))
    assert torch.equal(data, want)
    ops.check_status()


@pytest.mark.parametrize("src,dst,count,message", [(-1, 2, 5, "page index"), (4, 2, 5, "page index"), (0, 4, 5, "page index"),
                                                   (0, -3, 5, "page index"), (0, 2, 65, "out of range"), (0, 2, -1, "out of range")])
def test_copy_bad_entries_are_reported(ops, src, dst, count, message):
    data = randn((4, 2, 2, 1, 64, 64), torch.bfloat16, 1)
    want = data.clone()
    want[3, :, :, :, :9] = data[1, :, :, :, :9]
    ops.kv_copy(ops.KvPool(data), ints([src, 1]), ints([dst, 3]), ints([count, 9]))
    with pytest.raises(Yue2Error, match=message):
        ops.check_status()
    assert torch.equal(data, want)


def gather_reference(data, src_table, dst_table, begin, kept):
    want = data.clone()
    for s, keep in enumerate(kept):
        for i, p in enumerate(keep):
            t = begin[s] + i
            want[dst_table[s][t // 64], :, :, :, t % 64] = data[src_table[s][p // 64], :, :, :, p % 64]
    return want


@pytest.mark.parametrize("layers,kv,dim", [(1, 1, 64), (3, 2, 128), (2, 1, 256)])
def test_gather_in_place(ops, layers, kv, dim):
    rng = random.Random(dim)
    begin = [100, 0, 5, 64, 130, 0]
    kept = [[100, 101, 105, 140], [3], [], sorted(rng.sample(range(64, 320), 200)), list(range(131, 320)), list(range(320))]
    pages, table = make_pages(rng, [320] * 6)
    data = randn((pages, layers, 2, kv, 64, dim), torch.bfloat16, 1)
    want = gather_reference(data, table, table, begin, kept)
    ops.kv_gather(ops.KvPool(data), ints(table), None, ints(begin), offsets([len(k) for k in kept]), ints([p for k in kept for p in k]))
    ops.check_status()
    assert torch.equal(data, want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_gather_into_other_pages(ops, dtype):
    rng = random.Random(4)
    lens, begin = [500, 64, 1000], [0, 63, 10]
    kept = [rng.sample(range(500), 300), [63, 0, 0, 7], sorted(rng.sample(range(1000), 999))]
    pages, table = make_pages(rng, lens + [b + len(k) for b, k in zip(begin, kept)])
    data = randn((pages, 2, 2, 2, 64, 128), dtype, 1)
    src, dst = table[:3], table[3:]
    want = gather_reference(data, src, dst, begin, kept)
    ops.kv_gather(ops.KvPool(data), ints(src), ints(dst[:, :17]), ints(begin), offsets([len(k) for k in kept]), ints([p for k in kept for p in k]))
    ops.check_status()
    assert torch.equal(data, want)


@pytest.mark.parametrize("begin,keep,message", [(0, [0, 5, 5], "out of range"), (0, [5, 4], "out of range"), (10, [9], "out of range"),
                                                (0, [128], "out of range"), (0, [-1], "out of range"), (-1, [3], "out of range"),
                                                (0, [70], "page index")])
def test_gather_bad_entries_are_reported(ops, begin, keep, message):
    data = randn((4, 1, 2, 1, 64, 64), torch.bfloat16, 1)
    before = data.clone()
    table = [[2, 9], [1, 0]]
    ops.kv_gather(ops.KvPool(data), ints(table), None, ints([begin, 0]), ints([0, len(keep), len(keep) + 1]), ints(keep + [64]))
    with pytest.raises(Yue2Error, match=message):
        ops.check_status()
    assert torch.equal(data[1, :, :, :, 0], before[0, :, :, :, 0]) and torch.equal(data[[0, 3]], before[[0, 3]])


# ------------------------------------------------------------------ together
@pytest.mark.parametrize("heads,kv,dim,dtype", [(6, 2, 128, torch.bfloat16), (4, 2, 64, torch.float16)])
def test_a_step_over_a_batch(ops, heads, kv, dim, dtype):
    """Two prompts prefilled together, the first forked for a second take, a tree drafted for each
    take and one of its paths accepted, and the next token decoded: every output against the
    definition over the rows that the pages should hold."""
    rng = random.Random(7)
    prompts, layer, eps = [150, 37], 1, 1e-6
    data = torch.full((16, 2, 2, kv, 64, dim), float("nan"), dtype=dtype, device=DEV)
    pool = ops.KvPool(data)
    cos, sin = tables(512, dim)
    gains = 1 + 0.1 * randn((dim,), torch.float32, 1), 1 + 0.1 * randn((dim,), torch.float32, 2)
    order = rng.sample(range(16), 16)
    table = np.array([order[0:5], order[5:10], order[10:15]], dtype=np.int32)  # prompt 0, prompt 1, the fork of prompt 0

    def slot(s, p):
        return int(table[s, p // 64]) * 64 + p % 64

    def step(rows, positions, slots, seed):
        qkv = randn((rows, heads + 2 * kv, dim), dtype, seed)
        k_out = torch.empty((rows, kv, dim), dtype=dtype, device=DEV)
        q = ops.qk_rope_append(qkv, *gains, eps, cos, sin, ints(positions), pool, layer, ints(slots, torch.int64), k_out=k_out)
        return q, k_out, qkv[:, heads + kv:]

    # prompts
    q, k, v = step(sum(prompts), [p for n in prompts for p in range(n)], [slot(s, p) for s, n in enumerate(prompts) for p in range(n)], 3)
    got = ops.attention_packed(q, k, v, offsets(prompts))
    want, tol = packed_reference(q, k, v, prompts, 0, True, 1 / math.sqrt(dim))
    close(got, want, tol)
    held = [(k[:150], v[:150]), (k[150:], v[150:]), (k[:150], v[:150])]  # what each sequence should hold
    # the fork shares the two full pages and copies the third
    own = int(table[2, 2])
    table[2, :2] = table[0, :2]
    ops.kv_copy(pool, ints([table[0, 2]]), ints([own]), ints([150 - 128]))
    # a drafted tree for each sequence; a node's rotary position is its depth
    ctx, nodes = [150, 37, 150], [12, 5, 9]
    mask = tree_masks(rng, nodes)
    depth = [bin(int(m)).count("1") - 1 for m in mask]
    at = np.concatenate([[0], np.cumsum(nodes)])
    q, k, v = step(sum(nodes), [ctx[s] + depth[at[s] + j] for s in range(3) for j in range(nodes[s])],
                   [slot(s, ctx[s] + j) for s in range(3) for j in range(nodes[s])], 4)
    got = ops.attention_tree(q, pool, layer, ints(table), ints(ctx), offsets(nodes), mask=ints(mask.view(np.int64), torch.int64))
    path, keep = [], []
    for s in range(3):
        a, b = at[s], at[s + 1]
        kk, vv = torch.cat([held[s][0], k[a:b]]), torch.cat([held[s][1], v[a:b]])
        see = torch.ones((nodes[s], ctx[s] + nodes[s]), dtype=torch.bool, device=DEV)
        for i in range(nodes[s]):
            for j in range(nodes[s]):
                see[i, ctx[s] + j] = bool(int(mask[a + i]) >> j & 1)
        for h in range(heads):
            g = h // (heads // kv)
            want, tol = attend(q[a:b, h], kk[:, g], vv[:, g], see, 1 / math.sqrt(dim))
            close(got[a:b, h], want, tol, (s, h))
        leaf = int(max(range(nodes[s]), key=lambda j: depth[a + j]))
        path.append([j for j in range(nodes[s]) if int(mask[a + leaf]) >> j & 1])
        keep += [ctx[s] + j for j in path[s]]
        held[s] = torch.cat([held[s][0], k[a:b][path[s]]]), torch.cat([held[s][1], v[a:b][path[s]]])
    # the accepted paths, then one more token of each
    ops.kv_gather(pool, ints(table), None, ints(ctx), offsets([len(p) for p in path]), ints(keep))
    ctx = [c + len(p) for c, p in zip(ctx, path)]
    q, k, v = step(3, ctx, [slot(s, ctx[s]) for s in range(3)], 5)
    got = ops.attention_tree(q, pool, layer, ints(table), ints(ctx), offsets([1, 1, 1]))
    ops.check_status()
    for s in range(3):
        kk, vv = torch.cat([held[s][0], k[s:s + 1]]), torch.cat([held[s][1], v[s:s + 1]])
        see = torch.ones((1, ctx[s] + 1), dtype=torch.bool, device=DEV)
        for h in range(heads):
            g = h // (heads // kv)
            want, tol = attend(q[s:s + 1, h], kk[:, g], vv[:, g], see, 1 / math.sqrt(dim))
            close(got[s:s + 1, h], want, tol, (s, h))


def test_first_call_inside_a_capture_is_refused(ops, monkeypatch):
    # the status word would belong to the graph
    data = randn((2, 1, 2, 1, 64, 64), torch.bfloat16, 1)
    pool = ops.KvPool(data)
    src, dst = ints([0]), ints([1])
    monkeypatch.setattr(ops, "_status", {})
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(Yue2Error, match="before any capture"):
        ops.kv_copy(pool, src, dst)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    ops.kv_copy(pool, src, dst)
    ops.check_status()
    assert torch.equal(data[0], data[1])


def test_python_refusals(ops):
    q, k = randn((10, 4, 64), torch.bfloat16, 1), randn((10, 2, 64), torch.bfloat16, 2)
    cu = offsets([10])
    pool = ops.KvPool(randn((2, 1, 2, 2, 64, 64), torch.bfloat16, 3))
    bad = [lambda: ops.attention_packed(q.float(), k, k, cu), lambda: ops.attention_packed(q, k.half(), k, cu),
           lambda: ops.attention_packed(q, k, k[:9], cu), lambda: ops.attention_packed(q, k, k, cu.long()),
           lambda: ops.attention_packed(q.transpose(0, 1), k, k, cu), lambda: ops.attention_packed(q, k.cpu(), k, cu),
           lambda: ops.attention_packed(q[:, :, ::2], k, k, cu), lambda: ops.attention_packed(q[:, :3], k, k, cu),
           lambda: ops.attention_packed(q, k, k, cu, out=q[:5]), lambda: ops.KvPool(pool.data[:, :, :1]),
           lambda: ops.KvPool(pool.data.float()), lambda: ops.KvPool(pool.data.transpose(0, 3)), lambda: ops.KvPool(pool.data.cpu()),
           lambda: ops.attention_tree(q, pool, 1, ints([[0, 1]]), ints([3]), cu), lambda: ops.attention_tree(q, pool, 0, ints([0, 1]), ints([3]), cu),
           lambda: ops.attention_tree(q, pool, 0, ints([[0, 1]]), ints([3, 4]), cu), lambda: ops.attention_tree(q, pool, 0, ints([[0, 1]]), ints([3]), cu, mask=cu),
           lambda: ops.attention_tree(q.half(), pool, 0, ints([[0, 1]]), ints([3]), cu), lambda: ops.kv_copy(pool, ints([0]), ints([1, 0])),
           lambda: ops.kv_copy(pool, ints([0]), ints([1], torch.int64)), lambda: ops.kv_gather(pool, ints([[0]]), ints([[1], [0]]), ints([0]), cu, cu),
           lambda: ops.kv_gather(pool, ints([[0]]), None, ints([0, 0]), cu, cu)]
    for i, f in enumerate(bad):
        with pytest.raises(Yue2Error):
            f()
            pytest.fail(f"call {i} was taken")
    ops.check_status()


def test_rows_that_ask_for_a_gradient_are_refused(ops):
    q, k = randn((10, 4, 64), torch.bfloat16, 1), randn((10, 2, 64), torch.bfloat16, 2)
    cu, pos, slots = offsets([10]), ints(range(10)), ints(range(10), torch.int64)
    pool = ops.KvPool(randn((2, 1, 2, 2, 64, 64), torch.bfloat16, 3))
    cos = torch.ones(16, 32, device="cuda")
    gain = torch.ones(64, device="cuda")
    qkv = torch.cat([q, k, k], 1)

    def ask(t):
        return t.clone().requires_grad_()

    calls = [lambda: ops.attention_packed(ask(q), k, k, cu), lambda: ops.attention_packed(q, ask(k), k, cu),
             lambda: ops.attention_packed(q, k, ask(k), cu), lambda: ops.attention_tree(ask(q), pool, 0, ints([[0, 1]]), ints([0]), cu),
             lambda: ops.qk_rope_append(ask(qkv), None, None, 1e-6, cos, cos, pos, pool, 0, slots),
             lambda: ops.qk_rope_append(qkv, ask(gain), gain, 1e-6, cos, cos, pos, pool, 0, slots),
             lambda: ops.qk_rope_append(qkv, gain, ask(gain), 1e-6, cos, cos, pos, pool, 0, slots)]
    for f in calls:
        with pytest.raises(Yue2Error, match="gradient"):
            f()
        with torch.no_grad():
            f()
    ops.check_status()
