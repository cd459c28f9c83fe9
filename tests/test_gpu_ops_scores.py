"""Attention scores of -inf and close to the ends of f32, against plain 64-bit forms.

A key whose score is -inf has no weight, and a row without any weight is zero (as a row that sees
nothing). The tolerances are those of test_gpu_ops.attend over the keys that keep a weight: the
places that make a score infinite are taken out of the reference's keys before its products."""
import math
import random

import numpy as np
import pytest
import torch

from test_gpu_ops import check_packed as packed_as_before
from test_gpu_ops import DEV, attend, close, ints, make_pages, offsets, ops, randn  # noqa: F401 (ops is a fixture)

pytestmark = pytest.mark.gpu

C = 3  # the component that makes scores infinite; the queries' is positive there
LOWEST = torch.finfo(torch.bfloat16).min


def rows_of(n, heads, dim, dtype, seed):
    q = randn((n, heads, dim), dtype, seed)
    q[:, :, C] = q[:, :, C].abs() + 0.5
    return q


def reference(q, k, v, gone, see, scale):
    """Output and tolerance of rows q [n, heads, dim] over k and v [m, kv, dim]; the keys `gone` [m, kv]
    have no weight."""
    heads, kv = q.shape[1], k.shape[1]
    want = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(want)
    for h in range(heads):
        g = h // (heads // kv)
        lives = ~gone[:, g]
        kk = torch.where(lives[:, None], k[:, g], torch.zeros_like(k[:, g]))
        vv = torch.where(lives[:, None], v[:, g], torch.zeros_like(v[:, g]))
        want[:, h], tol[:, h] = attend(q[:, h], kk, vv, see & lives[None], scale)
    return want, tol


def sees(n, causal):
    i = torch.arange(n, device=DEV)
    return i[None] <= i[:, None] if causal else torch.ones((n, n), dtype=torch.bool, device=DEV)


def check_packed(ops, lens, dropped, causal, dtype, dim, rows=slice(None), heads=4, kv=2, low=0.0, huge=None):
    """`dropped`: keys of every sequence whose scores are -inf; `low` shifts all other scores."""
    n = sum(lens)
    q, k, v = rows_of(n, heads, dim, dtype, 1), randn((n, kv, dim), dtype, 2), randn((n, kv, dim), dtype, 3)
    if low:
        q[:, :, 5], k[:, :, 5] = 8, low
    gone = torch.zeros((n, kv), dtype=torch.bool, device=DEV)
    at = 0
    for m in lens:
        keys = [at + j for j in dropped if j < m]
        gone[keys] = True
        at += m
    k[..., C] = torch.where(gone, -math.inf, k[..., C])
    if huge is not None:
        v[gone] = huge
    got = ops.attention_packed(q, k, v, offsets(lens), causal=causal)
    ops.check_status()
    at = 0
    for m in lens:
        part = slice(at, at + m)
        want, tol = reference(q[part], k[part], v[part], gone[part], sees(m, causal), 1 / math.sqrt(dim))
        close(got[part][rows], want[rows], tol[rows], (m, causal))
        at += m


@pytest.mark.parametrize("low", [0.0, -200.0])  # -200: scores far below what 2^x holds relative to zero
@pytest.mark.parametrize("dim,dtype", [(64, torch.float16), (128, torch.bfloat16)])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("tiles", [1, 2])
def test_packed_first_tiles_without_a_weight(ops, tiles, causal, dim, dtype, low):
    # the rows behind them see ordinary scores in several tiles, first below and then above any
    # score so far
    check_packed(ops, [317 + 128 * tiles, 900, 640], range(128 * tiles), causal, dtype, dim, slice(128 * tiles, None), low=low)


def check_tree(ops, ctx, nodes, dropped, dtype, dim, heads=6, kv=2, mask=None, huge=None, scale=None, value=-math.inf):
    """One call over sequences of ctx[s] positions and nodes[s] drafted ones; dropped(s, n): its keys
    whose scores are -inf."""
    rng = random.Random(7)
    held = [c + t for c, t in zip(ctx, nodes)]
    pages, table = make_pages(rng, held)
    data = randn((pages, 1, 2, kv, 64, dim), dtype, 4)
    q = rows_of(sum(nodes), heads, dim, dtype, 5)
    expect, at = [], 0
    for s, (c, t) in enumerate(zip(ctx, nodes)):
        pos = torch.arange(c + t, device=DEV)
        page = ints(table[s]).long()[pos // 64]
        gone = torch.zeros(c + t, dtype=torch.bool, device=DEV)
        gone[list(dropped(s, c + t))] = True
        data[page[gone], 0, 0, :, pos[gone] % 64, C] = value
        if huge is not None:
            data[page[gone], 0, 1, :, pos[gone] % 64] = huge
        k, v = data[page, 0, 0, :, pos % 64], data[page, 0, 1, :, pos % 64]
        see = pos[None] <= c + torch.arange(t, device=DEV)[:, None]
        expect.append((slice(at, at + t), q[at:at + t], k, v, gone[:, None].expand(-1, kv), see))
        at += t
    got = ops.attention_tree(q, ops.KvPool(data), 0, ints(table), ints(ctx), offsets(nodes), scale=scale)
    ops.check_status()
    for rows, qq, k, v, gone, see in expect:
        want, tol = reference(qq, k, v, gone, see, 1 / math.sqrt(dim) if scale is None else scale)
        close(got[rows], want, tol, rows)


@pytest.mark.parametrize("dim,dtype", [(64, torch.float16), (128, torch.bfloat16)])
@pytest.mark.parametrize("ctx,nodes", [([700], [3]), ([5000, 300], [1, 9]), ([700], [64])])
def test_tree_first_tiles_without_a_weight(ops, ctx, nodes, dim, dtype):
    check_tree(ops, ctx, nodes, lambda s, n: range(256), dtype, dim)


@pytest.mark.parametrize("dtype,huge,dim", [(torch.bfloat16, 3.0e38, 128), (torch.float16, 65504.0, 64)])
@pytest.mark.parametrize("causal", [True, False])
def test_packed_single_keys_without_a_weight_add_nothing(ops, causal, dtype, huge, dim):
    # at places of either way of exponentials, their values as large as the type holds them
    check_packed(ops, [600, 1, 512], [0, 14, 15, 31, 62, 130, 142, 143, 158, 159, 254, 300, 399, 511], causal, dtype, dim, huge=huge)


@pytest.mark.parametrize("dtype,huge,dim", [(torch.bfloat16, 3.0e38, 128), (torch.float16, 65504.0, 64)])
@pytest.mark.parametrize("nodes", [1, 20, 64])
def test_tree_single_keys_without_a_weight_add_nothing(ops, nodes, dtype, huge, dim):
    places = [0, 14, 15, 31, 62, 130, 142, 143, 158, 159, 254, 300, 399, 511]
    check_tree(ops, [600, 2000], [nodes, 3], lambda s, n: places, dtype, dim, huge=huge)


@pytest.mark.parametrize("dtype,dim", [(torch.bfloat16, 128), (torch.float16, 64)])
@pytest.mark.parametrize("causal", [True, False])
def test_packed_rows_without_any_weight_are_zero(ops, causal, dtype, dim):
    check_packed(ops, [1, 100, 128, 300, 512], range(512), causal, dtype, dim)
    if causal:  # and rows with a weight in the same tiles
        check_packed(ops, [200, 517], range(150), causal, dtype, dim)


@pytest.mark.parametrize("dtype,dim", [(torch.bfloat16, 128), (torch.float16, 64)])
def test_tree_rows_without_any_weight_are_zero(ops, dtype, dim):
    # items of one share and items that are cut, rows of one side and of two; then other sequences
    # of the same call with ordinary scores
    check_tree(ops, [0, 5, 128, 700], [1, 64, 9, 64], lambda s, n: range(n), dtype, dim)
    check_tree(ops, [9000], [2], lambda s, n: range(n), dtype, dim)
    check_tree(ops, [9000, 3000, 40], [40, 2, 1], lambda s, n: range(n) if s < 2 else [], dtype, dim)
    # cut items whose first shares have no weight
    check_tree(ops, [9000], [2], lambda s, n: range(4000), dtype, dim)


def test_packed_unmasked_values_that_are_not_finite(ops):
    # every row sees every value of its sequence, whole tiles and the ragged last one alike
    for n, at in ((400, 399), (513, 512), (700, 645), (700, 40), (1100, 1030)):
        q, k, v = randn((n + 90, 4, 128), torch.bfloat16, 1), randn((n + 90, 2, 128), torch.bfloat16, 2), randn((n + 90, 2, 128), torch.bfloat16, 3)
        clean = ops.attention_packed(q, k, v, offsets([n, 90]), causal=False)
        v[at, 1, 5] = math.inf
        v[n:, :, 7] = math.nan  # the sequence behind
        got = ops.attention_packed(q, k, v, offsets([n, 90]), causal=False)
        ops.check_status()
        hit = torch.zeros_like(got, dtype=torch.bool)
        hit[:n, 2:, 5] = True
        hit[n:, :, 7] = True
        assert torch.equal(got[~hit], clean[~hit])
        assert (got[:n, 2:, 5] == math.inf).all() and torch.isnan(got[n:, :, 7]).all()


def test_packed_one_value_that_is_not_finite_costs_little(ops):
    # a pass over the whole sequence for every row would make the call tens of times as long
    n = 4001
    q, k, v = randn((n, 8, 128), torch.bfloat16, 1), randn((n, 8, 128), torch.bfloat16, 2), randn((n, 8, 128), torch.bfloat16, 3)
    cu, out = offsets([n]), torch.empty_like(q)

    def best():
        times = []
        for _ in range(6):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            ops.attention_packed(q, k, v, cu, causal=False, out=out)
            b.record()
            torch.cuda.synchronize()
            times.append(a.elapsed_time(b))
        return min(times)

    ordinary = best()
    v[n - 1] = math.nan
    assert best() < 3 * ordinary


@pytest.mark.parametrize("scale", [None, 1.0, 5.0, -1.0])
@pytest.mark.parametrize("causal", [True, False])
def test_packed_keys_at_the_lowest_value(ops, causal, scale):
    # scores near the end of f32, whose product with the scale passes it; rows that see nothing
    # else weigh those keys alike (their scores are one and the same number in 64 bits too)
    lens, dim, sign = [150, 700], 128, -1.0 if scale is not None and scale < 0 else 1.0
    n = sum(lens)
    q, k, v = randn((n, 4, dim), torch.bfloat16, 1), randn((n, 2, dim), torch.bfloat16, 2), randn((n, 2, dim), torch.bfloat16, 3)
    q[:, :, C] = 1
    gone = torch.zeros((n, 2), dtype=torch.bool, device=DEV)
    gone[:140] = True
    gone[150:150 + 300] = True
    k[..., C] = torch.where(gone, sign * LOWEST, k[..., C])
    got = ops.attention_packed(q, k, v, offsets(lens), causal=causal, scale=scale)
    ops.check_status()
    at = 0
    for m in lens:
        part, see = slice(at, at + m), sees(m, causal)
        want, tol = reference(q[part], k[part], v[part], gone[part], see, 1 / math.sqrt(dim) if scale is None else scale)
        alike, alike_tol = reference(torch.zeros_like(q[part]), torch.zeros_like(k[part]), v[part], torch.zeros_like(gone[part]), see, 1.0)
        only = ~(see & ~gone[part, 0][None]).any(1)
        want[only], tol[only] = alike[only], alike_tol[only]
        close(got[part], want, tol, m)
        at += m


@pytest.mark.parametrize("value", [2 * LOWEST / 3, -1.0e12])
@pytest.mark.parametrize("scale", [None, 1.0, 4.0])
@pytest.mark.parametrize("nodes", [1, 30, 64])
def test_tree_keys_at_the_lowest_value(ops, nodes, scale, value):
    check_tree(ops, [700, 6000], [nodes, 2], lambda s, n: range(300), torch.bfloat16, 128, scale=scale, value=value)


@pytest.mark.parametrize("ctx,dropped", [(9000, 4000), (700, 300), (24000, 20000)])
def test_tree_keys_without_a_share_add_nothing(ops, ctx, dropped):
    # scores so low that their weights are 0 beside the others', values of 2^110: in items that are cut,
    # whole shares of them
    check_tree(ops, [ctx], [2], lambda s, n: range(dropped), torch.bfloat16, 128, value=-1.0e12, huge=2.0 ** 110)


@pytest.mark.parametrize("dtype,mag", [(torch.bfloat16, 1.0e3), (torch.bfloat16, 1.0e5), (torch.bfloat16, 1.0e9), (torch.float16, 2.0e3)])
@pytest.mark.parametrize("causal", [True, False])
def test_packed_large_scores(ops, causal, dtype, mag):
    # scores of 10^6 to 10^18, whose product with the scale is rounded by more than the weights' range
    packed_as_before(ops, [300, 520], 4, 2, 128, dtype, causal, mag=mag)


@pytest.mark.parametrize("scale", [1.0, 3.0e38])
def test_packed_one_score_far_above_all_others(ops, scale):
    # a score times scale beyond f32: its key has all the weight
    n, at = 500, 201
    q, k, v = randn((n, 2, 128), torch.bfloat16, 1), randn((n, 1, 128), torch.bfloat16, 2), randn((n, 1, 128), torch.bfloat16, 3)
    q[:, :, C], k[at, :, C] = 1, -LOWEST
    got = ops.attention_packed(q, k, v, offsets([n]), scale=scale)
    ops.check_status()
    assert torch.equal(got[at:], v[at].expand(n - at, 2, 128))
    assert torch.isfinite(got[:at]).all()


def small_weights(n, dim):
    """One key far above n - 1 equal ones, 25.5 bits lower, which hold all that some columns get."""
    q, k = torch.zeros((n, 1, dim), dtype=torch.float16, device=DEV), torch.zeros((n, 1, dim), dtype=torch.float16, device=DEV)
    q[..., C], k[0, 0, C] = 4, 25.5 * math.log(2) * math.sqrt(dim) / 4
    v = 1 + randn((n, 1, dim), torch.float16, 3).abs()
    v[0, :, dim // 2:] = 0
    return q, k, v


def small_tolerance(q, k, v):
    # half a step for the output and for each weight, the f32 terms of test_gpu_ops, and for weights below
    # the normal range, which are kept 2^7 times larger than they are, 2^-32 of the largest one each;
    # an output below the normal range is off by 2^-25
    dim, scale = q.shape[-1], 1 / math.sqrt(q.shape[-1])
    s = q[:, 0].double() @ k[:, 0].double().T * scale
    p = torch.softmax(s, 1)
    out, size = p @ v[:, 0].double(), p @ v[:, 0].double().abs()
    delta = (dim + 4) * 2.0 ** -24 * scale * (q[:, 0].double().abs() @ k[:, 0].double().abs().T).amax(1, keepdim=True)
    tol = 2.0 ** -11 * out.abs() + (2.0 ** -11 + 2 * delta + 2.0 ** -20) * size
    return out, tol + 2.0 ** -32 * v[:, 0].double().abs().sum(0)[None] + 2.0 ** -25


@pytest.mark.parametrize("dim", [64, 128])
def test_packed_small_weights_in_half_precision(ops, dim):
    q, k, v = small_weights(2900, dim)
    got = ops.attention_packed(q, k, v, offsets([2900]), causal=False)
    want, tol = small_tolerance(q, k, v)
    close(got[:, 0], want, tol)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("rows", [1, 40])
def test_tree_small_weights_in_half_precision(ops, rows, dim):
    n = 6000
    q, k, v = small_weights(n, dim)
    pages, table = make_pages(random.Random(3), [n])
    data = torch.zeros((pages, 1, 2, 1, 64, dim), dtype=torch.float16, device=DEV)
    pos = torch.arange(n, device=DEV)
    page = ints(table[0]).long()[pos // 64]
    data[page, 0, 0, 0, pos % 64], data[page, 0, 1, 0, pos % 64] = k[:, 0], v[:, 0]
    mask = ints(np.full(rows, -1, dtype=np.int64), torch.int64)  # every row sees every drafted one
    got = ops.attention_tree(q[:rows], ops.KvPool(data), 0, ints(table), ints([n - rows]), offsets([rows]), mask=mask)
    ops.check_status()
    want, tol = small_tolerance(q[:rows], k, v)
    close(got[:, 0], want, tol)


@pytest.mark.parametrize("at", [5, 130, 401, 2000])
def test_infinitely_high_scores_make_their_rows_nan(ops, at):
    # inf - inf in the row's own maximum; rows and sequences that do not see the key stay as they were
    n, dim = 2500, 128
    q, k, v = rows_of(n + 50, 2, dim, torch.bfloat16, 1), randn((n + 50, 2, dim), torch.bfloat16, 2), randn((n + 50, 2, dim), torch.bfloat16, 3)
    cu = offsets([n, 50])
    rng = random.Random(5)
    pages, table = make_pages(rng, [n, 50])
    data = torch.zeros((pages, 1, 2, 2, 64, dim), dtype=torch.bfloat16, device=DEV)

    def both():
        for s, (a, m) in enumerate(((0, n), (n, 50))):
            pos = torch.arange(m, device=DEV)
            page = ints(table[s]).long()[pos // 64]
            data[page, 0, 0, :, pos % 64], data[page, 0, 1, :, pos % 64] = k[a:a + m], v[a:a + m]
        tree = ops.attention_tree(q[:7], ops.KvPool(data), 0, ints(table), ints([n - 3, 46]), offsets([3, 4]))
        out = ops.attention_packed(q, k, v, cu), ops.attention_packed(q, k, v, cu, causal=False), tree
        ops.check_status()
        return out

    clean = both()
    k[at, 1, C] = math.inf
    got = both()
    hit = torch.zeros_like(got[0], dtype=torch.bool)
    hit[at:n, 1] = True
    assert torch.isnan(got[0][hit]).all() and torch.equal(got[0][~hit], clean[0][~hit])
    hit[:n, 1] = True
    assert torch.isnan(got[1][hit]).all() and torch.equal(got[1][~hit], clean[1][~hit])
    assert torch.isnan(got[2][:3, 1]).all() and torch.equal(got[2][:, 0], clean[2][:, 0]) and torch.equal(got[2][3:], clean[2][3:])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("base", [0, 2 ** 11, 2 ** 14, 2 ** 15, 2 ** 18, 2 ** 22])
def test_weights_across_tiles_of_large_exact_scores(ops, base, dtype):
    # integer scores that f32 holds exactly, far above the differences that make the weights; every
    # tile raises the maximum by about what its predecessors' weights are scaled down for. The
    # exponent's constant is off by 2^-12 at most (a factor of 2^(2^-12) < 1 + 2^-12 for a tile
    # beside another), exp and the sums by 2^-20, each weight and the output by half a step.
    n, dim, nodes = 900, 64, 5
    q, k, v = (torch.zeros((n, 1, dim), dtype=dtype, device=DEV) for _ in range(3))
    side = 2 ** (math.frexp(max(base, 1))[1] // 2)
    q[..., 0], k[..., 0] = side, base // side
    g = torch.Generator(device=DEV).manual_seed(1)
    steps = torch.arange(n, device=DEV) // 128 * 50 + torch.randint(0, 50, (n,), generator=g, device=DEV)
    q[..., 1], q[..., 2], k[:, 0, 1], k[:, 0, 2] = 16, 1, (steps // 16).to(dtype), (steps % 16).to(dtype)
    v = randn((n, 1, dim), dtype, 3)
    scale = 1 / 8
    score = q[:, 0].double() @ k[:, 0].double().T
    assert torch.equal(score, score.round()) and float(score.max()) < 2 ** 23
    u = torch.finfo(dtype).eps / 2
    pages, table = make_pages(random.Random(3), [n])
    data = torch.zeros((pages, 1, 2, 1, 64, dim), dtype=dtype, device=DEV)
    pos = torch.arange(n, device=DEV)
    page = ints(table[0]).long()[pos // 64]
    data[page, 0, 0, 0, pos % 64], data[page, 0, 1, 0, pos % 64] = k[:, 0], v[:, 0]
    tree = ops.attention_tree(q[-nodes:], ops.KvPool(data), 0, ints(table), ints([n - nodes]), offsets([nodes]))
    for causal, got in ((True, ops.attention_packed(q, k, v, offsets([n]))), (False, ops.attention_packed(q, k, v, offsets([n]), causal=False)), (True, tree)):
        s = torch.where(sees(n, causal), score * scale, -math.inf)[-got.shape[0]:]
        p = torch.softmax(s, 1)
        want, size = p @ v[:, 0].double(), p @ v[:, 0].double().abs()
        tol = u * want.abs() + (u + 2 * 2.0 ** -12 + 2.0 ** -20) * size + 2.0 ** -32 * v[:, 0].double().abs().sum(0)[None]
        close(got[:, 0], want, tol, (base, causal))
    ops.check_status()
