"""Packed causal attention where single entries of its results can go wrong:
the far bucket's gradient, exactness of the keys', biases that drown the
scores, infinities that a row does see, rows far apart, autocast."""

import math

import pytest
import torch

from longctx_reference import (SECOND, SLACK, U, attention, bucket_by_count,
                               check)

pytestmark = pytest.mark.gpu


def _fd():
    from dynamic_load_balance_distributeddnn_amd.ops import functional as FD
    return FD


def _inputs(rows, heads, kv, d, seed=0, buckets=0, table_type=torch.float32):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, dtype=torch.bfloat16):
        return torch.randn(*shape, device="cuda", generator=gen).to(dtype)

    q, k, v = normal(rows, heads, d), normal(rows, kv, d), normal(rows, kv, d)
    do = normal(rows, heads, d)
    table = normal(buckets, heads, dtype=table_type) if buckets else None
    return q, k, v, do, table


def _run(q, k, v, do, lens, table=None, far=128):
    """All outputs by name."""
    FD = _fd()
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    extra = {}
    if table is not None:
        leaves.append(table.detach().requires_grad_())
        extra = dict(bias_table=leaves[3], max_distance=far)
    o = FD.packed_causal_attention(
        *leaves[:3], FD.PackedSequences(lens, device=q.device), **extra)
    grads = torch.autograd.grad(o, leaves, do)
    return dict(zip(("o", "dq", "dk", "dv", "dtable"),
                    (o.detach(), *grads)))


def _exact_delta(q, k, v, lens, do, table=None, far=128):
    """dK and the table's gradient in 64 bits, with bounds in which delta
    has no part: it is exact to fp32 there.

    A weight and its gradient are off by SLACK of the sums without signs
    (see the reference); dK's operand dS is rounded to bf16 once, the
    result once; the table's gradient is a sum in fp32 of each bucket's own
    pairs, so no other bucket is in its bound.
    """
    q, k, v, do = (t.detach().double() for t in (q, k, v, do))
    heads, d = q.shape[1:]
    group = heads // k.shape[1]
    val = {"dk": torch.zeros_like(k)}
    tol = {"dk": torch.zeros_like(k)}
    last_step = 2.0 ** -24
    if table is not None:
        last_step = U if table.dtype == torch.bfloat16 else last_step
        table = table.detach().double()
        val["dtable"] = torch.zeros_like(table)
        tol["dtable"] = torch.zeros_like(table)
        by = torch.tensor([bucket_by_count(n, table.shape[0], far)
                           for n in range(max(lens))], device=q.device)
    first = 0
    for n in lens:
        at = slice(first, first + n)
        first += n
        i = torch.arange(n, device=q.device)
        gap = i[:, None] - i
        for h in range(heads):
            g = h // group
            s = q[at, h] @ k[at, g].T * d ** -0.5
            if table is not None:
                which = by[gap.clamp(min=0)]
                s = s + table[:, h][which]
            s = s.masked_fill(gap < 0, -math.inf)
            top = s.amax(-1, keepdim=True)
            p = torch.exp(s - top.masked_fill(top == -math.inf, 0))
            total = p.sum(-1, keepdim=True)
            p = p / total.masked_fill(total == 0, 1)
            o, dh, vh = p @ v[at, g], do[at, h], v[at, g]
            ds = p * (dh @ vh.T - (dh * o).sum(-1, keepdim=True))
            e = SLACK * p * (dh.abs() @ vh.abs().T
                             + (dh * o).abs().sum(-1, keepdim=True))
            qh = q[at, h] * d ** -0.5
            val["dk"][at, g] += ds.T @ qh
            tol["dk"][at, g] += (U * ds.abs() + e).T @ qh.abs()
            if table is not None:
                for b in range(table.shape[0]):
                    there = (which == b) & (gap >= 0)
                    val["dtable"][b, h] += ds[there].sum()
                    tol["dtable"][b, h] += e[there].sum()
    tol["dk"] = SECOND * (tol["dk"] + U * val["dk"].abs())
    if table is not None:
        tol["dtable"] = SECOND * (tol["dtable"]
                                  + last_step * val["dtable"].abs())
    return val, tol


# ------------------------------------------------ the far bucket's gradient
@pytest.mark.parametrize("lens,far", [([35] * 20, 128), ([100, 64, 1], 128),
                                      ([300, 900], 2000)])
@pytest.mark.parametrize("heads,kv,d", [(4, 4, 64), (4, 2, 100)])
def test_a_bucket_that_no_pair_reaches_has_no_gradient(lens, far, heads, kv,
                                                       d):
    buckets = 32
    q, k, v, do, table = _inputs(sum(lens), heads, kv, d, buckets=buckets)
    reached = {bucket_by_count(n, buckets, far) for n in range(max(lens))}
    out = [b for b in range(buckets) if b not in reached]
    assert buckets - 1 in out
    got = _run(q, k, v, do, lens, table, far)["dtable"]
    assert bool((got[out] == 0).all()), got[out]


@pytest.mark.parametrize("low", [-math.inf, -1e4,
                                 torch.finfo(torch.float32).min])
@pytest.mark.parametrize("lens,far", [([700, 40], 128), ([2500], 2000)])
def test_a_far_bucket_that_masks_has_no_gradient(low, lens, far):
    """A row has a weight at distance 0, so what the far bucket takes out
    has one of 0, and 0 is its sum."""
    q, k, v, do, table = _inputs(sum(lens), 4, 2, 64, buckets=32)
    table[31] = low
    got = _run(q, k, v, do, lens, table, far)
    assert bool((got["dtable"][31] == 0).all()), got["dtable"][31]
    want, tol = _exact_delta(q, k, v, lens, do, table, far)
    for name in want:
        check(got[name], want[name], tol[name], name)


@pytest.mark.parametrize("row", [20, 34])
def test_a_gradient_that_is_no_number_stays_in_its_buckets(row):
    """The first sequence does not reach the far bucket, the second does.
    Its last row is what the tile repeats behind the sequence."""
    lens = [35, 300]
    q, k, v, do, table = _inputs(335, 2, 2, 64, buckets=32)
    want, tol = _exact_delta(q[35:], k[35:], v[35:], [300], do[35:], table)
    do[row] = math.nan
    got = _run(q, k, v, do, lens, table)["dtable"]
    far = [b for b in range(32) if bucket_by_count(35, 32, 128) < b]
    assert 31 in far and bool(torch.isnan(got[0]).all())
    check(got[far], want["dtable"][far], tol["dtable"][far], "dtable")


@pytest.mark.parametrize("lens,heads,kv,d,far", [
    ([130, 1, 64], 4, 2, 100, 128), ([600, 300], 2, 2, 128, 128),
    ([2500, 900, 33], 4, 2, 64, 128), ([2500, 900, 33], 4, 1, 64, 2000),
    ([3000], 2, 2, 128, 300), ([1500], 40, 1, 32, 64)])
@pytest.mark.parametrize("buckets", [2, 32])
def test_keys_and_table_gradients_are_exact_in_delta(lens, heads, kv, d, far,
                                                     buckets):
    """Each bucket by its own pairs; sequences whose lists are cut too."""
    q, k, v, do, table = _inputs(sum(lens), heads, kv, d, buckets=buckets)
    want, tol = _exact_delta(q, k, v, lens, do, table, far)
    got = _run(q, k, v, do, lens, table, far)
    for name in want:
        check(got[name], want[name], tol[name], name)


@pytest.mark.parametrize("lens,heads,kv,d", [
    ([700, 129], 4, 2, 64), ([3000, 200], 2, 1, 128), ([2500], 2, 2, 64)])
@pytest.mark.parametrize("buckets", [0, 32])
def test_values_with_a_mean(lens, heads, kv, d, buckets):
    """delta is large where what it is taken off is the same for all keys:
    from the stored output it would be off by 2**-8 of that, many times
    what these bounds have room for (one list is cut, one is not)."""
    q, k, v, do, table = _inputs(sum(lens), heads, kv, d, buckets=buckets)
    v = (v.float() * 0.1 + 8).bfloat16()
    want, tol = _exact_delta(q, k, v, lens, do, table)
    got = _run(q, k, v, do, lens, table)
    for name in want:
        check(got[name], want[name], tol[name], name)


@pytest.mark.parametrize("lens,heads,kv", [([700, 40], 4, 2),
                                           ([2500], 2, 2)])
def test_one_bucket_for_both_halves_of_a_block(lens, heads, kv):
    """Distances 1 to 999 are one bucket: both halves of a wave add to it
    in every block."""
    q, k, v, do, table = _inputs(sum(lens), heads, kv, 64, buckets=3)
    assert bucket_by_count(999, 3, 10 ** 6) == 1
    want, tol = _exact_delta(q, k, v, lens, do, table, 10 ** 6)
    got = _run(q, k, v, do, lens, table, 10 ** 6)
    check(got["dtable"], want["dtable"], tol["dtable"], "dtable")
    again = _run(q, k, v, do, lens, table, 10 ** 6)
    assert torch.equal(got["dtable"], again["dtable"])


# ------------------------------------------ a finite far bias, large scores
@pytest.mark.parametrize("low", [-1e5, -1e10, -1e20])
@pytest.mark.parametrize("length,heads", [(600, 2), (2500, 2), (600, 16)])
@pytest.mark.parametrize("d", [64, 128])
def test_far_bias_that_drowns_large_scores(low, length, heads, d):
    """The first hundred keys have scores of some hundreds and are seen by
    rows far enough behind through the far bucket alone."""
    q, k, v, do, table = _inputs(length, heads, heads, d, buckets=32)
    k[:100] *= 60
    table[31] = low
    want, tol = attention(q, k, v, [length], table=table, do=do)
    got = _run(q, k, v, do, [length], table)
    for name, t in got.items():
        assert bool(torch.isfinite(t).all()), name
    for name in ("o", "dq"):  # rows that do not see them otherwise
        check(got[name][230:], want[name][230:], tol[name][230:], name)
    for name in ("dk", "dv"):  # keys that no other row sees
        check(got[name][230:], want[name][230:], tol[name][230:], name)


@pytest.mark.parametrize("high", [300.0, 1e4])
def test_far_bias_that_outweighs_all(high):
    """Rows that reach the far bucket weigh its keys alone: their scores
    are rounded at the bias's size, 2**-11 at most as exponents of 2."""
    q, k, v, do, table = _inputs(700, 2, 2, 64, buckets=32)
    table[31] = high
    want, tol = attention(q, k, v, [700], table=table, do=do)
    got = _run(q, k, v, do, [700], table)
    assert all(bool(torch.isfinite(t).all()) for t in got.values())
    first = next(n for n in range(200) if bucket_by_count(n, 32, 128) == 31)
    rows = slice(first + 1, 700)
    # a weight is off by 2 ** 2**-11 of itself, its row's sum too
    room = 2 * (2.0 ** (2.0 ** -11) - 1)
    for h in range(2):
        i = torch.arange(700, device="cuda")
        s = q[:, h].double() @ k[:, h].double().T / 8
        s = s.masked_fill(i[:, None] - i < first, -math.inf)[rows]
        p = torch.softmax(s, -1) @ v[:, h].double().abs()
        check(got["o"][rows, h], want["o"][rows, h],
              tol["o"][rows, h] + room * p, "o")


# ------------------------------------------- infinities that a row does see
@pytest.mark.parametrize("value", [math.inf, -math.inf])
@pytest.mark.parametrize("length,at", [(150, 5), (150, 70), (150, 129),
                                       (2500, 3), (2500, 2470)])
@pytest.mark.parametrize("biased", [False, True])
def test_an_infinite_value_stays_one_for_the_rows_that_see_it(value, length,
                                                              at, biased):
    lens = [40, length, 45]
    rows = sum(lens)
    q, k, v, do, table = _inputs(rows, 2, 1, 64,
                                 buckets=32 if biased else 0)
    want, tol = attention(q, k, v, lens, table=table)
    v[40 + at, :, 3:] = value
    got = _run(q, k, v, do, lens, table)["o"]
    sees = torch.zeros(rows, dtype=torch.bool, device="cuda")
    sees[40 + at:40 + length] = True
    assert bool((got[sees][..., 3:] == value).all())
    check(got[sees][..., :3], want["o"][sees][..., :3],
          tol["o"][sees][..., :3], "beside it")
    check(got[~sees], want["o"][~sees], tol["o"][~sees], "not seen")


# ------------------------------------------------------------- row strides
@pytest.mark.parametrize("rows,stride", [(3, 2 ** 24), (3, 2 ** 25 + 1),
                                         (1, 2 ** 40), (1, 77)])
def test_rows_far_apart(rows, stride):
    """A row stride that the kernels do not take is copied; the one of a
    single row says nothing."""
    q, k, v, do, _ = _inputs(rows, 2, 2, 64)
    want = _run(q, k, v, do, [rows])
    room = torch.empty((rows - 1) * stride + 128, dtype=torch.bfloat16,
                       device="cuda")
    for turn in range(4):
        given = [q, k, v, do]
        far = room.as_strided((rows, 2, 64), (stride, 64, 1))
        far.copy_(given[turn])
        given[turn] = far
        got = _run(*given, [rows])
        for name in want:
            assert torch.equal(got[name], want[name]), (turn, name)


# ---------------------------------------------------------------- autocast
@pytest.mark.parametrize("wide", ["q", "k", "v", "kv", "qkv"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_autocast_casts_each_of_the_three(wide, dtype):
    """To bfloat16, the kernels' one type, whatever type autocast names."""
    FD = _fd()
    q, k, v, do, _ = _inputs(90, 2, 2, 64)
    want = _run(q, k, v, do, [90])
    leaves = [(t.float() if n in wide else t).detach().requires_grad_()
              for n, t in zip("qkv", (q, k, v))]
    with torch.autocast("cuda", dtype=dtype):
        o = FD.packed_causal_attention(
            *leaves, FD.PackedSequences([90], device="cuda"))
    assert torch.equal(o.detach(), want["o"])
    for leaf, grad, name in zip(leaves, torch.autograd.grad(o, leaves, do),
                                ("dq", "dk", "dv")):
        assert grad.dtype == leaf.dtype
        assert torch.equal(grad, want[name].to(grad.dtype))
