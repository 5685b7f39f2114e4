"""The bucketed relative position bias against its definition."""

import pytest
import torch

from longctx_reference import bucket_by_count

pytestmark = pytest.mark.gpu

HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8,
             torch.float16: 2.0 ** -11}


def _fd():
    from dynamic_load_balance_distributeddnn_amd.ops import functional as FD
    return FD


def _buckets(q_len, k_len, buckets, far, both):
    side = buckets // 2 if both else buckets
    by = torch.tensor([bucket_by_count(n, side, far)
                       for n in range(max(q_len, k_len, 1))])
    gap = (torch.arange(q_len)[:, None] + k_len - q_len
           - torch.arange(k_len))
    if both:
        return (by[gap.abs()] + (gap < 0) * side).cuda()
    return by[gap.clamp(min=0)].cuda()


def _table(buckets, heads, dtype, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(buckets, heads, device="cuda", generator=gen).to(dtype)


def _check_grad(got, dout, which, buckets, out_type):
    """Sums of fp32 values in any order of n additions: each is off by at
    most a half step of a partial sum, themselves below sum |x|; a thread
    adds 512 rows at most, then 8 or so of its neighbours' sums, then
    trees: below 2**10 additions in a row."""
    d = dout.double()
    for b in range(buckets):
        part = torch.where(which == b, d, 0.0)
        want = part.sum((1, 2))
        room = 2.0 ** 10 * 2.0 ** -24 * part.abs().sum((1, 2))
        room = room + HALF_STEP[out_type] * (want.abs() + room)
        off = (got[b].double() - want).abs()
        assert bool((off <= room + 1e-30).all()), (b, off, room)


SHAPES = [(1, 1), (1, 1000), (1, 4097), (7, 5), (5, 7), (64, 64), (65, 63),
          (127, 1025), (300, 300), (513, 511), (2, 2056), (3, 6001), (70, 3),
          (129, 2048), (1030, 17)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16,
                                   torch.float32])
@pytest.mark.parametrize("both", [False, True])
@pytest.mark.parametrize("q_len,k_len", SHAPES)
def test_forward_and_gradient(q_len, k_len, both, dtype):
    print(q_len, k_len, both, dtype, flush=True)
    FD = _fd()
    for heads, buckets, far in ((3, 32, 128), (1, 8, 9)):
        table = _table(buckets, heads, dtype).requires_grad_()
        out = FD.relative_position_bias(table, q_len, k_len, far, both)
        which = _buckets(q_len, k_len, buckets, far, both)
        assert out.dtype == dtype
        assert torch.equal(out, table.detach().t()[:, which])
        gen = torch.Generator(device="cuda").manual_seed(q_len)
        dout = torch.randn(out.shape, device="cuda", generator=gen).to(dtype)
        grad, = torch.autograd.grad(out, table, dout)
        assert grad.dtype == dtype
        _check_grad(grad, dout, which, buckets, dtype)


@pytest.mark.parametrize("q_len,k_len", [(900, 2500), (2500, 900)])
def test_far_apart_lengths(q_len, k_len):
    FD = _fd()
    for both in (False, True):
        table = _table(256, 2, torch.float32).requires_grad_()
        out = FD.relative_position_bias(table, q_len, k_len, 2000, both)
        which = _buckets(q_len, k_len, 256, 2000, both)
        assert torch.equal(out, table.detach().t()[:, which])
        dout = torch.randn_like(out)
        grad, = torch.autograd.grad(out, table, dout)
        _check_grad(grad, dout, which, 256, torch.float32)


def test_many_heads_and_repeats():
    FD = _fd()
    table = _table(32, 40, torch.bfloat16).requires_grad_()
    out = FD.relative_position_bias(table, 333, 1111)
    which = _buckets(333, 1111, 32, 128, False)
    assert torch.equal(out, table.detach().t()[:, which])
    dout = torch.randn_like(out)
    first, = torch.autograd.grad(out, table, dout, retain_graph=True)
    for _ in range(3):
        again, = torch.autograd.grad(out, table, dout, retain_graph=True)
        assert torch.equal(first, again)


def test_expanded_gradient_and_table_view():
    FD = _fd()
    wide = _table(32, 8, torch.float32)
    table = wide[:, ::2].requires_grad_()
    out = FD.relative_position_bias(table, 50, 60)
    which = _buckets(50, 60, 32, 128, False)
    assert torch.equal(out, table.detach().t()[:, which])
    grad, = torch.autograd.grad(out.sum(), table)
    counts = torch.bincount(which.flatten(), minlength=32).float()
    assert torch.equal(grad, counts[:, None].expand(32, 4))


@pytest.mark.parametrize("shift", [1, 3])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_gradient_without_alignment(dtype, shift):
    FD = _fd()
    table = _table(32, 3, dtype).requires_grad_()
    out = FD.relative_position_bias(table, 61, 77)
    room = torch.randn(out.numel() + shift, device="cuda").to(dtype)
    dout = room[shift:].view(out.shape)
    grad, = torch.autograd.grad(out, table, dout)
    _check_grad(grad, dout, _buckets(61, 77, 32, 128, False), 32, dtype)


def test_values_that_are_no_numbers():
    """They come through where they are, and only there."""
    FD = _fd()
    table = _table(32, 2, torch.float32)
    table[3] = float("-inf")
    table[7] = torch.finfo(torch.float32).min
    table[9] = float("nan")
    table.requires_grad_()
    out = FD.relative_position_bias(table, 70, 70)
    which = _buckets(70, 70, 32, 128, False)
    want = table.detach().t()[:, which]
    assert torch.equal(out.nan_to_num(1e9), want.nan_to_num(1e9))
    dout = torch.ones_like(out)
    dout[0, 30, 10] = float("nan")
    grad, = torch.autograd.grad(out, table, dout)
    hit = which[30, 10].item()
    assert torch.isnan(grad[hit, 0])
    assert int(torch.isnan(grad).sum()) == 1


def test_autocast_reads_the_master_in_bf16():
    """The grid is bf16, the master's gradient stays fp32."""
    FD = _fd()
    table = _table(32, 4, torch.float32).requires_grad_()
    with torch.autocast("cuda", dtype=torch.bfloat16):
        out = FD.relative_position_bias(table, 100, 100)
    which = _buckets(100, 100, 32, 128, False)
    assert torch.equal(out, table.detach().bfloat16().t()[:, which])
    dout = torch.randn_like(out)
    grad, = torch.autograd.grad(out, table, dout)
    assert grad.dtype == torch.float32
    _check_grad(grad, dout, which, 32, torch.float32)


def test_offsets_past_32_bits():
    FD = _fd()
    heads, keys, tail = 2, 2 ** 30 + 5, 400
    assert heads * keys > 2 ** 31
    table = _table(32, heads, torch.bfloat16).requires_grad_()
    out = FD.relative_position_bias(table, 1, keys)
    far = table.detach()[31]
    assert torch.equal(out[:, 0, -tail:],
                       FD.relative_position_bias(table, 1, tail)[:, 0])
    for start in (0, 2 ** 29, keys - tail - 1000):
        assert bool((out[:, 0, start:start + 1000] == far[:, None]).all())
    dout = torch.zeros_like(out)
    dout[:, :, -tail:] = torch.randn(heads, 1, tail, device="cuda")
    dout[:, :, :tail] = torch.randn(heads, 1, tail, device="cuda")
    got, = torch.autograd.grad(out, table, dout)
    ends = torch.cat([dout[:, :, :tail], dout[:, :, -tail:]], 2)
    which = torch.cat([torch.full((1, tail), 31, device="cuda"),
                       _buckets(1, tail, 32, 128, False)], 1)
    _check_grad(got, ends, which, 32, torch.bfloat16)


def test_empty():
    FD = _fd()
    table = _table(32, 4, torch.float32).requires_grad_()
    for q_len, k_len in ((0, 5), (5, 0), (0, 0)):
        out = FD.relative_position_bias(table, q_len, k_len)
        assert out.shape == (4, q_len, k_len)
        grad, = torch.autograd.grad(out, table, torch.zeros_like(out))
        assert bool((grad == 0).all())


def test_captured_and_replayed():
    FD = _fd()
    table = _table(32, 4, torch.bfloat16)
    dout = torch.randn(4, 129, 257, device="cuda").bfloat16()

    def both():
        leaf = table.detach().requires_grad_()
        out = FD.relative_position_bias(leaf, 129, 257)
        return out.detach(), torch.autograd.grad(out, leaf, dout)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, grad = both()
    for seed in range(4):
        table.copy_(_table(32, 4, torch.bfloat16, seed))
        dout.normal_()
        graph.replay()
        want = both()
        torch.cuda.synchronize()
        assert torch.equal(out, want[0]) and torch.equal(grad, want[1])


def test_with_attention_as_used():
    """A layer with the learned bias: fused attention agrees with the
    unfused one that reads the grid, and both train the same table."""
    from longctx_reference import attention, check

    from dynamic_load_balance_distributeddnn_amd.ops import layers
    FD = _fd()
    torch.manual_seed(0)
    lens, heads, kv, d = [90, 133, 1], 4, 2, 64
    rows = sum(lens)
    bias = layers.RelativePositionBias(heads).cuda()
    with torch.no_grad():
        bias.weight.normal_()
    proj = layers.Linear(48, (heads + 2 * kv) * d).cuda()
    x = torch.randn(rows, 48, device="cuda")
    packing = FD.PackedSequences(lens, device="cuda")
    with torch.autocast("cuda", dtype=torch.bfloat16):
        qkv = proj(x).view(rows, heads + 2 * kv, d)
        q, k, v = qkv.split([heads, kv, kv], dim=1)
        o = bias.attend(q, k, v, packing)
    do = torch.randn_like(o)
    grads = torch.autograd.grad(o, [qkv, bias.weight, proj.weight], do)
    want, tol = attention(q, k, v, lens, table=bias.weight, do=do)
    check(o, want["o"], tol["o"], "o")
    check(grads[1], want["dtable"], tol["dtable"], "dtable")
    check(grads[0], torch.cat([want["dq"], want["dk"], want["dv"]], 1),
          torch.cat([tol["dq"], tol["dk"], tol["dv"]], 1), "dqkv")
    assert bool(torch.isfinite(grads[2]).all())
    # the grid, as an unfused attention of the second sequence reads it
    grid = bias(lens[1], lens[1])
    at = slice(lens[0], lens[0] + lens[1])
    s = torch.einsum("ihd,jhd->hij", q[at].double(),
                     k[at].double().repeat_interleave(2, 1)) * d ** -0.5
    s = s + grid.double()
    s = s.masked_fill(torch.ones_like(s[0]).triu(1).bool(), float("-inf"))
    p = torch.softmax(s, -1)
    plain = torch.einsum("hij,jhd->ihd", p,
                         v[at].double().repeat_interleave(2, 1))
    check(o[at], plain, tol["o"][at] + 1e-6, "unfused")
