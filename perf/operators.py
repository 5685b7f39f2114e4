"""Cases, plain forms and sizes of the long-context attention operators.

Two operators, forward and backward:

- ``relative_position_bias``: a learned bias by bucketed distance, spread
  over a [heads, queries, keys] grid, and the gradient of its table;
- ``packed_causal_attention``: causal attention over sequences of
  different lengths packed behind each other, with grouped key/value
  heads and, if wanted, that bias added to the scores.

``run`` computes a case in plain torch operations, or with the
framework's kernels where ``own`` is true.
"""

import math

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16,
          "fp32": torch.float32}


def listed():
    return [
        # one generated token against the keys so far: latency alone
        dict(name="bias, one token", op="bias", heads=16, q=1, k=1000,
             buckets=32, far=128, both=False, type="bf16", train=False),
        # a prompt's whole grid, as an unfused attention reads it
        dict(name="bias, prompt", op="bias", heads=16, q=2048, k=2048,
             buckets=32, far=128, both=False, type="bf16", train=False),
        # odd lengths, keys on both sides, in the table's master type
        dict(name="bias, odd, trained", op="bias", heads=12, q=777, k=1001,
             buckets=32, far=128, both=True, type="fp32", train=True),
        # a long training window
        dict(name="bias, long, trained", op="bias", heads=32, q=4096,
             k=4096, buckets=64, far=512, both=False, type="bf16",
             train=True),
        # the language model's own batch: 20 sequences of its 35 tokens,
        # 2 heads of 100
        dict(name="attention, language model", op="attention", heads=2,
             kv=2, dim=100, lens="35*20", buckets=0, far=0, train=True),
        # a serving batch of short prompts, ragged, grouped heads
        dict(name="attention, short prompts", op="attention", heads=16,
             kv=4, dim=64,
             lens="1,300,17,64,129,2,250,33,90,5,211,128,63,77,301,12,"
                  "40,199,65,8,150,23,280,101,3,55,260,31,119,70,1,96",
             buckets=0, far=0, train=False),
        # one long prompt
        dict(name="attention, long prompt", op="attention", heads=32, kv=8,
             dim=128, lens="8192", buckets=0, far=0, train=False),
        # documents of mixed length packed into one training window
        dict(name="attention, packed, trained", op="attention", heads=16,
             kv=4, dim=128, lens="2048,1,1500,777,2500,130,1236",
             buckets=0, far=0, train=True),
        # one long training window, grouped heads
        dict(name="attention, long, trained", op="attention", heads=32,
             kv=8, dim=128, lens="8192", buckets=0, far=0, train=True),
        # a prompt with the bias in the scores
        dict(name="biased, prompt", op="attention", heads=12, kv=12,
             dim=64, lens="4001", buckets=32, far=128, train=False),
        # packed documents with the bias, its table learned
        dict(name="biased, packed, trained", op="attention", heads=16,
             kv=16, dim=64, lens="1024,2047,333,1,691", buckets=32,
             far=128, train=True),
    ]


def draw(rng):
    def spread(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    buckets = rng.choice([8, 16, 32, 48, 64])
    far = spread(buckets + 1, 1024)
    if rng.random() < 0.4:
        q = rng.choice([1, spread(2, 4096)])
        k = max(q, spread(1, 4096)) if rng.random() < 0.7 else spread(1, 4096)
        heads = rng.randint(1, 32)
        return dict(op="bias", heads=heads, q=q, k=k, buckets=buckets,
                    far=far, both=rng.random() < 0.5,
                    type=rng.choice(["bf16", "fp16", "fp32"]),
                    train=rng.random() < 0.6)
    dim = rng.choice([32, 40, 50, 64, 72, 80, 96, 100, 112, 128])
    group = rng.choice([1, 1, 2, 4, 8])
    kv = rng.choice([1, 2, 3, 4, 8])
    count = spread(1, 48)
    longest = spread(16, 4096)
    lens = [min(longest, spread(1, longest)) for _ in range(count - 1)]
    lens.append(longest)
    rng.shuffle(lens)
    # the padded grid of the plain form stays under that of the largest case
    while len(lens) > 1 and len(lens) * longest ** 2 * kv * group > 2 ** 30:
        lens.remove(min(lens))
    biased = rng.random() < 0.5
    return dict(op="attention", heads=kv * group, kv=kv, dim=dim,
                lens=",".join(map(str, lens)),
                buckets=buckets if biased else 0, far=far if biased else 0,
                train=rng.random() < 0.6)


def _lengths(case):
    lens = []
    for part in case["lens"].split(","):
        n, _, times = part.partition("*")
        lens += [int(n)] * int(times or 1)
    return lens


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)

    def normal(*shape, scale=1.0, dtype=torch.bfloat16):
        x = torch.empty(shape, device=dev).normal_(generator=gen)
        return x.mul_(scale).to(dtype)

    state = dict(case)
    if case["buckets"]:
        # the least distance of each bucket of one side: the whole numbers
        # up to half of them, then even steps of the distance's logarithm
        # up to `far`; bucket b + t of the L upper ones begins at the
        # first n with n >= b * (far / b) ** (t / L), in whole numbers
        side = case["buckets"] // 2 if case.get("both") else case["buckets"]
        b, far = side // 2, case["far"]
        steps = side - b
        starts = list(range(b + 1))
        for t in range(1, steps):
            n = starts[-1]
            while n ** steps < far ** t * b ** (steps - t):
                n += 1
            starts.append(n)
        state["starts"] = torch.tensor(starts, device=dev)
        state["reach"] = (max(case["q"], case["k"])
                          if case["op"] == "bias" else max(_lengths(case)))
    if case["op"] == "bias":
        dtype = _TYPES[case["type"]]
        state["table"] = normal(case["buckets"], case["heads"], dtype=dtype)
        if case["train"]:
            state["table"].requires_grad_()
            state["dout"] = normal(case["heads"], case["q"], case["k"],
                                   dtype=dtype)
        return state

    lens = _lengths(case)
    total, heads, kv, dim = sum(lens), case["heads"], case["kv"], case["dim"]
    state["q"] = normal(total, heads, dim)
    state["k"] = normal(total, kv, dim)
    state["v"] = normal(total, kv, dim)
    if case["buckets"]:
        state["table"] = normal(case["buckets"], heads)
    if case["train"]:
        state["do"] = normal(total, heads, dim)
        for name in ("q", "k", "v", "table"):
            if name in state:
                state[name].requires_grad_()
    # where each sequence's rows stand, for the padded plain form
    n = torch.tensor(lens, device=dev)
    pos = torch.arange(max(lens), device=dev)
    state["there"] = pos < n[:, None]
    first = n.cumsum(0) - n
    state["rows"] = (first[:, None] + pos).masked_fill(~state["there"], 0)
    if own:
        from dynamic_load_balance_distributeddnn_amd.ops import \
            functional as FD
        state["packing"] = FD.PackedSequences(lens, device=dev)
    return state


# ------------------------------------------------------------ plain forms
def _bucket_of(distance, starts):
    return (distance[:, None] >= starts).sum(-1) - 1


def _bucket_of_gap(state, gap, both):
    """Buckets of `gap`, how far the key stands behind the query."""
    by_distance = _bucket_of(torch.arange(state["reach"], device=gap.device),
                             state["starts"])
    if both:
        return by_distance[gap.abs()] + (gap < 0) * len(state["starts"])
    return by_distance[gap.clamp(min=0)]


def _bias_grid(state, table, q_len, k_len, both):
    """[heads, q, k] bias in 32 bits."""
    i = torch.arange(q_len, device=table.device)[:, None] + (k_len - q_len)
    gap = i - torch.arange(k_len, device=table.device)
    return table.float().t()[:, _bucket_of_gap(state, gap, both)]


def _table_grad(state, dgrid, both):
    """Sums of [heads, q, k] by bucket, in 64 bits: they run long.  Rows
    shifted against each other turn diagonals into columns."""
    heads, q_len, k_len = dgrid.shape
    wide = q_len + k_len - 1
    skewed = torch.nn.functional.pad(dgrid.flip(1), (0, q_len))
    skewed = skewed.reshape(heads, -1)[:, :q_len * wide]
    sums = skewed.reshape(heads, q_len, wide).sum(1, dtype=torch.float64)
    gap = k_len - 1 - torch.arange(wide, device=dgrid.device)
    hot = (_bucket_of_gap(state, gap, both)[:, None]
           == torch.arange(state["buckets"], device=dgrid.device)).double()
    return (sums @ hot).t().to(state["table"].dtype)


def _plain_bias(state):
    table = state["table"]
    bias = _bias_grid(state, table, state["q"], state["k"], state["both"])
    out = {"bias": bias.to(table.dtype)}
    if state["train"]:
        out["dtable"] = _table_grad(state, state["dout"], state["both"])
    return out


def _plain_attention(state):
    rows, there = state["rows"], state["there"]
    heads, kv, dim = state["heads"], state["kv"], state["dim"]
    batch, longest = rows.shape
    scale = dim ** -0.5

    def padded(x):  # [batch, kv, heads per kv head, longest, dim], 32 bits
        x = x.float()[rows] * there[:, :, None, None]
        x = x.reshape(batch, longest, kv, -1, dim)
        return x.permute(0, 2, 3, 1, 4).contiguous()

    def packed(x):  # and back
        x = x.permute(0, 3, 1, 2, 4).reshape(batch, longest, -1, dim)
        return x[there].to(torch.bfloat16)

    q, k, v = padded(state["q"]), padded(state["k"]), padded(state["v"])
    s = (q @ k.transpose(-1, -2).contiguous()).mul_(scale)
    if state["buckets"]:
        bias = _bias_grid(state, state["table"], longest, longest, False)
        s += bias.reshape(kv, -1, longest, longest)
    at = torch.arange(longest, device=s.device)
    s.masked_fill_(at[:, None] < at, -math.inf)
    p = s.sub_(s.amax(-1, keepdim=True)).exp_()
    p /= p.sum(-1, keepdim=True)
    out = {"o": packed(p @ v)}
    if not state["train"]:
        return out
    do = padded(state["do"])
    dv = (p.transpose(-1, -2).contiguous() @ do).sum(2, keepdim=True)
    ds = do @ v.transpose(-1, -2).contiguous()
    ds -= (p * ds).sum(-1, keepdim=True)
    ds *= p
    del p
    out["dv"] = packed(dv)
    if state["buckets"]:
        out["dtable"] = _table_grad(
            state, ds.sum(0).reshape(heads, longest, longest), False)
    out["dq"] = packed((ds @ k).mul_(scale))
    out["dk"] = packed((ds.transpose(-1, -2).contiguous() @ q)
                       .sum(2, keepdim=True).mul_(scale))
    return out


def _own_bias(state):
    from dynamic_load_balance_distributeddnn_amd.ops import functional as FD
    bias = FD.relative_position_bias(
        state["table"], state["q"], state["k"],
        max_distance=state["far"], bidirectional=state["both"])
    if not state["train"]:
        return {"bias": bias}
    dtable, = torch.autograd.grad(bias, state["table"], state["dout"])
    return {"bias": bias.detach(), "dtable": dtable}


def _own_attention(state):
    from dynamic_load_balance_distributeddnn_amd.ops import functional as FD
    extra = {}
    if state["buckets"]:
        extra = dict(bias_table=state["table"], max_distance=state["far"])
    o = FD.packed_causal_attention(state["q"], state["k"], state["v"],
                                   state["packing"], **extra)
    if not state["train"]:
        return {"o": o}
    names = ["q", "k", "v"] + (["table"] if state["buckets"] else [])
    grads = torch.autograd.grad(o, [state[n] for n in names], state["do"])
    return {"o": o.detach(), **{"d" + n: g for n, g in zip(names, grads)}}


def run(state):
    if own:
        return (_own_bias if state["op"] == "bias" else _own_attention)(state)
    with torch.no_grad():
        return (_plain_bias if state["op"] == "bias"
                else _plain_attention)(state)


def work(case):
    if case["op"] == "bias":
        size = 4 if case["type"] == "fp32" else 2
        grid = case["heads"] * case["q"] * case["k"]
        table = case["heads"] * case["buckets"]
        return {"bytes": (2 if case["train"] else 1) * (grid + table) * size,
                "flops": grid if case["train"] else 0}
    lens = _lengths(case)
    pairs = sum(n * (n + 1) // 2 for n in lens) * case["heads"]
    row = sum(lens) * case["dim"] * 2
    table = case["heads"] * case["buckets"] * 2
    # forward: the scores and the weighted values; backward: the scores
    # again, the weights' gradient, and the products to q, k and v
    products, heads_moved = 2, 2 * case["heads"] + 2 * case["kv"]
    if case["train"]:
        products += 5
        heads_moved += 2 * case["heads"] + 2 * case["kv"]
        table *= 2
    return {"bytes": row * heads_moved + table,
            "flops": 2 * products * pairs * case["dim"]}


# ------------------------------------------------- the definition, 64 bits
def _bucket_by_count(longest, side, far):
    """Bucket of every distance below `longest`: itself below half the
    buckets, else half plus how many steps of the logarithm it has passed."""
    half = side // 2
    steps = side - half
    found = []
    for n in range(longest):
        if n < half:
            found.append(n)
        elif n >= far:
            found.append(side - 1)
        else:
            passed = [t for t in range(1, steps)
                      if n ** steps * half ** t >= far ** t * half ** steps]
            found.append(half + len(passed))
    return found


def exact(case, seed):
    state = prepare(case, seed)
    buckets = case["buckets"]
    if case["op"] == "bias":
        q_len, k_len, both = case["q"], case["k"], case["both"]
        side = buckets // 2 if both else buckets
        table = state["table"].detach().double()
        by = torch.tensor(_bucket_by_count(max(q_len, k_len), side,
                                           case["far"]), device=table.device)
        out = torch.empty(case["heads"], q_len, k_len, dtype=torch.float64,
                          device=table.device)
        grad = torch.zeros_like(table)
        rows = torch.arange(q_len, device=table.device) + k_len - q_len
        gap = rows[:, None] - torch.arange(k_len, device=table.device)
        which = torch.where(gap >= 0, by[gap.clamp(min=0)],
                            by[(-gap).clamp(min=0)] + side if both
                            else torch.zeros_like(gap))
        for h in range(case["heads"]):
            out[h] = table[:, h][which]
            if case["train"]:
                d = state["dout"][h].double()
                for b in range(buckets):
                    grad[b, h] = d[which == b].sum()
        return {"bias": out, **({"dtable": grad} if case["train"] else {})}

    lens, dim = _lengths(case), case["dim"]
    group = case["heads"] // case["kv"]
    q, k, v = (state[n].detach().double() for n in "qkv")
    o, dq, dk, dv = (torch.zeros_like(x) for x in (q, q, k, v))
    if buckets:
        table = state["table"].detach().double()
        dtable = torch.zeros_like(table)
        by = torch.tensor(_bucket_by_count(max(lens), buckets, case["far"]),
                          device=q.device)
    first = 0
    for n in lens:
        at = slice(first, first + n)
        first += n
        i = torch.arange(n, device=q.device)
        gap = i[:, None] - i
        for h in range(case["heads"]):
            g = h // group
            s = q[at, h] @ k[at, g].t() / math.sqrt(dim)
            if buckets:
                which = by[gap.clamp(min=0)]
                s = s + table[:, h][which]
            p = torch.softmax(s.masked_fill(gap < 0, -math.inf), -1)
            o[at, h] = p @ v[at, g]
            if not case["train"]:
                continue
            d = state["do"][at, h].double()
            dv[at, g] += p.t() @ d
            dp = d @ v[at, g].t()
            ds = p * (dp - (p * dp).sum(-1, keepdim=True))
            dq[at, h] = ds @ k[at, g] / math.sqrt(dim)
            dk[at, g] += ds.t() @ q[at, h] / math.sqrt(dim)
            if buckets:
                for b in range(buckets):
                    dtable[b, h] += ds[(which == b) & (gap >= 0)].sum()
    out = {"o": o}
    if case["train"]:
        out.update(dq=dq, dk=dk, dv=dv)
        if buckets:
            out["dtable"] = dtable
    return out
