"""Measured cases of the attention operators for training and serving: the forward over grouped heads that also gives
every row's log-sum-exp, its backward pass, and the learned relative position bias by buckets inside both.

`run` computes a case either in its plain form (elementary torch operations in float32) or, with `own` set, through the
calls a program makes of emmyptx.runtime. `exact` is the definition in float64, written apart from the plain form.
"""
import math
import os
import sys

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _case(op, dtype, batch, heads, kv_heads, sq, sk, d, causal=False, align="start", ragged=False, buckets=0, max_distance=128,
          bidirectional=True, rows_first=False, name=None):
    """`align`: where the queries stand among the keys ("start": query i at key i, "end": the last query at the last
    key); `ragged`: every batch entry has its own number of keys; `rows_first`: [batch, row, head, d] in memory instead
    of [batch, head, row, d]; `buckets`: size of the relative position table (0: no bias)."""
    c = {"op": op, "dtype": dtype, "batch": batch, "heads": heads, "kv_heads": kv_heads, "sq": sq, "sk": sk, "d": d, "causal": causal,
         "align": align, "ragged": ragged, "buckets": buckets, "max_distance": max_distance, "bidirectional": bidirectional,
         "rows_first": rows_first}
    if name is not None:
        c["name"] = name
    return c


def listed():
    return [
        # one request's single token against a short cache: launch latency
        _case("fwd", "bf16", 1, 8, 2, 1, 77, 128, causal=True, align="end", name="fwd_token_1x77"),
        # single tokens of a serving batch, grouped heads, every request with its own cache length: bound by the cache's bytes
        _case("fwd", "bf16", 32, 32, 8, 1, 8192, 128, causal=True, align="end", ragged=True, name="fwd_token_32x8192"),
        # fp32 attention at the size of the repository's own fp32 cases, with a bias
        _case("fwd", "f32", 2, 4, 4, 128, 128, 64, buckets=32, name="fwd_f32_128"),
        # an encoder layer with a relative position bias
        _case("fwd", "f16", 8, 12, 12, 512, 512, 64, buckets=32, name="fwd_bias_512"),
        # a prompt of odd length, grouped heads, rows first in memory as a projection leaves them
        _case("fwd", "bf16", 2, 32, 8, 2001, 2001, 128, causal=True, rows_first=True, name="fwd_causal_2001"),
        # the benchmark's attention configuration with the log-sum-exp a training step keeps
        _case("fwd", "bf16", 16, 16, 16, 4096, 4096, 128, name="fwd_4096"),
        # the smallest training step
        _case("bwd", "bf16", 1, 4, 4, 64, 64, 64, name="bwd_64"),
        # fp32 gradients, bias included, ragged keys
        _case("bwd", "f32", 2, 4, 4, 128, 128, 64, ragged=True, buckets=32, name="bwd_f32_128"),
        # the encoder layer's gradients, the bias table's among them
        _case("bwd", "f16", 8, 12, 12, 512, 512, 64, buckets=32, name="bwd_bias_512"),
        # a decoder's gradients with a one-sided bias, odd length, padded batch
        _case("bwd", "bf16", 4, 16, 16, 1000, 1000, 128, causal=True, ragged=True, buckets=32, bidirectional=False, name="bwd_bias_1000"),
        # grouped heads, causal, rows first
        _case("bwd", "bf16", 2, 32, 8, 2048, 2048, 128, causal=True, rows_first=True, name="bwd_causal_2048"),
        # the benchmark's long sequences
        _case("bwd", "bf16", 4, 16, 16, 4096, 4096, 128, name="bwd_4096"),
    ]


def _log_uniform(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """The same ranges: lengths 1 to 4096 (single tokens: caches up to 8192), odd ones included, every type; a case's
    pairs of rows and its cache bytes stay within the listed ones'."""
    op = rng.choice(["fwd", "bwd"])
    token = op == "fwd" and rng.random() < 0.3
    dtype = rng.choice(["f16", "bf16", "bf16"]) if token else rng.choice(["f16", "f16", "bf16", "bf16", "bf16", "f32"])
    d = rng.choice([64, 128]) if dtype != "f32" else rng.choice([32, 64, 96, 128])
    kv_heads = rng.choice([1, 2, 4, 8, 12, 16])
    group = rng.choice([1, 1, 2, 4, 8]) if kv_heads <= 8 else 1
    heads = kv_heads * group
    causal, align = rng.random() < 0.5, "start"
    if token:
        sq, sk = rng.choice([1, 1, 1, 2, 5]), _log_uniform(rng, 16, 8192)
        batch = _log_uniform(rng, 1, max(1, min(32, (32 * 8 * 8192) // (kv_heads * sk))))
        causal, align = True, "end"
    elif dtype == "f32":
        sq = _log_uniform(rng, 1, 256)
        sk = sq if rng.random() < 0.6 else _log_uniform(rng, 1, 256)
        batch = _log_uniform(rng, 1, max(1, min(4, 16 // heads)))
    else:
        sq = _log_uniform(rng, 32, 4096)
        sk = sq if causal or rng.random() < 0.6 else _log_uniform(rng, 32, 4096)
        pairs = (256 if op == "fwd" else 64) * 4096 * 4096 // 2
        batch = _log_uniform(rng, 1, max(1, min(16, pairs // (heads * sq * sk))))
        if causal and rng.random() < 0.4:                       # a chunk of queries at the end of a longer sequence
            sq, align = _log_uniform(rng, 1, sk), "end"
    buckets = rng.choice([0, 0, 8, 32, 64])
    return _case(op, dtype, batch, heads, kv_heads, sq, sk, d, causal=causal, align=align, ragged=rng.random() < 0.4, buckets=buckets,
                 max_distance=rng.choice([64, 128, 200]), bidirectional=not causal, rows_first=rng.random() < 0.4)


def _lens(case):
    """The key counts of the batch: the same multiset whatever the seed."""
    b, sk = case["batch"], case["sk"]
    if not case["ragged"]:
        return [sk] * b
    return [max(1, sk - sk // 5)] if b == 1 else [max(1, sk - (sk // 2) * i // (b - 1)) for i in range(b)]


def _pairs(case):
    """Visible (query, key) pairs of one head, over the batch."""
    sq, total = case["sq"], 0
    for n in _lens(case):
        if not case["causal"]:
            total += sq * n
            continue
        off = n - sq if case["align"] == "end" else 0
        total += sum(min(max(i + off + 1, 0), n) for i in range(sq))
    return total


def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    q = case["batch"] * case["heads"] * case["sq"] * case["d"]
    kv = sum(_lens(case)) * case["kv_heads"] * case["d"]
    rows = case["batch"] * case["heads"] * case["sq"]
    table = case["buckets"] * case["heads"] * 4
    pairs = _pairs(case) * case["heads"]
    if case["op"] == "fwd":
        return {"bytes": size * (2 * q + 2 * kv) + 4 * rows + table, "flops": 4.0 * case["d"] * pairs}
    # q, o, do in, dq out; k, v in, dk, dv out (of every key); lse in; the table in and its gradient out
    kv_out = case["batch"] * case["sk"] * case["kv_heads"] * case["d"]
    return {"bytes": size * (4 * q + 2 * kv + 2 * kv_out) + 4 * rows + 2 * table, "flops": 10.0 * case["d"] * pairs}


# ---- the relative position buckets -----------------------------------------------------------------------------------
def _side(case):
    nb = case["buckets"] // 2 if case["bidirectional"] else case["buckets"]
    return nb, nb // 2


def _first_distances(nb, e, max_distance):
    """The smallest distance of every bucket of one direction, in whole numbers: n / e >= (max_distance / e)^(k / m)."""
    m = nb - e
    far = [next(n for n in range(e, max_distance + 1) if n ** m >= e ** (m - k) * max_distance ** k) for k in range(m)]
    return list(range(e)) + far


def _runs(case):
    """Distances (key position - query position) in rising order as runs of one bucket: [(first distance, bucket)]."""
    nb, e = _side(case)
    first = _first_distances(nb, e, case["max_distance"])
    last = [b + 1 for b in range(nb - 1)]
    behind = [(-(first[b + 1] - 1), b) for b in reversed(range(len(last))) if first[b + 1] > first[b]]
    runs = [(-(1 << 30), nb - 1)] + behind
    if case["bidirectional"]:
        runs += [(first[b], nb + b) for b in range(1, nb) if b + 1 == nb or first[b + 1] > first[b]]
    return runs


# ---- inputs ----------------------------------------------------------------------------------------------------------
def _tensor(g, case, heads, rows, scale=1.0):
    b, d = case["batch"], case["d"]
    shape = (b, rows, heads, d) if case["rows_first"] else (b, heads, rows, d)
    t = torch.empty(shape, dtype=DTYPES[case["dtype"]], device="cuda").normal_(generator=g)
    if scale != 1.0:
        t.mul_(scale)
    return t.transpose(1, 2) if case["rows_first"] else t


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = {"case": dict(case)}
    s["q"] = _tensor(g, case, case["heads"], case["sq"])
    s["k"] = _tensor(g, case, case["kv_heads"], case["sk"])
    s["v"] = _tensor(g, case, case["kv_heads"], case["sk"])
    s["scale"] = case["d"] ** -0.5
    lens = torch.tensor(_lens(case), dtype=torch.int32)
    perm = torch.randperm(case["batch"], generator=torch.Generator().manual_seed(seed))
    s["lens"] = lens[perm].cuda() if case["ragged"] else None
    s["table"] = s["first"] = s["bucket"] = None
    if case["buckets"]:
        s["table"] = torch.empty(case["buckets"], case["heads"], device="cuda").normal_(generator=g)
        runs = _runs(case)
        s["first"] = torch.tensor([r[0] for r in runs[1:]], device="cuda")          # where each run but the first begins
        s["bucket"] = torch.tensor([r[1] for r in runs], device="cuda")
    if case["op"] == "bwd":
        s["do"] = _tensor(g, case, case["heads"], case["sq"])
        s["o"], s["lse"] = _plain_fwd(s)                                            # what the forward of the step left behind
    return s


# ---- the plain form --------------------------------------------------------------------------------------------------
def _positions(s):
    """Position of every query among the keys, [batch or 1, sq]; the keys' own positions, [sk]; key counts, [batch or 1, 1]."""
    c = s["case"]
    n = s["lens"].long()[:, None] if s["lens"] is not None else torch.full((1, 1), c["sk"], device="cuda")
    q_pos = torch.arange(c["sq"], device="cuda")[None, :] + (n - c["sq"] if c["align"] == "end" else 0 * n)
    return q_pos, torch.arange(c["sk"], device="cuda"), n


def _wide(t, s):
    """A key or value tensor in float32, one plane for every query head."""
    group = s["case"]["heads"] // s["case"]["kv_heads"]
    return t.float() if group == 1 else t.float().repeat_interleave(group, 1)


def _scores(s, q, k):
    """scale q k^T + bias with -inf where a query does not see a key."""
    q_pos, k_pos, n = _positions(s)
    x = torch.matmul(q, k.transpose(-1, -2)).mul_(s["scale"])
    if s["table"] is not None:
        dist = k_pos[None, None, :] - q_pos[:, :, None]
        bucket = s["bucket"][torch.bucketize(dist, s["first"], right=True)]
        x += s["table"].float().t()[:, bucket].transpose(0, 1)
    if s["lens"] is not None or s["case"]["causal"]:
        hidden = (k_pos[None, :] >= n)[:, None, :]
        if s["case"]["causal"]:
            hidden = hidden | (k_pos[None, None, :] > q_pos[:, :, None])
        x.masked_fill_(hidden[:, None], -math.inf)
    return x


def _plain_fwd(s):
    x = _scores(s, s["q"].float(), _wide(s["k"], s))
    m = x.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, torch.zeros_like(m), m)
    p = x.sub_(m).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p, _wide(s["v"], s)) / torch.where(total == 0, torch.ones_like(total), total)
    out = torch.empty_like(s["q"])
    out.copy_(o)
    return out, (m + total.log())[..., 0]


def _plain_bwd(s):
    c = s["case"]
    q, k, v, do = s["q"].float(), _wide(s["k"], s), _wide(s["v"], s), s["do"].float()
    lse = s["lse"][..., None]
    p = _scores(s, q, k).sub_(torch.where(lse == -math.inf, torch.zeros_like(lse), lse)).exp_()
    dv = torch.matmul(p.transpose(-1, -2), do)
    row = (do * s["o"].float()).sum(-1, keepdim=True)
    ds = torch.matmul(do, v.transpose(-1, -2)).sub_(row).mul_(p)
    dq = torch.matmul(ds, k).mul_(s["scale"])
    dk = torch.matmul(ds.transpose(-1, -2), q).mul_(s["scale"])
    shared = (c["batch"], c["kv_heads"], c["heads"] // c["kv_heads"], c["sk"], c["d"])
    grads = [dq.to(s["q"].dtype), dk.view(shared).sum(2).to(s["q"].dtype), dv.view(shared).sum(2).to(s["q"].dtype)]
    if s["table"] is None:
        return grads
    # a bucket's keys of one query are neighbours: differences of running sums at the runs' borders
    q_pos, _, _ = _positions(s)
    run = torch.nn.functional.pad(ds.cumsum(-1, dtype=torch.float64), (1, 0))
    border = (q_pos[:, :, None] + s["first"]).clamp(0, c["sk"])
    border = torch.nn.functional.pad(torch.nn.functional.pad(border, (1, 0)), (0, 1), value=c["sk"])
    sums = run.gather(-1, border[:, None].expand(c["batch"], c["heads"], -1, -1)).diff(dim=-1).sum((0, 2))
    dtable = torch.zeros(c["buckets"], c["heads"], dtype=torch.float64, device="cuda")
    dtable[s["bucket"]] = sums.t()
    return grads + [dtable.float()]


# ---- the framework's calls -------------------------------------------------------------------------------------------
def _runtime():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "emmy-ptx-compiler_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    from emmyptx import runtime
    return runtime


def _own(s):
    rt, c = _runtime(), s["case"]
    how = {"scale": s["scale"], "causal": c["causal"], "align": c["align"], "key_lens": s["lens"], "bias_table": s["table"],
           "max_distance": c["max_distance"], "bidirectional": c["bidirectional"]}
    if c["op"] == "fwd":
        return rt.attention_heads(s["q"], s["k"], s["v"], **how)
    return rt.attention_heads_backward(s["do"], s["q"], s["k"], s["v"], s["o"], s["lse"], **how)


def run(state):
    if own:
        return list(_own(state))
    return list(_plain_fwd(state) if state["case"]["op"] == "fwd" else _plain_bwd(state))


# ---- the definition in 64 bits ---------------------------------------------------------------------------------------
def _bucket_of(dist, case):
    nb, e = _side(case)
    side = torch.zeros_like(dist)
    n = -dist
    if case["bidirectional"]:
        side, n = (dist > 0).long() * nb, dist.abs()
    n = n.clamp(min=0)
    steps = torch.log(n.clamp(min=1).double() / e) / math.log(case["max_distance"] / e) * (nb - e)
    far = (e + torch.floor(steps + 1e-9).long()).clamp(max=nb - 1)                  # 1e-9: a border that is a whole number
    return side + torch.where(n < e, n, far)


def exact(case, seed):
    s = prepare(case, seed)
    c, scale = case, s["scale"]
    group = c["heads"] // c["kv_heads"]
    outs = {"o": [], "lse": [], "dq": [], "dk": [], "dv": []}
    dtable = torch.zeros(max(1, c["buckets"]), c["heads"], dtype=torch.float64, device="cuda")
    kp = torch.arange(c["sk"], device="cuda")
    for b in range(c["batch"]):
        n = int(s["lens"][b]) if s["lens"] is not None else c["sk"]
        qp = torch.arange(c["sq"], device="cuda") + (n - c["sq"] if c["align"] == "end" else 0)
        seen = (kp[None, :] < n).expand(c["sq"], c["sk"])
        if c["causal"]:
            seen = seen & (kp[None, :] <= qp[:, None])
        bucket = _bucket_of(kp[None, :] - qp[:, None], c) if c["buckets"] else None
        for hk in range(c["kv_heads"]):
            k, v = s["k"][b, hk].double(), s["v"][b, hk].double()
            dk, dv = torch.zeros_like(k), torch.zeros_like(v)
            for h in range(hk * group, (hk + 1) * group):
                q = s["q"][b, h].double()
                x = (q @ k.T) * scale
                if c["buckets"]:
                    x = x + s["table"][:, h].double()[bucket]
                x = torch.where(seen, x, torch.full_like(x, -math.inf))
                if c["op"] == "fwd":
                    lse = torch.logsumexp(x, -1)
                    p = torch.exp(x - lse[:, None]).nan_to_num(0.0)
                    outs["o"].append(p @ v)
                    outs["lse"].append(lse)
                    continue
                do, o, lse = s["do"][b, h].double(), s["o"][b, h].double(), s["lse"][b, h].double()
                p = torch.where(seen, torch.exp(x - lse[:, None]), torch.zeros_like(x))
                ds = p * (do @ v.T - (do * o).sum(-1, keepdim=True))
                dv += p.T @ do
                dk += (ds.T @ q) * scale
                outs["dq"].append((ds @ k) * scale)
                for i in range(c["buckets"]):
                    dtable[i, h] += ds[bucket == i].sum()
            outs["dk"].append(dk)
            outs["dv"].append(dv)

    def whole(name, heads, *tail):
        return torch.stack(outs[name]).view(c["batch"], heads, *tail)
    if c["op"] == "fwd":
        return [whole("o", c["heads"], c["sq"], c["d"]), whole("lse", c["heads"], c["sq"])]
    grads = [whole("dq", c["heads"], c["sq"], c["d"]), whole("dk", c["kv_heads"], c["sk"], c["d"]), whole("dv", c["kv_heads"], c["sk"], c["d"])]
    return grads + [dtable] if c["buckets"] else grads
