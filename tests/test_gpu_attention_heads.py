"""Attention over heads (forward with log-sum-exp, backward, relative position bias) against the definition in float64.

Bounds, elementwise, with u half a step of the output type (bf16 2^-8, f16 2^-11, fp32 2^-24), g the relative error of a
probability in fp32 and |.| the same sums over absolute values:
    g:       a score is a d-term fp32 sum, off by at most (d + 8) 2^-24 scale |q|.|k| (+ as much for lse), and the exponential
             by 2^-20: g = 4 ((d + 8) 2^-24 max(scale |q|.|k| + |bias|) + 2^-20)
    o:       u |o| + (w + g) sum p |v|
    dv:      u |dv| + (w + g) sum p |do|
    dq, dk:  u |dq| + scale sum (w |ds| + g p (|do|.|v| + |do|.|o|)) |k|         (|q| for dk)
    dtable:  u |dtable| + g sum p (|do|.|v| + |do|.|o|)
    lse:     g
w is the rounding of a probability (or of its gradient) to 16 bits before the second product: 1.5 half steps where the tensor
cores run (bf16 values are cut after scaling by 1 + 2^-8 / ln 4, off by at most 2^-7 less that: 1.28 half steps), none in fp32 arithmetic. f16
probabilities below 2^-14 of the row's largest lose bits: 2^-24 sum |v| more in o. An f16 output below 2^-14 is off by up to
2^-25, half a step there. The backward keeps p 2^14 and ds 2^14 g in f16, g the power of two at or below 1 / B with B = max |dO row| max
|v row| of a key head; below 2^-14 those values are off by up to 2^-25 too, which is 2^-39 of p and 2^-39 / g <= 2^-38 B of ds: another
2^-39 sum |do| in dv, scale 2^-38 B sum |k| in dq (|q| in dk), over the pairs that are seen. (A score range of hundreds, as in
test_large_scores, has keys whose whole gradient is of that size.)
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _bucket(dist, buckets, max_distance, bidirectional):
    m = buckets // 2 if bidirectional else buckets
    e = m // 2
    side = (dist > 0).long() * m if bidirectional else torch.zeros_like(dist)
    n = dist.abs() if bidirectional else (-dist).clamp(min=0)
    far = e + torch.floor(torch.log(n.clamp(min=1).double() / e) / math.log(max_distance / e) * (m - e) + 1e-9).long()
    return side + torch.where(n < e, n, far.clamp(max=m - 1))


class Case:
    def __init__(self, cuda, dtype, b, h, hk, sq, sk, d, causal=False, align="start", lens=None, buckets=0, max_distance=128, bidirectional=True,
                 rows_first=False, seed=0, table_dtype=torch.float32, scale=None, spread=1.0):
        g = torch.Generator(device=cuda).manual_seed(seed)
        t = TYPES[dtype]

        def make(heads, rows, f=1.0):
            x = torch.randn(b, rows, heads, d, generator=g, device=cuda).mul_(f).to(t)
            return x.transpose(1, 2) if rows_first else x.transpose(1, 2).contiguous()
        self.q, self.k, self.v, self.do = make(h, sq, spread), make(hk, sk), make(hk, sk), make(h, sq)
        self.lens = None if lens is None else torch.tensor(lens, dtype=torch.int32, device=cuda)
        self.table = torch.randn(buckets, h, generator=g, device=cuda).to(table_dtype) if buckets else None
        self.scale = d ** -0.5 if scale is None else scale
        self.how = dict(scale=self.scale, causal=causal, align=align, key_lens=self.lens, bias_table=self.table, max_distance=max_distance,
                        bidirectional=bidirectional)
        self.causal, self.align, self.cores = causal, align, dtype == "f32" or d not in (64, 128)

    def reference(self, o=None, lse=None):
        """Everything in float64, with the sums of absolute values the bounds need. With o and lse: the backward from them."""
        q, k, v, do = (x.double() for x in (self.q, self.k, self.v, self.do))
        b, h, sq, d = q.shape
        hk, sk = k.shape[1], k.shape[2]
        r = {}
        kx, vx = k.repeat_interleave(h // hk, 1), v.repeat_interleave(h // hk, 1)
        n = torch.full((b,), sk, device=q.device) if self.lens is None else self.lens.long().clamp(0, sk)
        qp = torch.arange(sq, device=q.device)[None] + ((n - sq)[:, None] if self.align == "end" else 0 * n[:, None])
        kp = torch.arange(sk, device=q.device)
        seen = (kp < n[:, None])[:, None, :].expand(b, sq, sk)
        if self.causal:
            seen = seen & (kp <= qp[:, :, None])
        seen = seen[:, None].expand(b, h, sq, sk)
        # rows that are not seen may hold anything
        live = (kp < n[:, None])[:, None, :, None]
        kx, vx = torch.where(live, kx, 0.0), torch.where(live, vx, 0.0)
        s = q @ kx.transpose(-1, -2) * self.scale
        size = q.abs() @ kx.abs().transpose(-1, -2) * self.scale
        if self.table is not None:
            bucket = _bucket(kp - qp[:, :, None], self.table.shape[0], self.how["max_distance"], self.how["bidirectional"])     # [b, sq, sk]
            bias = self.table.double().t()[:, bucket].transpose(0, 1)
            s, size = s + bias, size + torch.where(bias > -1e30, bias.abs(), 0.0)
            seen = seen & (bias > -1e30)
        s = torch.where(seen, s, -math.inf)
        r["lse"] = torch.logsumexp(s, -1) if sk else torch.full((b, h, sq), -math.inf, device=q.device, dtype=torch.float64)
        top = float(size[seen].max()) if bool(seen.any()) else 0.0
        r["g"] = 4 * ((d + 8) * 2.0 ** -24 * top + 2.0 ** -20)
        p = torch.where(seen, torch.exp(s - (r["lse"] if lse is None else lse.double())[..., None]), 0.0)
        r["o"], r["o_abs"], r["v_sum"] = p @ vx, p @ vx.abs(), torch.where(seen, 1.0, 0.0).double() @ vx.abs()
        o = r["o"] if o is None else o.double()
        ds = p * (do @ vx.transpose(-1, -2) - (do * o).sum(-1, keepdim=True))
        ds_abs = p * (do.abs() @ vx.abs().transpose(-1, -2) + (do * o).abs().sum(-1, keepdim=True))

        def shared(x):
            return x.view(b, hk, h // hk, sk, d).sum(2)
        r["dq"], r["dk"], r["dv"] = ds @ kx * self.scale, shared(ds.transpose(-1, -2) @ q) * self.scale, shared(p.transpose(-1, -2) @ do)
        r["dv_abs"] = shared(p.transpose(-1, -2) @ do.abs())
        for w, x in (("ds", ds.abs()), ("fp", ds_abs)):
            r[f"dq_{w}"], r[f"dk_{w}"] = x @ kx.abs() * self.scale, shared(x.transpose(-1, -2) @ q.abs()) * self.scale
        once = torch.where(seen, 1.0, 0.0).double()
        big = do.norm(dim=-1).amax() * vx.norm(dim=-1).amax() if do.numel() and vx.numel() else 0.0
        r["dv_tiny"] = 2.0 ** -39 * shared(once.transpose(-1, -2) @ do.abs())
        r["dq_tiny"], r["dk_tiny"] = 2.0 ** -38 * big * self.scale * (once @ kx.abs()), 2.0 ** -38 * big * self.scale * shared(once.transpose(-1, -2) @ q.abs())
        if self.table is not None:
            flat = bucket[:, None].expand_as(ds).transpose(0, 1).reshape(h, -1)
            r["dtable"] = torch.zeros(h, self.table.shape[0], dtype=torch.float64, device=q.device).scatter_add_(1, flat, ds.transpose(0, 1).reshape(h, -1)).t()
            r["dtable_abs"] = torch.zeros(h, self.table.shape[0], dtype=torch.float64, device=q.device).scatter_add_(1, flat, ds_abs.transpose(0, 1).reshape(h, -1)).t()
        return r

    def check(self, what, got, want, bound):
        assert got.shape == want.shape
        if got.dtype == torch.float16:
            bound = bound + 2.0 ** -25
        got = got.double()
        assert torch.equal(torch.isfinite(got), torch.isfinite(want)), f"{what}: not finite where the definition is"
        both = torch.isfinite(want)
        assert torch.equal(got[~both], want[~both])
        if bool(both.any()):
            worst = ((got - want).abs() / (bound + 1e-30))[both].max().item() if not isinstance(bound, float) else (got - want).abs()[both].max().item() / bound
            assert worst <= 1.0, f"{what}: {worst:.2f}x its bound"

    def run(self):
        from emmyptx import runtime
        o, lse = runtime.attention_heads(self.q, self.k, self.v, **self.how)
        r = self.reference()
        u = torch.finfo(o.dtype).eps / 2
        w = 0.0 if self.cores else 1.5 * u
        tiny = 2.0 ** -24 if o.dtype == torch.float16 and not self.cores else 0.0
        self.check("lse", lse, r["lse"], r["g"])
        self.check("o", o, r["o"], u * r["o"].abs() + (w + r["g"]) * r["o_abs"] + tiny * r["v_sum"])
        r = self.reference(o, lse)
        grads = runtime.attention_heads_backward(self.do, self.q, self.k, self.v, o, lse, **self.how)
        torch.cuda.synchronize()
        assert runtime.device_status() == 0
        assert len(grads) == (3 if self.table is None else 4)
        f16 = 1.0 if tiny else 0.0
        self.check("dv", grads[2], r["dv"], u * r["dv"].abs() + (w + r["g"]) * r["dv_abs"] + f16 * r["dv_tiny"])
        self.check("dq", grads[0], r["dq"], u * r["dq"].abs() + w * r["dq_ds"] + r["g"] * r["dq_fp"] + f16 * r["dq_tiny"])
        self.check("dk", grads[1], r["dk"], u * r["dk"].abs() + w * r["dk_ds"] + r["g"] * r["dk_fp"] + f16 * r["dk_tiny"])
        if self.table is not None:
            ut = torch.finfo(self.table.dtype).eps / 2
            self.check("dtable", grads[3], r["dtable"], ut * r["dtable"].abs() + r["g"] * r["dtable_abs"])
        return o, lse, grads


SHAPES = [  # b, h, hk, sq, sk, d
    (1, 1, 1, 1, 1, 64), (1, 2, 1, 1, 77, 128), (2, 3, 3, 64, 64, 64), (2, 4, 2, 100, 130, 128), (1, 2, 2, 129, 257, 64), (1, 8, 2, 127, 128, 128),
    (3, 2, 1, 5, 300, 64), (2, 2, 2, 300, 5, 128), (1, 1, 1, 640, 700, 128), (2, 6, 2, 383, 383, 64), (1, 2, 2, 90, 110, 32), (2, 2, 1, 70, 130, 96),
]


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("shape", SHAPES)
def test_forward_and_backward(shape, causal, dtype, cuda):
    Case(cuda, dtype, *shape, causal=causal, seed=sum(shape)).run()


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("d", [64, 96, 128])
@pytest.mark.parametrize("causal,align", [(False, "start"), (True, "start"), (True, "end")])
def test_more_tiles_than_SMs(causal, align, d, dtype, cuda):
    """Several waves of blocks, and the CUDA-core kernels' larger tiles, with everything at once."""
    Case(cuda, dtype, 5, 16, 8, 150, 210, d, causal=causal, align=align, lens=[210, 100, 64, 1, 199], buckets=32, rows_first=True, seed=d).run()


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("bidirectional,causal", [(True, False), (False, True), (False, False), (True, True)])
@pytest.mark.parametrize("b,h,hk,sq,sk,d,buckets,max_distance", [
    (2, 4, 2, 100, 130, 64, 32, 128), (1, 2, 2, 300, 300, 128, 8, 64), (1, 2, 1, 513, 400, 64, 128, 200), (3, 2, 2, 1, 200, 128, 32, 128),
    (2, 2, 2, 260, 1, 64, 4, 3), (1, 1, 1, 900, 900, 64, 64, 700)])
def test_bias(b, h, hk, sq, sk, d, buckets, max_distance, bidirectional, causal, dtype, cuda):
    Case(cuda, dtype, b, h, hk, sq, sk, d, causal=causal, buckets=buckets, max_distance=max_distance, bidirectional=bidirectional, seed=sq + buckets).run()


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_bias_over_more_distances_than_the_table_holds(dtype, cuda):
    """Distances spread over more than 4096: the runs are searched instead of looked up."""
    Case(cuda, dtype, 1, 2, 1, 700, 650, 64, buckets=64, max_distance=9000, seed=31).run()
    Case(cuda, dtype, 2, 2, 2, 150, 5000, 128, causal=True, align="end", lens=[5000, 4700], buckets=32, max_distance=4500, bidirectional=False, seed=32).run()


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("heads,kv_heads,sq,buckets", [(4, 2, 1, 0), (4, 1, 3, 0), (2, 2, 2, 32)])
def test_tokens_against_long_caches(heads, kv_heads, sq, buckets, dtype, cuda):
    """Few rows against 200003 keys: the keys are split over many CTAs, some of which lie behind a short request's last key."""
    Case(cuda, dtype, 3, heads, kv_heads, sq, 200003, 64, causal=True, align="end", lens=[200003, 1, 130000], buckets=buckets, seed=33).run()


def test_runs_of_the_caller(cuda, lib):
    """The C entry points take any runs of distance: one run alone, and runs that name a bucket twice and leave one out."""
    import ctypes
    from emmyptx import runtime
    c = Case(cuda, "bf16", 2, 2, 2, 150, 200, 64, buckets=4, seed=34)
    lse = torch.empty(2, 2, 150, device=cuda)
    o, dq, dk, dv = (torch.empty_like(x) for x in (c.q, c.q, c.k, c.v))
    dtable = torch.empty_like(c.table)
    for runs in ([(0, 2)], [(0, 1), (-100, 3), (-5, 0), (0, 3), (7, 1)], [(0, 0), (-(1 << 30), 1), (1 << 30, 3)]):
        d = runtime.HeadsDesc()
        d.dtype, d.scale, d.bias_dtype, d.buckets, d.n_runs = runtime.BF16, c.scale, runtime.F32, 4, len(runs)
        d.batch, d.heads, d.kv_heads, d.seq_q, d.seq_k, d.d = 2, 2, 2, 150, 200, 64
        for n, x in (("q", c.q), ("k", c.k), ("v", c.v), ("o", o), ("do", c.do), ("dq", dq), ("dk", dk), ("dv", dv)):
            getattr(d, f"{n}_stride")[:] = x.stride()[:3]
        d.bias_stride[:] = c.table.stride()
        d.run_first[:len(runs)], d.run_bucket[:len(runs)] = [r[0] for r in runs], [r[1] for r in runs]
        ws = torch.empty(max(lib.emmyb200_attention_heads_workspace_bytes(ctypes.byref(d), 1), 256), dtype=torch.uint8, device=cuda)
        stream = torch.cuda.current_stream().cuda_stream
        assert lib.emmyb200_attention_heads_fwd(ctypes.byref(d), c.q.data_ptr(), c.k.data_ptr(), c.v.data_ptr(), None, c.table.data_ptr(), o.data_ptr(),
                                                lse.data_ptr(), ws.data_ptr(), ws.numel(), stream) == 0
        assert lib.emmyb200_attention_heads_bwd(ctypes.byref(d), c.do.data_ptr(), c.q.data_ptr(), c.k.data_ptr(), c.v.data_ptr(), o.data_ptr(), lse.data_ptr(),
                                                None, c.table.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), dtable.data_ptr(), ws.data_ptr(),
                                                ws.numel(), stream) == 0
        dist = torch.arange(200, device=cuda)[None] - torch.arange(150, device=cuda)[:, None]
        bucket = torch.full_like(dist, runs[0][1])
        for first, b in runs[1:]:
            bucket[dist >= first] = b
        q, k, v, table = (x.double() for x in (c.q, c.k, c.v, c.table))
        p = torch.softmax(q @ k.transpose(-1, -2) * c.scale + table.t()[:, bucket], -1)
        ds = p * (c.do.double() @ v.transpose(-1, -2) - (c.do.double() * o.double()).sum(-1, keepdim=True))
        want = torch.stack([ds[:, :, bucket == b].sum((0, 2)) for b in range(4)])
        # one rounding of o and of p, and of the result: 2^-8 each in the 2-norm; dtable is fp32 throughout, its sums cancel to some 1e-3 of their terms
        assert (o.double() - p @ v).norm() <= 3 * 2.0 ** -8 * (p @ v).norm()
        assert (dtable.double() - want).abs().max() <= 1e-5 * ds.abs().sum()
        assert all(torch.all(dtable[b] == 0) for b in range(4) if b not in [r[1] for r in runs])


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("align", ["start", "end"])
@pytest.mark.parametrize("buckets", [0, 32])
def test_key_counts(buckets, align, causal, dtype, cuda):
    """Key counts of zero, one, inside a tile, on a tile's border, all, and out of range (clamped); with the queries at the end
    of fewer keys than there are queries, the first rows see nothing."""
    c = Case(cuda, dtype, 7, 4, 2, 140, 300, 64, causal=causal, align=align, lens=[0, 1, 63, 128, 300, 1000, -4], buckets=buckets, seed=3)
    o, lse, grads = c.run()
    assert torch.all(o[0] == 0) and torch.all(lse[0] == -math.inf) and torch.all(grads[1][0] == 0) and torch.all(grads[0][6] == 0)
    assert torch.all(grads[1][2, :, 63:] == 0) and torch.all(grads[2][3, :, 128:] == 0)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_keys_behind_the_count_are_not_read(dtype, cuda):
    """Padding that holds NaN and infinities leaves no trace, gradients included."""
    from emmyptx import runtime
    lens = [37, 200, 129]
    c = Case(cuda, dtype, 3, 4, 2, 60, 200, 128, lens=lens, buckets=32, seed=9)
    o, lse = runtime.attention_heads(c.q, c.k, c.v, **c.how)
    grads = runtime.attention_heads_backward(c.do, c.q, c.k, c.v, o, lse, **c.how)
    for i, n in enumerate(lens):
        c.k[i, :, n:] = math.nan
        c.v[i, :, n:] = math.inf
    again, lse2 = runtime.attention_heads(c.q, c.k, c.v, **c.how)
    for x, y in zip((o, lse, *grads), (again, lse2, *runtime.attention_heads_backward(c.do, c.q, c.k, c.v, o, lse, **c.how))):
        assert torch.equal(x, y)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("value", [-math.inf, -1e38, "lowest"])
def test_bias_that_masks(value, dtype, cuda):
    """Table entries of -inf or a type's lowest value mask their pairs; where that leaves a row nothing, it gives zeros."""
    low = torch.finfo(torch.float32).min if value == "lowest" else value
    c = Case(cuda, dtype, 2, 2, 2, 150, 150, 64, buckets=8, max_distance=32, bidirectional=False, causal=True, seed=1)
    c.table[0, 0] = low                                    # the query's own position, one head
    c.table[:, 1] = low                                    # everything, the other head
    o, lse, grads = c.run()
    assert torch.all(o[:, 0, 0] == 0) and torch.all(lse[:, 0, 0] == -math.inf) and torch.all(o[:, 1] == 0) and torch.all(lse[:, 1] == -math.inf)
    assert torch.all(grads[0][:, 1] == 0) and torch.all(grads[1][:, 1] == 0) and torch.all(grads[3][:, 1] == 0) and torch.all(grads[3][0] == 0)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_table_types_and_strides(dtype, cuda):
    c = Case(cuda, dtype, 2, 4, 4, 150, 170, 64, buckets=32, table_dtype=TYPES[dtype], seed=5)
    assert c.run()[2][3].dtype == TYPES[dtype]
    wide = torch.randn(4, 64, device=cuda)
    c.table = c.how["bias_table"] = wide[:, ::2].t()        # [32 buckets, 4 heads] with strides (2, 64)
    c.run()


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("layout", ["rows_first", "packed", "shared", "odd"])
def test_strides(layout, dtype, cuda):
    """The layouts a projection leaves: rows before heads, q k v in one buffer, one key head expanded to all (stride 0), and
    row strides and starts that are not multiples of 16 bytes."""
    from emmyptx import runtime
    t = TYPES[dtype]
    c = Case(cuda, dtype, 2, 4, 4, 150, 150, 64, causal=True, seed=8, rows_first=layout == "rows_first")
    if layout == "packed":
        qkv = torch.randn(2, 150, 3, 4, 64, device=cuda).to(t)
        c.q, c.k, c.v = (qkv[:, :, i].transpose(1, 2) for i in range(3))
    elif layout == "shared":
        c.k, c.v = c.k[:, :1].expand(2, 4, 150, 64), c.v[:1].expand(2, 4, 150, 64)
    elif layout == "odd":
        wide = torch.randn(4, 2, 4, 150, 67, device=cuda).to(t)
        c.q, c.k, c.v, c.do = wide[0, ..., 3:], wide[1, ..., :64], wide[2, ..., 1:65], wide[3, ..., 2:66]
    o, lse, grads = c.run()
    dense = Case(cuda, dtype, 2, 4, 4, 150, 150, 64, causal=True, seed=8)
    dense.q, dense.k, dense.v, dense.do = (x.contiguous() for x in (c.q, c.k, c.v, c.do))
    o2, lse2, grads2 = dense.run()
    if layout != "odd":                                     # the same kernels
        for x, y in zip((o, lse, *grads), (o2, lse2, *grads2)):
            assert torch.equal(x, y)
    # outputs into strided buffers the caller owns; nothing between the rows is touched
    buf = torch.full((2, 150, 4, 72), 7.0, device=cuda, dtype=t)
    out = buf[..., :64].transpose(1, 2)
    runtime.attention_heads(c.q, c.k, c.v, out=out, **c.how)
    assert torch.equal(out, o) and torch.all(buf[..., 64:] == 7)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("b,h,hk,sq,sk", [(2, 4, 2, 0, 40), (2, 4, 2, 40, 0), (0, 4, 2, 40, 40), (2, 4, 2, 0, 0)])
def test_empty_extents(b, h, hk, sq, sk, dtype, cuda):
    from emmyptx import runtime
    t = TYPES[dtype]
    q, k = torch.randn(b, h, sq, 64, device=cuda).to(t), torch.randn(b, hk, sk, 64, device=cuda).to(t)
    table = torch.randn(8, h, device=cuda)
    how = dict(bias_table=table, max_distance=32)
    o, lse = runtime.attention_heads(q, k, k, **how)
    assert torch.all(o == 0) and torch.all(lse == -math.inf)
    fill = [torch.full_like(x, 3.0) for x in (q, k, k, table)]
    dq, dk, dv, dt = runtime.attention_heads_backward(q, q, k, k, o, lse, dq=fill[0], dk=fill[1], dv=fill[2], dtable=fill[3], **how)
    assert all(torch.all(x == 0) for x in (dq, dk, dv, dt))


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_large_scores(dtype, cuda):
    """Scores spread over hundreds: the running maximum moves often, most probabilities vanish."""
    Case(cuda, dtype, 2, 2, 2, 200, 700, 64, spread=6.0, scale=0.7, seed=4).run()
    c = Case(cuda, dtype, 1, 2, 2, 130, 900, 128, seed=6)
    c.k[:, :, 500:] *= 8
    c.run()


@pytest.mark.parametrize("size", [1e-4, 300.0])
def test_gradients_of_any_size_in_f16(size, cuda):
    """f16 keeps its bits when the incoming gradient is tiny (a loss without scaling) or large: dS is scaled by a power of two
    before it is rounded. The outputs themselves are kept in range by the test's own sizes."""
    c = Case(cuda, "f16", 2, 4, 2, 200, 200, 64, seed=2)
    c.do = (c.do.float() * size).half()
    c.v = c.v * (0.01 if size > 1 else 1)
    c.run()


def test_gradient_against_differences(cuda):
    """The f32 path's gradients against central differences of its own forward: for a random direction x, the change of
    sum(o * do) over a step of 2 h is 2 h (gradient . x) up to h^2 of the third derivative and the forward's fp32 error over h."""
    from emmyptx import runtime
    c = Case(cuda, "f32", 1, 2, 1, 20, 24, 32, causal=True, align="end", buckets=8, max_distance=16, seed=12)
    o, lse = runtime.attention_heads(c.q, c.k, c.v, **c.how)
    grads = runtime.attention_heads_backward(c.do, c.q, c.k, c.v, o, lse, **c.how)
    h = 2.0 ** -7
    gen = torch.Generator(device=cuda).manual_seed(1)
    for i, name in enumerate(("q", "k", "v", "table")):
        x = torch.randn(getattr(c, name).shape, generator=gen, device=cuda)
        x /= x.norm()
        ends = []
        for sign in (1, -1):
            args = {"q": c.q, "k": c.k, "v": c.v, "table": c.table, name: getattr(c, name) + sign * h * x}
            got, _ = runtime.attention_heads(args["q"], args["k"], args["v"], **{**c.how, "bias_table": args["table"]})
            ends.append((got.double() * c.do.double()).sum())
        slope, want = float(ends[0] - ends[1]) / (2 * h), float((grads[i].double() * x.double()).sum())
        # o is off by some 2^-21 of values of order one, 40 rows x 32 columns of random sign: about 2^-21 sqrt(1280) / h = 2e-3
        assert abs(slope - want) <= 5e-3 * max(1.0, abs(want)), (name, slope, want)


def test_training_step_matches_autograd_in_double(cuda):
    """Forward, then backward on what it left, as a training step runs them, against torch's own gradients of the formula."""
    from emmyptx import runtime
    c = Case(cuda, "bf16", 2, 4, 2, 333, 333, 128, causal=True, buckets=32, bidirectional=False, seed=21)
    o, lse = runtime.attention_heads(c.q, c.k, c.v, **c.how)
    grads = runtime.attention_heads_backward(c.do, c.q, c.k, c.v, o, lse, **c.how)
    q, k, v, table = (x.double().requires_grad_() for x in (c.q, c.k, c.v, c.table))
    pos = torch.arange(333, device=cuda)
    s = q @ k.repeat_interleave(2, 1).transpose(-1, -2) * c.scale + table.t()[:, _bucket(pos[None] - pos[:, None], 32, 128, False)]
    s = s.masked_fill(pos[None] > pos[:, None], -math.inf)
    (torch.softmax(s, -1) @ v.repeat_interleave(2, 1) * c.do.double()).sum().backward()
    # one rounding of o (2^-8, carried by D), one of p or ds, one of the result: 3 x 2^-8 in the 2-norm
    for name, got, want in zip(("dq", "dk", "dv", "dtable"), grads, (q.grad, k.grad, v.grad, table.grad)):
        off = (got.double() - want).norm() / want.norm()
        assert off <= 3 * 2.0 ** -8, (name, float(off))


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_results_repeat_bit_for_bit(dtype, cuda):
    from emmyptx import runtime
    c = Case(cuda, dtype, 3, 8, 2, 260, 390, 64, lens=[390, 17, 200], buckets=32, seed=5)

    def once():
        o, lse = runtime.attention_heads(c.q, c.k, c.v, **c.how)
        return (o, lse, *runtime.attention_heads_backward(c.do, c.q, c.k, c.v, o, lse, **c.how))
    first = once()
    for _ in range(3):
        assert all(torch.equal(x, y) for x, y in zip(first, once()))


def test_another_stream_and_the_current_one(cuda):
    """Work on a stream of its own behind a kernel that delays its input, and `stream=` named from the outside."""
    from emmyptx import runtime
    c = Case(cuda, "bf16", 2, 4, 2, 200, 200, 128, causal=True, buckets=32, seed=5)
    o, lse = runtime.attention_heads(c.q, c.k, c.v, **c.how)
    grads = runtime.attention_heads_backward(c.do, c.q, c.k, c.v, o, lse, **c.how)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        big = torch.randn(4096, 4096, device=cuda)
        q = (c.q + (big @ big).sum().to(torch.bfloat16) * 0)
        o2, lse2 = runtime.attention_heads(q, c.k, c.v, **c.how)
        g2 = runtime.attention_heads_backward(c.do, q, c.k, c.v, o2, lse2, **c.how)
    side.synchronize()
    o3, lse3 = runtime.attention_heads(c.q, c.k, c.v, stream=side, **c.how)
    g3 = runtime.attention_heads_backward(c.do, c.q, c.k, c.v, o3, lse3, stream=side, **c.how)
    side.synchronize()
    for x, y, z in zip((o, lse, *grads), (o2, lse2, *g2), (o3, lse3, *g3)):
        assert torch.equal(x, y) and torch.equal(x, z)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_captured_and_replayed(dtype, cuda):
    """A step captured into a graph and replayed on new inputs, with a second captured graph beside it."""
    from emmyptx import runtime
    cases = [Case(cuda, dtype, 2, 4, 2, 150, 150, 64, lens=[150, 90], buckets=32, seed=s) for s in (1, 2)]
    graphs, outs = [], []
    for c in cases:
        def step():
            o, lse = runtime.attention_heads(c.q, c.k, c.v, **c.how)
            return (o, lse, *runtime.attention_heads_backward(c.do, c.q, c.k, c.v, o, lse, **c.how))
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step())
        graphs.append(g)
    fresh = [Case(cuda, dtype, 2, 4, 2, 150, 150, 64, lens=[20, 150], buckets=32, seed=s) for s in (3, 4)]
    for c, f in zip(cases, fresh):
        for name in ("q", "k", "v", "do", "lens", "table"):
            getattr(c, name).copy_(getattr(f, name))
    for g in graphs:
        g.replay()
    torch.cuda.synchronize()
    for f, got in zip(fresh, outs):
        o, lse = runtime.attention_heads(f.q, f.k, f.v, **f.how)
        want = (o, lse, *runtime.attention_heads_backward(f.do, f.q, f.k, f.v, o, lse, **f.how))
        assert all(torch.equal(x, y) for x, y in zip(got, want))


def test_two_streams_at_once(cuda):
    """The same step on two streams without any order between them, several times over."""
    from emmyptx import runtime
    c = Case(cuda, "f16", 2, 8, 2, 500, 500, 64, causal=True, buckets=32, seed=41)

    def step():
        o, lse = runtime.attention_heads(c.q, c.k, c.v, **c.how)
        return (o, lse, *runtime.attention_heads_backward(c.do, c.q, c.k, c.v, o, lse, **c.how))
    want = step()
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], []
    for _ in range(4):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(step())
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for g in got for x, y in zip(want, g))


def test_offsets_beyond_32_bits(cuda):
    """A cache whose batch entries and heads lie more than 2^31 elements apart."""
    from emmyptx import runtime
    c = Case(cuda, "bf16", 2, 2, 2, 3, 300, 64, causal=True, align="end", seed=14)
    o, lse = runtime.attention_heads(c.q, c.k, c.v, **c.how)
    grads = runtime.attention_heads_backward(c.do, c.q, c.k, c.v, o, lse, **c.how)
    pool = torch.empty(2 ** 31 + 2 ** 20, dtype=torch.bfloat16, device=cuda)
    far = [torch.as_strided(pool, (2, 2, 300, 64), (2 ** 31, 300 * 64, 64, 1), at) for at in (0, 2 ** 19)]
    far[0].copy_(c.k)
    far[1].copy_(c.v)
    o2, lse2 = runtime.attention_heads(c.q, far[0], far[1], **c.how)
    g2 = runtime.attention_heads_backward(c.do, c.q, far[0], far[1], o2, lse2, **c.how)
    for x, y in zip((o, lse, *grads), (o2, lse2, *g2)):
        assert torch.equal(x, y)


def test_workspaces_and_outputs_of_the_caller(cuda):
    from emmyptx import runtime
    c = Case(cuda, "bf16", 2, 4, 2, 150, 170, 64, buckets=32, seed=5)
    o, lse = runtime.attention_heads(c.q, c.k, c.v, **c.how)
    grads = runtime.attention_heads_backward(c.do, c.q, c.k, c.v, o, lse, **c.how)
    ws = torch.full((1 << 24,), 0xFF, dtype=torch.uint8, device=cuda)              # NaN patterns
    o2, lse2 = runtime.attention_heads(c.q, c.k, c.v, workspace=ws, out=torch.full_like(c.q, math.nan), lse=torch.full_like(lse, math.nan), **c.how)
    g2 = runtime.attention_heads_backward(c.do, c.q, c.k, c.v, o2, lse2, workspace=ws, dq=torch.full_like(c.q, math.nan), dk=torch.full_like(c.k, math.nan),
                                          dv=torch.full_like(c.v, math.nan), dtable=torch.full_like(c.table, math.nan), **c.how)
    for x, y in zip((o, lse, *grads), (o2, lse2, *g2)):
        assert torch.equal(x, y)


def test_python_refusals(cuda):
    from emmyptx import runtime
    q, k = torch.zeros(2, 4, 10, 64, dtype=torch.bfloat16, device=cuda), torch.zeros(2, 2, 20, 64, dtype=torch.bfloat16, device=cuda)
    table = torch.zeros(32, 4, device=cuda)
    lse = torch.zeros(2, 4, 10, device=cuda)
    lens = torch.zeros(2, dtype=torch.int32, device=cuda)
    fwd, bwd = runtime.attention_heads, runtime.attention_heads_backward
    for bad in (dict(key_lens=lens.long()), dict(key_lens=lens[:1]), dict(key_lens=lens.cpu()), dict(bias_table=table[:, :3]), dict(bias_table=table.long()),
                dict(bias_table=table.cpu()), dict(align="left"), dict(out=q.float()), dict(out=q[:, :2]), dict(lse=lse.double()), dict(lse=lse[:, :, :5])):
        with pytest.raises(ValueError):
            fwd(q, k, k, **bad)
    with pytest.raises(ValueError, match="contiguous"):
        fwd(q.transpose(-1, -2).contiguous().transpose(-1, -2), k, k)
    with pytest.raises(ValueError):
        fwd(q, k.half(), k.half())
    with pytest.raises(runtime.KernelError, match="multiple"):
        fwd(q[:, :3], k, k)
    with pytest.raises(runtime.KernelError, match="scale"):
        fwd(q, k, k, scale=0.0)
    with pytest.raises(runtime.KernelError, match="overlap"):
        fwd(q, k, k, out=q[:, :1].expand(2, 4, 10, 64))
    with pytest.raises(runtime.KernelError, match="max_distance"):
        fwd(q, k, k, bias_table=table, max_distance=4)
    with pytest.raises(runtime.KernelError, match="head dim"):
        fwd(q[..., :48], k[..., :48], k[..., :48])
    for bad in (dict(dq=q[:, :2]), dict(dk=q), dict(dtable=table), dict(workspace=torch.empty(8, dtype=torch.uint8, device=cuda))):
        with pytest.raises(ValueError):
            bwd(q, q, k, k, q, lse, **bad)
    with pytest.raises(ValueError, match="lse"):
        bwd(q, q, k, k, q, lse.half())
    with pytest.raises(ValueError):
        bwd(q[:, :, :5], q, k, k, q, lse)
