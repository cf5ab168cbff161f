"""Attention over heads without a GPU: the bucket scheme's borders against whole-number arithmetic, and every refusal of
the C entry points and of the Python calls."""
import ctypes

import pytest


def _first_distances(m, e, max_distance):
    """Smallest distance of every bucket of one direction, by n^(m-e) >= e^(m-e-k) max_distance^k in Python's integers."""
    out, steps = list(range(e)), m - e
    for k in range(steps):
        lo, hi = e, max_distance
        while lo < hi:
            mid = (lo + hi) // 2
            lo, hi = (lo, mid) if mid ** steps >= e ** (steps - k) * max_distance ** k else (mid + 1, hi)
        out.append(lo)
    return out


@pytest.mark.parametrize("bidirectional", [True, False])
@pytest.mark.parametrize("buckets", [4, 6, 8, 32, 64, 128])
@pytest.mark.parametrize("max_distance", [64, 65, 128, 1000, 4096, 1 << 20])
def test_bucket_borders_are_exact(buckets, max_distance, bidirectional):
    from emmyptx import runtime
    m = buckets // 2 if bidirectional else buckets
    e = m // 2
    if max_distance <= e:
        with pytest.raises(runtime.KernelError, match="max_distance"):
            runtime.relative_runs(buckets, max_distance, bidirectional)
        return
    first = _first_distances(m, e, max_distance) + [1 << 40]
    runs = runtime.relative_runs(buckets, max_distance, bidirectional)
    assert [r[0] for r in runs[1:]] == sorted(set(r[0] for r in runs[1:]))

    def bucket(dist):
        n, side = (abs(dist), m if dist > 0 else 0) if bidirectional else (max(-dist, 0), 0)
        return side + max(k for k in range(m) if first[k] <= n)

    def by_runs(dist):
        return [b for i, (d0, b) in enumerate(runs) if i == 0 or d0 <= dist][-1]
    near = {s * (f + o) for f in first[:-1] for o in (-1, 0, 1) for s in (-1, 1)} | {0, 1 << 29, -(1 << 29)}
    for dist in near:
        assert by_runs(dist) == bucket(dist), dist


@pytest.mark.parametrize("args", [(1, 128, False), (2, 128, True), (5, 128, True), (130, 999, False), (0, 128, False), (32, 8, True), (32, 16, False),
                                  (8, (1 << 30) + 1, True), (-2, 8, False)])
def test_bucket_schemes_that_are_refused(args):
    from emmyptx import runtime
    with pytest.raises(runtime.KernelError):
        runtime.relative_runs(*args)


def _desc(runtime, backward=False, **change):
    d = runtime.HeadsDesc()
    d.dtype, d.flags, d.scale = runtime.BF16, 0, 0.125
    d.batch, d.heads, d.kv_heads, d.seq_q, d.seq_k, d.d = 2, 4, 2, 10, 20, 64
    for n, rows, heads in (("q", 10, 4), ("o", 10, 4), ("do", 10, 4), ("dq", 10, 4), ("k", 20, 2), ("v", 20, 2), ("dk", 20, 2), ("dv", 20, 2)):
        getattr(d, f"{n}_stride")[:] = (heads * rows * 64, rows * 64, 64)
    for n, v in change.items():
        if isinstance(v, tuple):
            getattr(d, n)[:len(v)] = v
        else:
            setattr(d, n, v)
    return d


BAD = [
    ({"dtype": 3}, -4, "dtype"), ({"flags": 4}, -1, "flags"), ({"batch": -1}, -2, "negative extent"), ({"seq_k": -5}, -2, "negative extent"),
    ({"d": 80}, -4, "head dim"), ({"d": 160}, -4, "head dim"), ({"d": 0}, -4, "head dim"), ({"kv_heads": 3}, -2, "multiple"), ({"kv_heads": 0}, -2, "multiple"),
    ({"heads": 0}, -2, "without query heads"), ({"scale": 0.0}, -1, "scale"), ({"scale": -1.0}, -1, "scale"), ({"scale": float("nan")}, -1, "scale"),
    ({"scale": float("inf")}, -1, "scale"), ({"seq_q": 1 << 30}, -2, "2^30"), ({"batch": 1 << 20, "heads": 1 << 12, "kv_heads": 1 << 12}, -2, "batch * heads"),
    ({"k_stride": (-64, 64, 64)}, -2, "negative stride"), ({"n_runs": 129}, -1, "runs"), ({"n_runs": -1}, -1, "runs"),
    ({"n_runs": 1, "buckets": 0}, -1, "buckets"), ({"n_runs": 1, "buckets": 129}, -1, "buckets"), ({"n_runs": 1, "buckets": 4, "bias_dtype": 3}, -4, "bias dtype"),
    ({"n_runs": 1, "buckets": 4, "run_bucket": (4,)}, -1, "bucket"), ({"n_runs": 3, "buckets": 4, "run_first": (0, 5, 5)}, -1, "rise"),
    ({"n_runs": 1, "buckets": 4, "bias_stride": (-1, 1)}, -2, "negative stride"),
]


@pytest.mark.parametrize("change,status,text", BAD)
def test_descriptions_that_are_refused(change, status, text, lib):
    from emmyptx import runtime
    p, ref = ctypes.c_void_p(4096), ctypes.byref                                  # never dereferenced
    d = _desc(runtime, **change)
    assert lib.emmyb200_attention_heads_fwd(ref(d), p, p, p, None, p, p, p, None, 0, None) == status
    assert text in lib.emmyb200_last_error().decode()
    assert lib.emmyb200_attention_heads_bwd(ref(d), p, p, p, p, p, p, None, p, p, p, p, None, None, 0, None) == status
    assert lib.emmyb200_attention_heads_workspace_bytes(ref(d), 0) == -1 and lib.emmyb200_attention_heads_workspace_bytes(ref(d), 1) == -1


def test_calls_that_are_refused(lib):
    from emmyptx import runtime
    p, ref = ctypes.c_void_p(4096), ctypes.byref
    fwd, bwd = lib.emmyb200_attention_heads_fwd, lib.emmyb200_attention_heads_bwd
    assert fwd(None, p, p, p, None, None, p, p, None, 0, None) == -1
    d = _desc(runtime)
    for hole in range(6):                                                         # Q K V O lse in turn
        if hole == 3:
            continue
        args = [p, p, p, None, p, p]
        args[hole] = None
        assert fwd(ref(d), args[0], args[1], args[2], None, None, args[4], args[5], None, 0, None) == -1
    assert fwd(ref(_desc(runtime, n_runs=1, buckets=4)), p, p, p, None, None, p, p, None, 0, None) == -1 and b"table" in lib.emmyb200_last_error()
    assert fwd(ref(_desc(runtime, o_stride=(640, 0, 64))), p, p, p, None, None, p, p, None, 0, None) == -2 and b"overlap" in lib.emmyb200_last_error()
    assert fwd(ref(_desc(runtime, o_stride=(2560, 640, 32))), p, p, p, None, None, p, p, None, 0, None) == -2
    assert bwd(ref(_desc(runtime, dk_stride=(640, 0, 64))), p, p, p, p, p, p, None, None, p, p, p, None, p, 1 << 20, None) == -2
    need = lib.emmyb200_attention_heads_workspace_bytes(ref(d), 1)
    assert need >= 2 * 2 * 4 * 10 * 4
    assert bwd(ref(d), p, p, p, p, p, p, None, None, p, p, p, None, p, need - 1, None) == -1 and b"workspace" in lib.emmyb200_last_error()
    assert bwd(ref(d), p, p, p, p, p, p, None, None, p, p, p, None, None, need, None) == -1
    assert bwd(ref(d), p, p, p, p, p, p, None, None, p, p, p, None, ctypes.c_void_p(4096 + 16), need, None) == -1
    assert bwd(ref(d), p, p, p, p, p, p, None, None, p, p, p, p, p, need, None) == -1 and b"without a table" in lib.emmyb200_last_error()
    for hole in (0, 1, 2, 3, 4, 5):
        args = [p] * 6
        args[hole] = None
        assert bwd(ref(d), *args, None, None, p, p, p, None, p, need, None) == -1
    for hole in (0, 1, 2):
        args = [p] * 3
        args[hole] = None
        assert bwd(ref(d), p, p, p, p, p, p, None, None, *args, None, p, need, None) == -1
    # nothing to do: accepted without buffers and without a device
    assert fwd(ref(_desc(runtime, batch=0)), None, None, None, None, None, None, None, None, 0, None) == 0
    assert fwd(ref(_desc(runtime, seq_q=0)), None, p, p, None, None, None, None, None, 0, None) == 0
    assert bwd(ref(_desc(runtime, batch=0)), None, None, None, None, None, None, None, None, None, None, None, None, None, 0, None) == 0
    assert lib.emmyb200_relative_runs(32, 128, 1, None, None) == -1


def test_python_calls_that_are_refused():
    import torch
    from emmyptx import runtime
    q, k = torch.zeros(2, 4, 10, 64, dtype=torch.bfloat16), torch.zeros(2, 2, 20, 64, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="no CPU path"):
        runtime.attention_heads(q, k, k)
    with pytest.raises(RuntimeError, match="no CPU path"):
        runtime.attention_heads_backward(q, q, k, k, q, torch.zeros(2, 4, 10))
    with pytest.raises(ValueError, match="q is"):
        runtime.attention_heads(q[0], k, k)
    with pytest.raises(ValueError, match="agree"):
        runtime.attention_heads(q, k, k[:, :1])
    with pytest.raises(ValueError, match="agree"):
        runtime.attention_heads(q, k[..., :32], k[..., :32])
    with pytest.raises(TypeError):
        runtime.attention_heads(q.double(), k.double(), k.double())
