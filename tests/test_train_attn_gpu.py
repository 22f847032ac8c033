"""-m gpu: attention of packed training sequences, forward and backward, against the formulas in 64 bits.

Tolerances are computed per element from the roundings that the kernels make, each at most half a step (2^-8 of a bf16 value):
  O    P enters its product as bf16: 2^-8 sum P |V|; O itself 2^-8 |O|
  dV   2^-8 sum P |dO|, and 2^-8 |dV|
  dS   = P (dP - D): rounded to bf16, 2^-8 |dS|, about the D of the stored O, which is off by at most
       sum |dO| (2^-8 sum P |V| + 2^-8 |O|): what it leaves out of dS enters as P times that
  dQ, dK  sums of (dS's errors) |K| or |Q| times the scale, and 2^-8 of the result
What is fp32 (S, exponentials, sums) adds FP = 2^-10 of the same magnitudes: |S| < 64 here, so that rounding it costs an exponential at most
64 * 2^-18 (64 products and a sum of 64 terms, each a rounding of 2^-24: 2^6 * 2^-24 of the sum of magnitudes, below 64 times 4)."""
import math

import pytest

pytestmark = pytest.mark.gpu
HALF, FP = 2.0 ** -8, 2.0 ** -10


def ptr(t):
    return None if t is None else t.data_ptr()


def offsets(lens):
    import torch
    return torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32, device="cuda")


def make(lens_q, lens_k, heads, kv, dim, causal=1, chunk=0, seed=0, tail=3, fused=False, scale=None, std=1.0, max_q=None, max_k=None):
    """rows behind the last sequence hold NaN in the inputs, and 5 in the outputs"""
    import tffn
    import torch
    g = torch.Generator("cuda").manual_seed(seed)
    nq, nk = sum(lens_q) + tail, sum(lens_k) + tail

    def rows(n, used, h, buf=None, std=std):
        t = torch.empty(n, h, dim, dtype=torch.bfloat16, device="cuda") if buf is None else buf
        t.copy_(torch.randn((n, h, dim), generator=g, device="cuda") * std)
        t[used:] = float("nan")
        return t
    if fused:  # parts of one projection's output (as many queries as keys)
        whole = torch.empty(nq, (heads + 2 * kv) * dim, dtype=torch.bfloat16, device="cuda")
        parts = whole.split([heads * dim, kv * dim, kv * dim], 1)
        q, k, v = (rows(nq, sum(lens_q), h, p.unflatten(1, (h, dim))) for p, h in zip(parts, (heads, kv, kv)))
        grads = torch.full_like(whole, 5.0)
        dq, dk, dv = (p.unflatten(1, (h, dim)) for p, h in zip(grads.split([heads * dim, kv * dim, kv * dim], 1), (heads, kv, kv)))
    else:
        q, k, v = rows(nq, sum(lens_q), heads), rows(nk, sum(lens_k), kv), rows(nk, sum(lens_k), kv)
        dq, dk, dv = (torch.full_like(t, 5.0) for t in (q, k, v))
    dout = rows(nq, sum(lens_q), heads)
    shape = tffn.AttentionShape(n_seqs=len(lens_q), heads=heads, kv_heads=kv, head_dim=dim, rows_q=nq, rows_k=nk, max_q=max_q or max(lens_q, default=0),
                                max_k=max_k or max(lens_k, default=0), causal=causal, chunk=chunk, q_stride=q.stride(0), k_stride=k.stride(0), v_stride=v.stride(0),
                                out_stride=heads * dim, scale=scale or dim ** -0.5)
    return dict(q=q, k=k, v=v, dout=dout, out=torch.full((nq, heads, dim), 5.0, dtype=torch.bfloat16, device="cuda"), lse=torch.full((heads, nq), 5.0, device="cuda"), dq=dq,
                dk=dk, dv=dv, cu_q=offsets(lens_q), cu_k=offsets(lens_k), lens=(lens_q, lens_k), shape=shape)


def forward(s, stream=0):
    import tffn
    tffn.attention_forward(s["shape"], *(ptr(s[n]) for n in ("cu_q", "cu_k", "q", "k", "v", "out", "lse")), stream=stream)


def backward(s, stream=0, workspace=None):
    import tffn
    import torch
    size = tffn.attention_backward_workspace(s["shape"])
    ws = torch.empty(size, dtype=torch.uint8, device="cuda") if workspace is None else workspace
    tffn.attention_backward(s["shape"], *(ptr(s[n]) for n in ("cu_q", "cu_k", "q", "k", "v", "out", "lse", "dout", "dq", "dk", "dv")), ptr(ws), size, stream=stream)


def mask(s, nq, nk):
    import torch
    if not s["shape"].causal:
        return torch.ones(nq, nk, dtype=torch.bool, device="cuda")
    at, key = torch.arange(nk - nq, nk, device="cuda")[:, None], torch.arange(nk, device="cuda")
    see = key <= at
    if s["shape"].chunk:
        see &= key >= at.clamp_min(0) // s["shape"].chunk * s["shape"].chunk
    return see


def near(got, want, tol):
    d = (got.double() - want).abs()
    bad = ~(d <= tol + 1e-30)
    assert not bad.any(), (int(bad.sum()), float(d[bad].max()), float((d / (tol + 1e-30))[bad].max()))


def check(s, grads=True):
    import torch
    q, k, v, do = (s[n].double() for n in ("q", "k", "v", "dout"))
    scale, (lens_q, lens_k) = s["shape"].scale, s["lens"]
    G = q.shape[1] // k.shape[1]
    q0 = k0 = 0
    for nq, nk in zip(lens_q, lens_k):
        rq, rk = slice(q0, q0 + nq), slice(k0, k0 + nk)
        q0, k0 = q0 + nq, k0 + nk
        see = mask(s, nq, nk)
        some = see.any(-1) if nk else torch.zeros(nq, dtype=torch.bool, device="cuda")
        for g in range(k.shape[1]):
            Q, dO = q[rq, g * G:(g + 1) * G].transpose(0, 1), do[rq, g * G:(g + 1) * G].transpose(0, 1)
            K, V = k[rk, g], v[rk, g]
            S = torch.where(see, Q @ K.T * scale, -math.inf)
            lse = torch.logsumexp(S, -1) if nk else torch.full((G, nq), -math.inf, device="cuda", dtype=torch.float64)
            P = torch.where(see, torch.exp(S - lse.nan_to_num(neginf=0.0)[..., None]), 0.0)
            O, around = P @ V, P @ V.abs()
            near(s["out"][rq, g * G:(g + 1) * G].transpose(0, 1), O, HALF * O.abs() + (HALF + FP) * around)
            got = s["lse"][g * G:(g + 1) * G, rq].double()
            assert (got[:, ~some] == -math.inf).all()
            near(got[:, some], lse[:, some], 1e-4 + 2 ** -23 * lse[:, some].abs())
            if not grads:
                continue
            dP, D = dO @ V.T, (dO * O).sum(-1, keepdim=True)
            dS = P * (dP - D)
            d_tol = (dO.abs() * (HALF * O.abs() + (HALF + FP) * around)).sum(-1, keepdim=True)
            s_tol = HALF * dS.abs() + P * d_tol + FP * P * (dO.abs() @ V.abs().T + (dO * O).abs().sum(-1, keepdim=True))
            dQ = scale * (dS @ K)
            near(s["dq"][rq, g * G:(g + 1) * G].transpose(0, 1), dQ, HALF * dQ.abs() + scale * (s_tol @ K.abs()))
            dK, dV = scale * (dS.transpose(1, 2) @ Q).sum(0), (P.transpose(1, 2) @ dO).sum(0)
            near(s["dk"][rk, g], dK, HALF * dK.abs() + scale * (s_tol.transpose(1, 2) @ Q.abs()).sum(0))
            near(s["dv"][rk, g], dV, HALF * dV.abs() + ((HALF + FP) * P.transpose(1, 2) @ dO.abs()).sum(0))
    # rows behind the last sequence
    assert (s["out"][q0:] == 5).all() and (s["lse"][:, q0:] == 5).all()
    assert (s["dq"][q0:] == 5).all() and (s["dk"][k0:] == 5).all() and (s["dv"][k0:] == 5).all()
    import tffn
    assert tffn.train_status() == 0


HEADS = [(1, 1, 64), (14, 2, 64), (2, 2, 128), (7, 1, 128), (3, 1, 40), (2, 1, 8), (4, 2, 96)]
LENS = [[1], [5, 1, 2], [63, 64, 65], [127, 128, 129], [0, 7, 0, 300, 0], [257, 31]]


@pytest.mark.parametrize("heads,kv,dim", HEADS)
@pytest.mark.parametrize("lens", LENS)
def test_causal(lens, heads, kv, dim):
    s = make(lens, lens, heads, kv, dim, seed=len(lens))
    forward(s)
    check_forward_only(s)
    backward(s)
    check(s)


def check_forward_only(s):
    check(s, grads=False)


@pytest.mark.parametrize("heads,kv,dim", [(14, 2, 64), (3, 1, 128)])
@pytest.mark.parametrize("lens_q,lens_k", [([1, 1], [300, 64]), ([5, 130], [200, 131]), ([64, 3], [64, 400]),        # keys before the queries
                                           ([200, 9, 70], [60, 9, 0]), ([129], [1]), ([3, 5], [0, 0])])                # queries that see nothing
def test_queries_and_keys_of_other_lengths(lens_q, lens_k, heads, kv, dim):
    for causal in (1, 0):
        s = make(lens_q, lens_k, heads, kv, dim, causal=causal, seed=5)
        forward(s)
        backward(s)
        check(s)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("chunk", [1, 7, 64, 100, 128, 1000])
def test_chunks(chunk, dim):
    for lens_q, lens_k in (([300, 65], [300, 65]), ([150, 40], [333, 90]), ([90], [50])):
        s = make(lens_q, lens_k, 4, 2, dim, chunk=chunk, seed=chunk)
        forward(s)
        backward(s)
        check(s)


@pytest.mark.parametrize("dim", [32, 64, 128])
def test_parts_of_one_projection(dim):
    s = make([100, 41], [100, 41], 6, 2, dim, fused=True, seed=8)
    forward(s)
    backward(s)
    check(s)


def test_many_sequences_and_one_long_one():
    """blocks that add up all query heads of a kv head, and blocks that share them; twice the same bits"""
    import torch
    for lens, heads, kv, dim in (([3] * 400, 4, 2, 64), ([17] * 310, 6, 1, 128), ([2100], 3, 1, 64), ([1500, 600], 2, 1, 128)):
        s = make(lens, lens, heads, kv, dim, seed=9)
        forward(s)
        backward(s)
        check(s)
        first = {n: s[n].clone() for n in ("out", "lse", "dq", "dk", "dv")}
        forward(s)
        backward(s)
        for n, t in first.items():
            assert torch.equal(t, s[n]), n


def test_sharp_and_flat_scores():
    """the running maximum moves often, or never; scores beyond what exp holds"""
    import torch
    for std, scale in ((6.0, None), (0.05, None), (1.0, 3.0)):
        s = make([400], [400], 2, 1, 64, seed=10, std=std, scale=scale)
        if std == 6.0:
            s["dout"].mul_(0.1)
            s["k"][:400] = (s["k"][:400].float() * 0.2).to(torch.bfloat16)  # |S| stays below 64
            s["q"][:400] *= torch.linspace(0.02, 1, 400, device="cuda")[:, None, None].to(torch.bfloat16)
        if scale:
            s["q"][:400] *= 0.25
        forward(s)
        backward(s)
        check(s)


def test_gradient_by_differences():
    """the three gradients along random directions, against differences of the formula in 64 bits"""
    import torch
    lens, heads, dim = [70], 2, 64
    s = make(lens, lens, heads, 1, dim, seed=11, tail=0)
    forward(s)
    backward(s)
    g = torch.Generator("cuda").manual_seed(3)

    def loss(q, k, v):
        S = torch.einsum("qhd,kd->hqk", q, k[:, 0]) * s["shape"].scale
        P = torch.softmax(S.masked_fill(~mask(s, 70, 70), -math.inf), -1)
        return (torch.einsum("hqk,kd->qhd", P, v[:, 0]) * s["dout"].double()).sum()
    args = [s[n].double() for n in "qkv"]
    for i, n in enumerate(("dq", "dk", "dv")):
        way = torch.randn(args[i].shape, generator=g, device="cuda", dtype=torch.float64)
        h = 1e-5
        up, down = ([a + (sign * h * way if j == i else 0.0) for j, a in enumerate(args)] for sign in (1, -1))
        slope = (loss(*up) - loss(*down)) / (2 * h)
        size = (s[n].double() * way).abs().sum()
        assert abs((s[n].double() * way).sum() - slope) <= 4 * HALF * size  # roundings of P, dS, D and the result, all of one sign


def test_offsets_past_32_bits():
    """rows that start more than 2^31 elements behind the first"""
    import tffn
    import torch
    stride, lens = 1 << 22, [400, 200]
    s = make(lens, lens, 2, 1, 64, seed=12, tail=0)
    for n in ("q", "k", "v", "dq", "dk", "dv"):
        flat = torch.empty((600 - 1) * stride + 128, dtype=torch.bfloat16, device="cuda")
        t = torch.as_strided(flat, s[n].shape, (stride, 64, 1))
        t.copy_(s[n])
        s[n] = t
    for n in ("q_stride", "k_stride", "v_stride"):
        setattr(s["shape"], n, stride)
    forward(s)
    backward(s)
    check(s)
    assert tffn.train_status() == 0


def test_offsets_outside_the_buffers_stay_inside():
    """offsets that go past the buffers or back are cut to what there is; a bound that is too small leaves the rest"""
    import tffn
    import torch
    s = make([60, 40], [60, 40], 2, 1, 64, seed=13, tail=2)
    for t in ("q", "k", "v", "dout"):
        s[t][100:] = 0
    s["cu_q"].copy_(torch.tensor([-5, 60, 5000], dtype=torch.int32))
    s["cu_k"].copy_(torch.tensor([60, 10, 2000000000], dtype=torch.int32))
    forward(s)
    backward(s)
    torch.cuda.synchronize()
    assert tffn.train_status() == 0


def test_without_lse():
    import tffn
    import torch
    s = make([90, 3], [90, 3], 4, 2, 64, seed=14)
    forward(s)
    kept = s["out"].clone()
    s["out"].fill_(5)
    tffn.attention_forward(s["shape"], *(ptr(s[n]) for n in ("cu_q", "cu_k", "q", "k", "v", "out")), None)
    assert torch.equal(kept, s["out"])


def test_streams_graphs_and_workspaces():
    """two streams at once with workspaces of their own; a captured pair replayed on new inputs and other lengths"""
    import tffn
    import torch
    a, b = (make([200, 90], [200, 90], 4, 2, 64, seed=i) for i in (15, 16))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for s, st in zip((a, b), streams):
        forward(s, st.cuda_stream)
        backward(s, st.cuda_stream, torch.empty(tffn.attention_backward_workspace(s["shape"]), dtype=torch.uint8, device="cuda"))
    torch.cuda.synchronize()
    check(a)
    check(b)
    st, graph = streams[0], torch.cuda.CUDAGraph()
    ws = torch.empty(tffn.attention_backward_workspace(a["shape"]), dtype=torch.uint8, device="cuda")
    with torch.cuda.graph(graph, stream=st):
        forward(a, st.cuda_stream)
        backward(a, st.cuda_stream, ws)
    for seed, lens in ((17, [200, 90]), (18, [150, 140])):
        new = make(lens, lens, 4, 2, 64, seed=seed)
        for n in ("q", "k", "v", "dout", "cu_q"):
            a[n].copy_(new[n])
        a["cu_k"].copy_(new["cu_k"])
        a["lens"] = (lens, lens)
        graph.replay()
        torch.cuda.synchronize()
        check(a)
