"""-m gpu: log-probabilities of sampled tokens and the clipped policy loss, against the formulas in 64 bits.

Tolerances, with arg = (x - max) log2 e <= 90 here: an exponential is off by the rounding of its argument, 2^-24 * 90 * ln 2 = 3.7e-6, plus
2^-22 of its own; a thread adds at most 152 000 / (128 * 1) = 1 200 terms where a row is one block of 128 threads (rows of 24 KB: 6 000 values,
47 terms) and at most 152 000 / 512 = 297 in larger blocks, 297 * 2^-24 = 1.8e-5 of the sum in the worst case. SUM = 2.5e-5 bounds the relative
error of the sum S of the other tokens' exponentials. lp = -log(1 + S / e) moves by at most SUM times 1 - p, plus one rounding to fp32.
The ratio moves by ratio * SUM, the gradient by (SUM of p) plus that of its slope, plus one rounding to the stored type."""
import math

import pytest

pytestmark = pytest.mark.gpu
SUM = 2.5e-5
TYPES = ["bfloat16", "float32"]


def ptr(t):
    return None if t is None else t.data_ptr()


def make(rows, vocab, dtype, seed=0, stride=None, offset=0, spread=3.0, boost=6.0):
    import torch
    g = torch.Generator("cuda").manual_seed(seed)
    t = getattr(torch, dtype)
    stride = stride or vocab
    flat = torch.full((rows * stride + offset,), float("nan"), dtype=t, device="cuda")
    x = flat[offset:].view(rows, stride)[:, :vocab]
    x.copy_(torch.randn((rows, vocab), generator=g, device="cuda") * spread)
    y = torch.randint(0, vocab, (rows,), generator=g, device="cuda", dtype=torch.int32)
    at = (torch.arange(rows, device="cuda"), y.long())
    x[at] = (x[at].float() + torch.randn(rows, generator=g, device="cuda") * 3 + boost).to(t)
    now = torch.log_softmax(x.double(), -1)[at].float()
    n = lambda std: torch.randn(rows, generator=g, device="cuda") * std  # noqa: E731
    return dict(x=x, y=y, old=now + n(0.2), ref=now + n(0.3), adv=n(1.0), weight=torch.rand(rows, generator=g, device="cuda") + 0.1, stride=stride, dtype=dtype)


def logprob(s, stream=0):
    import tffn
    import torch
    rows, vocab = s["x"].shape
    out = torch.full((rows,), float("nan"), device="cuda")
    tffn.token_logprobs(s["dtype"], ptr(s["x"]), ptr(s["y"]), rows, vocab, ptr(out), row_stride=s["stride"], stream=stream)
    return out


def policy(s, low=0.2, high=0.28, beta=0.1, grad=None, want=("loss", "row_loss", "lp", "kl", "grad"), stream=0):
    import tffn
    import torch
    rows, vocab = s["x"].shape
    out = {n: torch.full((rows,), float("nan"), device="cuda") for n in ("row_loss", "lp", "kl")} | {"loss": torch.full((1,), float("nan"), device="cuda")}
    if grad is None and "grad" in want:
        grad = torch.full((rows, s["stride"]), float("nan"), dtype=s["x"].dtype, device="cuda")[:, :vocab]
    out["grad"] = grad
    p = {n: ptr(out[n]) if n in want else None for n in out}
    tffn.policy_loss(s["dtype"], ptr(s["x"]), ptr(s["y"]), ptr(s["old"]), ptr(s["ref"]), ptr(s["adv"]), ptr(s["weight"]), rows, vocab, low, high, beta, p["loss"],
                     p["row_loss"], p["lp"], p["kl"], p["grad"], row_stride=s["stride"], stream=stream)
    return out


def truth(s, low=0.2, high=0.28, beta=0.1, x=None):
    """by autograd in 64 bits; rows of weight 0 and of targets outside are left out"""
    import torch
    x = (s["x"] if x is None else x).detach().double().clone().requires_grad_()
    rows, vocab = x.shape
    y = s["y"].long()
    w = torch.ones(rows, device="cuda", dtype=torch.float64) if s["weight"] is None else s["weight"].double()
    live = (w != 0) & (y >= 0) & (y < vocab)
    xs, ys = x[live], y[live]
    lp = xs.gather(1, ys[:, None])[:, 0] - torch.logsumexp(xs, -1)
    ratio = (lp - s["old"].double()[live]).exp()
    away = s["ref"].double()[live] - lp if s["ref"] is not None else lp * 0
    kl = torch.expm1(away) - away
    adv = s["adv"].double()[live]
    gain = torch.where(ratio * adv <= ratio.clamp(1 - low, 1 + high) * adv, ratio * adv, ratio.detach().clamp(1 - low, 1 + high) * adv)
    each = w[live] * (beta * kl - gain)
    grad = torch.autograd.grad(each.sum(), x)[0] if len(xs) else torch.zeros_like(x)
    full = lambda t: torch.zeros(rows, device="cuda", dtype=torch.float64).index_put((live.nonzero()[:, 0],), t.detach())  # noqa: E731
    # where the gradient is discontinuous both sides are right within the error of the ratio
    edge = torch.zeros(rows, dtype=torch.bool, device="cuda")
    edge[live] = (((ratio - (1 + high)).abs() < 1e-4) | ((ratio - (1 - low)).abs() < 1e-4)).detach()
    return dict(row_loss=full(each), lp=full(lp), kl=full(kl), ratio=full(ratio), away=full(away), grad=grad, loss=each.sum().detach(), live=live, edge=edge, w=w)


def check(s, got, low=0.2, high=0.28, beta=0.1, x=None):
    import torch
    t = truth(s, low, high, beta, x)
    step = torch.finfo(s["x"].dtype).eps / 2
    adv = s["adv"].double()
    lp_tol = SUM + 2 ** -24 * t["lp"].abs()
    assert ((got["lp"].double() - t["lp"]).abs() <= lp_tol).all()
    kl_tol = SUM * torch.expm1(t["away"]).abs() + SUM ** 2 + 2 ** -24 * t["kl"]
    assert ((got["kl"].double() - t["kl"]).abs() <= kl_tol + 1e-12).all()
    row_tol = t["w"].abs() * (beta * (kl_tol + 1e-12) + t["ratio"] * adv.abs() * SUM) + 2 ** -23 * t["row_loss"].abs() + 1e-12
    assert ((got["row_loss"].double() - t["row_loss"]).abs() <= row_tol).all()
    assert (got["loss"].double() - t["loss"]).abs() <= row_tol.sum() + 2 ** -24 * t["loss"].abs()
    slope_tol = t["w"].abs() * SUM * (beta * t["away"].exp() + t["ratio"] * adv.abs())
    p = torch.where(t["live"][:, None], torch.softmax((s["x"] if x is None else x).double(), -1), 0.0)  # rows that are not read may hold anything
    tol = (step + 3 * SUM) * t["grad"].abs() + slope_tol[:, None] * p.clamp_min(1e-30) + 1e-12
    at = (torch.arange(len(adv), device="cuda")[t["live"]], s["y"].long()[t["live"]])
    tol[at] += slope_tol[t["live"]]
    if s["dtype"] == "bfloat16":
        tol = tol + 1e-38  # flushed below the smallest normal number
    ok = ((got["grad"].double() - t["grad"]).abs() <= tol) | t["edge"][:, None]
    assert ok.all()
    assert not got["grad"][~t["live"]].any()


VOCABS = [1, 2, 3, 64, 100, 1000, 1024, 4099, 6144, 6151, 32768, 60001, 151936]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", VOCABS)
def test_losses(vocab, dtype):
    """one row, a few, and more than a cluster per SM; twice the same bits"""
    import torch
    for rows in (1, 7, 150):
        s = make(rows, vocab, dtype, seed=rows)
        lp = logprob(s)
        t = truth(s)
        assert ((lp.double() - t["lp"]).abs() <= SUM + 2 ** -24 * t["lp"].abs()).all()
        got = policy(s)
        check(s, got)
        again = policy(s)
        assert all(torch.equal(got[n], again[n]) for n in got)
        assert torch.equal(lp, logprob(s))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("stride,offset", [(1001, 0), (1008, 0), (1007, 3), (1016, 1)])
def test_rows_of_other_strides(stride, offset, dtype):
    """padded vocabularies and rows on any element; what lies between the rows stays"""
    import torch
    s = make(9, 1000, dtype, seed=2, stride=stride, offset=offset)
    assert ((logprob(s).double() - truth(s)["lp"]).abs() <= 2 * SUM).all()
    flat = torch.full((9 * stride + offset,), 7.0, dtype=s["x"].dtype, device="cuda")
    whole = flat[offset:].view(9, stride)
    got = policy(s, grad=whole[:, :1000])
    check(s, got)
    assert (whole[:, 1000:] == 7).all() and (flat[:offset] == 7).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [1000, 1001, 151936])
def test_gradient_over_the_logits(vocab, dtype):
    s = make(40, vocab, dtype, seed=4)
    kept = s["x"].clone()
    got = policy(s, grad=s["x"])
    check(s, got, x=kept)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [50, 1003, 60000])
def test_masks(vocab, dtype):
    """rows of weight 0 and targets outside the vocabulary are not read; masked vocabulary entries weigh nothing"""
    import torch
    s = make(12, vocab, dtype, seed=6)
    s["weight"][[0, 5, 11]] = 0.0
    s["x"][0] = float("nan")
    s["x"][5, :] = float("inf")
    s["y"][3], s["y"][4] = -100, vocab
    s["x"][3] = float("nan")
    lowest = torch.finfo(s["x"].dtype).min
    for r, low in ((1, -math.inf), (2, lowest), (6, -math.inf), (7, lowest)):
        keep = s["x"][r, s["y"][r]].clone()
        s["x"][r, ::2] = low
        s["x"][r, s["y"][r]] = keep
    for r, low in ((8, -math.inf), (9, lowest)):  # nothing left but the token
        keep = s["x"][r, s["y"][r]].clone()
        s["x"][r] = low
        s["x"][r, s["y"][r]] = keep
    live = [1, 2, 6, 7, 8, 9]
    at = (torch.tensor(live, device="cuda"), s["y"].long()[live])
    now = torch.log_softmax(s["x"][live].double(), -1)[torch.arange(len(live), device="cuda"), at[1]].float()
    s["old"][live], s["ref"][live] = now + 0.05, now - 0.1
    got = policy(s)
    check(s, got)
    for n in ("lp", "kl", "row_loss"):
        assert not got[n][[0, 3, 4, 5, 11]].any()
    assert got["lp"][8] == 0 and got["lp"][9] == 0 and not got["grad"][8].any()
    lp = logprob(s)
    assert lp[3] == 0 and lp[4] == 0 and (lp[live] - got["lp"][live]).abs().max() <= 2 * SUM
    # a token that is masked itself
    s["x"][1, s["y"][1]] = -math.inf
    assert logprob(s)[1] == -math.inf


def test_clip_branches_and_ties():
    """ratios on both sides of each edge with advantages of both signs, exactly on an edge, and an advantage of zero"""
    import torch
    s = make(10, 64, "float32", seed=8)
    now = torch.log_softmax(s["x"].double(), -1).gather(1, s["y"].long()[:, None])[:, 0]
    ratio = torch.tensor([1.0, 1.27, 1.29, 1.5, 0.81, 0.79, 0.5, 1.5, 0.5, 1.0], device="cuda", dtype=torch.float64)
    s["old"] = (now - ratio.log()).float()
    s["adv"] = torch.tensor([1.0, 1.0, 1.0, -1.0, 1.0, 1.0, -1.0, 0.0, 0.0, 0.0], device="cuda")
    got = policy(s, beta=0.0)
    check(s, got, beta=0.0)
    moves = got["grad"].abs().amax(1) > 0
    assert moves.tolist() == [True, True, False, True, True, True, False, False, False, False]
    # no clipping range at all: the tie at ratio 1 goes to the branch with a gradient
    got = policy(s, low=0.0, high=0.0, beta=0.3)
    check(s, got, low=0.0, high=0.0, beta=0.3)


def test_optional_outputs_and_inputs():
    import tffn
    import torch
    s = make(20, 5000, "float32", seed=9)
    full = policy(s)
    for want in (("lp",), ("grad",), ("row_loss", "loss"), ("kl", "row_loss")):
        got = policy(s, want=want)
        for n in want:
            assert torch.equal(got[n], full[n])
        for n in set(full) - set(want) - {"grad"}:
            assert got[n].isnan().all()
    s["ref"] = s["weight"] = None
    check(s, policy(s))
    loss = torch.ones(1, device="cuda")
    tffn.policy_loss("float32", None, None, None, None, None, None, 0, 10, 0.2, 0.2, 0.1, ptr(loss), None, None, None, None)
    assert loss.item() == 0
    tffn.token_logprobs("float32", None, None, 0, 10, None)


def test_gradient_by_differences():
    """loss along a random direction, stepped in the logits of the formula in 64 bits"""
    import torch
    s = make(6, 200, "float32", seed=10)
    s["adv"] = s["adv"].abs() + 0.1
    s["old"] = s["old"] * 0 + (truth(s)["lp"] - 0.02).float()  # ratios off the edges
    got = policy(s)
    way = torch.randn(s["x"].shape, device="cuda", dtype=torch.float64, generator=torch.Generator("cuda").manual_seed(1))
    h = 1e-5
    up, down = truth(s, x=s["x"].double() + h * way)["loss"], truth(s, x=s["x"].double() - h * way)["loss"]
    slope = (up - down) / (2 * h)
    assert abs((got["grad"].double() * way).sum() - slope) <= 1e-4 * (got["grad"].double() * way).abs().sum()


def test_offsets_past_32_bits():
    """the last row starts more than 2^31 elements behind the first"""
    import torch
    vocab, rows, stride = 1000, 18, 1 << 27
    flat = torch.empty((rows - 1) * stride + vocab, dtype=torch.bfloat16, device="cuda")
    x = torch.as_strided(flat, (rows, vocab), (stride, 1))
    s = make(rows, vocab, "bfloat16", seed=12)
    x.copy_(s["x"])
    s["x"], s["stride"] = x, stride
    assert ((logprob(s).double() - truth(s)["lp"]).abs() <= 2 * SUM).all()
    kept = x.clone()
    check(s, policy(s, grad=x), x=kept)


def test_streams_and_graph():
    import torch
    s = make(30, 32768, "float32", seed=13)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    got = policy(s, stream=st.cuda_stream)
    logprob(s, stream=st.cuda_stream)
    st.synchronize()
    check(s, got)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        got, lp = policy(s, stream=st.cuda_stream), logprob(s, stream=st.cuda_stream)
    for seed in (14, 15):
        new = make(30, 32768, "float32", seed=seed)
        for n in ("x", "y", "old", "ref", "adv", "weight"):
            s[n].copy_(new[n])
        graph.replay()
        torch.cuda.synchronize()
        check(s, got)
        assert (lp - got["lp"]).abs().max() <= 2 * SUM
