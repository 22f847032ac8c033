"""-m gpu: rows of logits at the ends of the range for the losses: vocabularies that are masked as a whole, finite logits of any size. Oracle and
tolerances are those of test_train_loss_gpu.py, which hold here: an exponential's argument is (x - max) log2 e, and where that is far below zero
the exponential is zero on both sides."""
import math

import pytest
import test_train_loss_gpu as loss

pytestmark = pytest.mark.gpu


def plain(vocab, dtype, rows, seed=0, **kw):
    """without a reference: what a KL term of such rows is belongs to another test"""
    s = loss.make(rows, vocab, dtype, seed=seed, **kw)
    s["ref"] = None
    return s


def shifted(s):
    """the same rows with their maximum at 0: x[y] - logsumexp(x) of the oracle has steps of 2^75 at 3.4e38, in 64 bits"""
    x = s["x"].double()
    return x - x.amax(-1, keepdim=True)


def settle(s, rows):
    """old log-probabilities next to the present ones, where those are ordinary numbers"""
    import torch
    now = loss.truth(s, x=shifted(s))["lp"]
    s["old"][rows] = torch.where(now[rows] > -1e4, now[rows] + 0.05, torch.zeros_like(now[rows])).float()


def compare(s):
    import torch
    x = s["x"].double()
    want = torch.log_softmax(x, -1).gather(1, s["y"].long()[:, None])[:, 0]
    lp = loss.logprob(s)
    near = (lp.double() - want).abs() <= loss.SUM + 2 ** -24 * want.abs()
    assert (near | ((want < torch.finfo(torch.float32).min) & (lp == -math.inf))).all(), (lp, want)
    loss.check(s, loss.policy(s), x=shifted(s))


@pytest.mark.parametrize("dtype", loss.TYPES)
@pytest.mark.parametrize("vocab,stride,offset", [(1, None, 0), (50, None, 0), (1003, None, 0), (1000, 1008, 0), (60000, None, 0), (60001, 60001, 1), (151936, None, 0)])
def test_whole_rows_at_one_value(vocab, stride, offset, dtype):
    """every logit at the type's lowest value, the token's included: -log V by the formula; so at any other value"""
    import torch
    t = getattr(torch, dtype)
    values = [torch.finfo(t).min, torch.finfo(t).max, -1e30, -2e30, 1e30, 3e9, -7e12, 0.0]
    s = plain(vocab, dtype, len(values) + 2, seed=1, stride=stride, offset=offset)
    for r, v in enumerate(values):
        s["x"][r] = v
    settle(s, list(range(len(values))))
    compare(s)
    lp = loss.logprob(s)[:len(values)]
    assert ((lp.double() + math.log(vocab)).abs() <= loss.SUM + 2 ** -24 * math.log(vocab)).all()
    assert loss.policy(s)["grad"].isfinite().all()


@pytest.mark.parametrize("dtype", loss.TYPES)
@pytest.mark.parametrize("vocab", [2, 64, 1003, 60000])
def test_finite_logits_of_any_size(vocab, dtype):
    """masked as a whole beside -inf; the token or one other entry alone above the rest; differences that no fp32 number holds"""
    import torch
    t = getattr(torch, dtype)
    low, top = torch.finfo(t).min, torch.finfo(t).max
    s = plain(vocab, dtype, 12, seed=2)
    x, y = s["x"], s["y"].long()
    other = (y + 1) % vocab
    x[0] = -math.inf                       # nothing but the token, and that masked by the lowest value
    x[0, y[0]] = low
    x[1] = -math.inf                       # two entries at the lowest value
    x[1, y[1]], x[1, other[1]] = low, low
    x[2] = low                             # the token half as low
    x[2, y[2]] = low / 2
    x[3] = low                             # another entry half as low
    x[3, other[3]] = low / 2
    x[4] = low                             # another entry is an ordinary number
    x[4, other[4]] = 1.5
    x[5, y[5]] = low                       # only the token is masked
    x[6], x[6, y[6]] = low, top            # both ends
    x[7], x[7, other[7]] = low, top        # a log-probability below all fp32 numbers: left to the other operator
    s["weight"][7] = 0.0
    x[8], x[8, y[8]], x[8, other[8]] = -top / 2, top, top
    x[9] = x[9] * 1e30                     # any order of size
    x[10] = x[10] - 2e9
    settle(s, list(range(11)))
    compare(s)
    assert loss.policy(s)["grad"].isfinite().all()


def test_masked_rows_over_their_own_logits_and_of_weight_zero():
    import torch
    for dtype in loss.TYPES:
        s = plain(1000, dtype, 6, seed=3)
        low = torch.finfo(s["x"].dtype).min
        s["x"][[0, 2, 5]] = low
        s["weight"][2] = 0.0
        settle(s, [0, 5])
        kept = shifted(s)
        loss.check(s, loss.policy(s, grad=s["x"]), x=kept)


@pytest.mark.parametrize("dtype", loss.TYPES)
@pytest.mark.parametrize("vocab", [100, 60000])
def test_a_divergence_that_is_only_watched(vocab, dtype):
    """kl_coef 0: the same bits as without a reference, also where the token is masked, or so far below its reference that the divergence is infinite"""
    import torch
    s = loss.make(8, vocab, dtype, seed=4)
    at = torch.arange(8, device="cuda"), s["y"].long()
    for r, v in ((1, -math.inf), (3, torch.finfo(s["x"].dtype).min), (4, -1000.0)):
        s["x"][r, s["y"][r]] = v
    lp = torch.log_softmax(s["x"].double(), -1)[at]
    s["ref"][[1, 3, 4]] = -2.0
    s["old"][[1, 3, 4]] = -3.0
    got = loss.policy(s, beta=0.0)
    without = loss.policy(dict(s, ref=None), beta=0.0)
    for n in ("loss", "row_loss", "lp", "grad"):
        assert got[n].isfinite().all() or n == "lp", n
        assert torch.equal(got[n], without[n]), n
    assert got["lp"][1] == -math.inf and got["kl"][[1, 3, 4]].eq(math.inf).all()
    keep = [0, 2, 5, 6, 7]
    away = s["ref"].double() - lp
    kl = torch.expm1(away) - away
    assert ((got["kl"].double() - kl)[keep].abs() <= (loss.SUM * torch.expm1(away).abs() + loss.SUM ** 2 + 2 ** -24 * kl)[keep] + 1e-12).all()


def test_no_advantage_and_a_ratio_out_of_range():
    """an advantage of 0 gains nothing, also where the ratio is beyond all numbers"""
    import torch
    s = plain(200, "float32", 5, seed=5)
    s["adv"] = torch.tensor([0.0, 0.0, 1.0, 0.0, -0.0], device="cuda")
    s["old"][[0, 1, 2, 4]] = torch.tensor([-2000.0, -math.inf, -2000.0, -900.0], device="cuda")
    got = loss.policy(s)
    assert not got["row_loss"][[0, 1, 3, 4]].any() and not got["grad"].any()
    want = -s["weight"][2].double() * (1 + 0.28)  # clipped
    assert abs(got["row_loss"][2].double() - want) <= 2 ** -23 * abs(want)
    assert abs(got["loss"][0].double() - want) <= 2 ** -23 * abs(want)
