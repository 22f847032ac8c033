"""-m gpu: bounds and offsets of the training attention that are far from its sequences. Oracles and tolerances are those of test_train_attn_gpu.py."""
import pytest
import test_train_attn_gpu as attn

pytestmark = pytest.mark.gpu
RESULTS = ("out", "lse", "dq", "dk", "dv")


def both(s):
    attn.forward(s)
    attn.backward(s)
    return {n: s[n].clone() for n in RESULTS}


@pytest.mark.parametrize("heads,kv,dim,rows,n", [(64, 1, 8, 1 << 18, 8192), (14, 2, 64, 1 << 17, 3000), (4, 4, 128, 1 << 16, 70)])
def test_bounds_as_long_as_the_buffers(heads, kv, dim, rows, n):
    """a few sequences among many empty ones: 2^30 blocks by the bounds and more, a few hundred by the rows; the same bits as under tight bounds"""
    import torch
    lens = [0] * n
    for i in range(20):
        lens[i * (n // 20) + i % 7] = 1 + 37 * i
    s = attn.make(lens, lens, heads, kv, dim, seed=n, tail=rows - sum(lens))
    tight = both(s)
    attn.check(s)
    for name in RESULTS:
        s[name].fill_(5)
    s["shape"].max_q = s["shape"].max_k = rows
    loose = both(s)
    for name, t in tight.items():
        assert torch.equal(t, loose[name]), name


@pytest.mark.parametrize("dim", [64, 128])
def test_offsets_that_go_back_and_forth(dim):
    """not ascending: rows that many sequences claim. No result, but nothing outside of the buffers is touched, and every call ends"""
    import tffn
    import torch
    s = attn.make([64] * 40, [64] * 40, 6, 2, dim, seed=3, tail=0, max_q=5000, max_k=5000)
    rows = 64 * 40
    for turn in ([0, rows] * 20 + [0], [rows, 0] * 20 + [rows], [0] * 40 + [rows], [-7] + [2 ** 31 - 1] * 40):
        for name in ("cu_q", "cu_k"):
            s[name].copy_(torch.tensor(turn, dtype=torch.int32))
        both(s)
        torch.cuda.synchronize()
        assert tffn.train_status() == 0


MANY = [([5] * 200 + [1500] + [17] * 300, 0, 0), ([1] * 1500 + [130, 0, 900], 100, 256), ([0, 40] * 100 + [1100] + [64] * 37, 30, 200),
        ([2] * 4000 + [700], 0, 128)]


@pytest.mark.parametrize("heads,kv,dim", [(14, 2, 64), (4, 1, 128)])
@pytest.mark.parametrize("lens,prefix,chunk", MANY)
def test_many_short_sequences_and_a_long_one(lens, prefix, chunk, heads, kv, dim):
    """each 32 sequences in an order of their own; twice the same bits"""
    import torch
    s = attn.make(lens, [n + (i * 7 % (prefix + 1)) for i, n in enumerate(lens)], heads, kv, dim, chunk=chunk, seed=len(lens))
    first = both(s)
    long = max(range(len(lens)), key=lambda i: lens[i])
    near = [i for i in range(len(lens)) if lens[i] and (abs(i - long) < 20 or i < 20 or i % 97 == 0)]
    check_some(s, near)
    for name, t in both(s).items():
        assert torch.equal(first[name], t), name


def check_some(s, chosen):
    """the oracle on some sequences, moved together"""
    import torch
    lens_q, lens_k = s["lens"]
    at_q, at_k = [0], [0]
    for a, b in zip(lens_q, lens_k):
        at_q.append(at_q[-1] + a)
        at_k.append(at_k[-1] + b)
    rows_q = torch.cat([torch.arange(at_q[i], at_q[i + 1], device="cuda") for i in chosen])
    rows_k = torch.cat([torch.arange(at_k[i], at_k[i + 1], device="cuda") for i in chosen])
    part = {n: s[n][rows_q] for n in ("q", "dout", "out", "dq")} | {n: s[n][rows_k] for n in ("k", "v", "dk", "dv")}
    attn.check(dict(part, lse=s["lse"][:, rows_q], lens=([lens_q[i] for i in chosen], [lens_k[i] for i in chosen]), shape=s["shape"]))
    assert (s["out"][at_q[-1]:] == 5).all() and (s["dq"][at_q[-1]:] == 5).all() and (s["dk"][at_k[-1]:] == 5).all()
    for n in ("out", "dq", "dk", "dv"):  # no row of any sequence is left as it was
        rows = at_q[-1] if n in ("out", "dq") else at_k[-1]
        assert not (s[n][:rows] == 5).flatten(1).all(1).any(), n


def test_time_goes_by_the_rows():
    """one long sequence among thousands of short ones takes about what the same rows take in a few: not sequences times longest (ten times as long)"""
    import tffn
    import torch

    def time(lens):
        s = attn.make(lens, lens, 2, 1, 64, seed=1)
        ws = torch.empty(tffn.attention_backward_workspace(s["shape"]), dtype=torch.uint8, device="cuda")
        stream, best = torch.cuda.current_stream().cuda_stream, 1e9
        for _ in range(4):
            a, b = torch.cuda.Event(True), torch.cuda.Event(True)
            a.record()
            attn.forward(s, stream)
            attn.backward(s, stream, ws)
            b.record()
            torch.cuda.synchronize()
            best = min(best, a.elapsed_time(b))
        assert tffn.train_status() == 0
        return best
    few, many = time([2000] * 32 + [8192]), time([16] * 2000 + [8192] + [16] * 2000)
    assert many < 3 * few, (few, many)
