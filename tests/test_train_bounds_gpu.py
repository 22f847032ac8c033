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
