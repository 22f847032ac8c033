"""-m gpu: how the training operators deal their work out: attention calls of more work than the blocks take at once (a unit of work to each
group of warps, more than 32 sequences, chunks and prefixes that do not line up with blocks, sequences without rows in between), norm rows
that do not start on 16 bytes. Oracles and tolerances are those of test_train_attn_gpu.py and test_train_norm_gpu.py."""
import random

import pytest
import test_train_attn_gpu as attn
import test_train_norm_gpu as norm

pytestmark = pytest.mark.gpu


def lengths(n, most, seed, empty=0.0):
    r = random.Random(seed)
    return [0 if r.random() < empty else r.randint(1, most) for _ in range(n)] + [most]


def both(s):
    import torch
    attn.forward(s)
    attn.backward(s)
    attn.check(s)
    first = {n: s[n].clone() for n in ("out", "lse", "dq", "dk", "dv")}
    attn.forward(s)
    attn.backward(s)
    for n, t in first.items():
        assert torch.equal(t, s[n]), n


@pytest.mark.parametrize("chunk", [0, 200, 256])
@pytest.mark.parametrize("heads,kv,dim", [(14, 2, 64), (6, 2, 128), (5, 5, 48)])
def test_units_of_their_own(heads, kv, dim, chunk):
    """more sequences than lanes of a warp, and enough units for every group of every SM to have several"""
    lens = lengths(70, 600, 1 + chunk, empty=0.1)
    both(attn.make(lens, lens, heads, kv, dim, chunk=chunk, seed=chunk))


@pytest.mark.parametrize("heads,kv,dim", [(14, 2, 64), (4, 1, 128)])
@pytest.mark.parametrize("n,prefix,chunk", [(3, 300, 256), (3, 77, 128), (1, 1000, 384), (40, 150, 256), (2, 130, 5000), (5, 0, 0), (33, 64, 0), (3, 200, 130)])
def test_keys_before_the_queries(n, prefix, chunk, heads, kv, dim):
    lens = lengths(n - 1, 900, n + prefix, empty=0.1)
    r = random.Random(chunk)
    both(attn.make(lens, [x + r.randint(0, prefix) for x in lens], heads, kv, dim, chunk=chunk, seed=n))


def test_every_query_sees_every_key():
    lens = lengths(40, 500, 4, empty=0.2)
    both(attn.make(lens, lens[::-1], 14, 2, 64, causal=0, seed=4))


def test_bounds_longer_than_any_sequence():
    """max_q and max_k are bounds, not lengths"""
    for n in (6, 80):
        lens = lengths(n, 300, 5)
        for chunk in (0, 128, 1 << 30):
            both(attn.make(lens, lens, 4, 2, 64, chunk=chunk, seed=5, max_q=5000, max_k=2 ** 31 - 1))


@pytest.mark.parametrize("dtype", norm.TYPES)
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("rows,width", [(1, 1111), (1500, 263), (2500, 1111), (1203, 3585), (700, 4099), (640, 8191), (300, 16381)])
def test_norm_rows_that_start_anywhere(rows, width, kind, dtype):
    """many rows of odd widths, with and without what passes by, over their own inputs, twice the same bits"""
    import torch
    s = norm.make(rows, width, dtype, kind, seed=rows)
    y, mean, rstd = norm.forward(s, kind, dtype)
    norm.check_forward(s, kind, dtype, y, mean, rstd)
    for skip in (True, False):
        out = norm.backward(s, kind, dtype, mean, rstd, skip=skip)
        norm.check_backward(s, kind, dtype, mean, rstd, *out, skip=skip)
        again = norm.backward(s, kind, dtype, mean, rstd, skip=skip)
        assert all(torch.equal(a, b) for a, b in zip(out, again) if a is not None)
    for over in ("x", "dy", "skip"):
        mine = dict(s, **{over: s[over].clone()})
        dx, dw, db = norm.backward(mine, kind, dtype, mean, rstd, dx=mine[over])
        norm.check_backward(s, kind, dtype, mean, rstd, dx, dw, db)


@pytest.mark.parametrize("dtype", norm.TYPES)
def test_norm_weights_that_start_anywhere(dtype):
    """rows on 16 bytes, weight and bias not"""
    import torch
    for kind, rows, width in (("rms", 700, 896), ("layer", 700, 896), ("layer", 90, 6144), ("rms", 5000, 64)):
        s = norm.make(rows, width, dtype, kind, seed=7)
        for n in ("weight", "bias"):
            if s[n] is not None:
                moved = torch.empty(width + 1, dtype=s[n].dtype, device="cuda")[1:]
                s[n] = moved.copy_(s[n])
        y, mean, rstd = norm.forward(s, kind, dtype)
        norm.check_forward(s, kind, dtype, y, mean, rstd)
        norm.check_backward(s, kind, dtype, mean, rstd, *norm.backward(s, kind, dtype, mean, rstd))


@pytest.mark.parametrize("dtype", norm.TYPES)
def test_norm_leaves_what_is_around_odd_rows(dtype):
    """neither the bytes in front of the first row nor those behind the last one change, though rows share 16-byte units with them"""
    import torch
    t = getattr(torch, dtype)
    rows, width, front = 50, 1111, 16
    s = norm.make(rows, width, dtype, "rms", seed=8)
    flat = [torch.full((front + rows * width + 9,), 5.0, dtype=t, device="cuda") for _ in range(2)]
    y, dx = (f[front:front + rows * width].view(rows, width) for f in flat)
    _, mean, rstd = norm.forward(s, "rms", dtype, y=y)
    norm.backward(s, "rms", dtype, mean, rstd, dx=dx)
    norm.check_forward(s, "rms", dtype, y, mean, rstd)
    for f in flat:
        assert (f[:front] == 5).all() and (f[-9:] == 5).all()


def test_two_threads():
    """calls of two host threads on streams and workspaces of their own"""
    import threading

    import tffn
    import torch
    lens = [[300, 5, 129], [64, 700]]
    states = [attn.make(x, x, 6, 2, 64, seed=i) for i, x in enumerate(lens)]
    norms = [norm.make(400, 896, "bfloat16", "rms", seed=i) for i in range(2)]
    out, errors = [None, None], []
    torch.cuda.synchronize()

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                stream = torch.cuda.current_stream()
                ws = torch.empty(tffn.attention_backward_workspace(states[i]["shape"]), dtype=torch.uint8, device="cuda")
                for _ in range(20):
                    attn.forward(states[i], stream.cuda_stream)
                    attn.backward(states[i], stream.cuda_stream, ws)
                    out[i] = norm.forward(norms[i], "rms", "bfloat16", stream=stream.cuda_stream)
                stream.synchronize()
        except Exception as e:  # noqa: BLE001 - told to the test
            errors.append(e)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors
    for i in range(2):
        attn.check(states[i])
        norm.check_forward(norms[i], "rms", "bfloat16", *out[i])


@pytest.mark.parametrize("lens,heads,kv,dim", [([700] * 24, 14, 2, 64), ([1000, 400, 30], 14, 2, 64), ([90] * 9, 16, 2, 128), ([800, 769], 6, 3, 128)])
def test_parts_of_the_heads(lens, heads, kv, dim):
    """dK and dV of all heads of a kv head in one block, and of some of them in several, evenly dealt and not"""
    both(attn.make(lens, lens, heads, kv, dim, seed=20))
