"""-m gpu: what calls of the training operators share, or must not: the device's status word, workspaces, streams, threads."""
import pytest
import test_train_norm_gpu as norm

pytestmark = pytest.mark.gpu


def test_status_of_one_step():
    """a wait that runs out (on a barrier that nothing signals, with a short limit) is reported once: the steps behind it are their own"""
    import tffn
    tffn.train_status()
    tffn.op_train_wait_selftest()
    assert tffn.train_status() == 5
    assert tffn.train_status() == 0
    tffn.op_train_wait_selftest()
    tffn.op_train_wait_selftest()
    assert tffn.train_status() == 5
    s = norm.make(20, 896, "bfloat16", "rms")
    y, mean, rstd = norm.forward(s, "rms", "bfloat16")
    norm.check_backward(s, "rms", "bfloat16", mean, rstd, *norm.backward(s, "rms", "bfloat16", mean, rstd))
    assert tffn.train_status() == 0


def test_two_streams_with_workspaces_that_live():
    """attention in both directions on two streams at once, over and over: each has its own workspace for as long as either runs"""
    import test_train_attn_gpu as attn
    import tffn
    import torch
    lens = [900, 40, 1300]
    states = [attn.make(lens, lens, 14, 2, 64, seed=i) for i in (1, 2)]
    streams = [torch.cuda.Stream() for _ in states]
    spaces = [torch.full((tffn.attention_backward_workspace(s["shape"]),), 255, dtype=torch.uint8, device="cuda") for s in states]
    assert spaces[0].data_ptr() != spaces[1].data_ptr() and streams[0].cuda_stream != streams[1].cuda_stream
    torch.cuda.synchronize()
    for _ in range(15):
        for s, st, ws in zip(states, streams, spaces):
            attn.forward(s, st.cuda_stream)
            attn.backward(s, st.cuda_stream, ws)
    torch.cuda.synchronize()
    for s in states:
        attn.check(s)


def test_losses_and_norms_on_streams_of_their_own():
    """what a call overwrites is filled on the stream that the call is on"""
    import test_train_loss_gpu as loss
    import torch
    streams = [torch.cuda.Stream() for _ in range(2)]
    made = [(loss.make(40, 32768, "float32", seed=i), norm.make(700, 1111, "float32", "layer", seed=i)) for i in range(2)]
    torch.cuda.synchronize()
    got = [None, None]
    for turn in range(10):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                policy, lp = loss.policy(made[i][0], stream=st.cuda_stream), loss.logprob(made[i][0], stream=st.cuda_stream)
                y, mean, rstd = norm.forward(made[i][1], "layer", "float32", stream=st.cuda_stream)
                got[i] = policy, lp, (y, mean, rstd), norm.backward(made[i][1], "layer", "float32", mean, rstd, stream=st.cuda_stream)
    torch.cuda.synchronize()
    for (s, n), (policy, lp, stats, back) in zip(made, got):
        loss.check(s, policy)
        assert (lp - policy["lp"]).abs().max() <= 2 * loss.SUM
        norm.check_forward(n, "layer", "float32", *stats)
        norm.check_backward(n, "layer", "float32", *stats[1:], *back)


def test_losses_and_norm_gradients_from_two_threads():
    import threading

    import test_train_loss_gpu as loss
    import torch
    made = [(loss.make(30 + i, 60001, "bfloat16", seed=i), norm.make(300 + i, 3584, "bfloat16", "rms", seed=i)) for i in range(2)]
    torch.cuda.synchronize()
    got, errors = [None, None], []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                at = torch.cuda.current_stream().cuda_stream
                for _ in range(20):
                    policy, lp = loss.policy(made[i][0], stream=at), loss.logprob(made[i][0], stream=at)
                    y, mean, rstd = norm.forward(made[i][1], "rms", "bfloat16", stream=at)
                    got[i] = policy, lp, (y, mean, rstd), norm.backward(made[i][1], "rms", "bfloat16", mean, rstd, stream=at)
                torch.cuda.current_stream().synchronize()
        except Exception as e:  # noqa: BLE001 - told to the test
            errors.append(e)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors
    for (s, n), (policy, lp, stats, back) in zip(made, got):
        loss.check(s, policy)
        assert (lp - policy["lp"]).abs().max() <= 2 * loss.SUM
        norm.check_forward(n, "rms", "bfloat16", *stats)
        norm.check_backward(n, "rms", "bfloat16", *stats[1:], *back)


SUMS = [(5000, 64), (3001, 896), (1300, 3584), (4099, 1111), (131, 16384), (2000, 1001)]


@pytest.mark.parametrize("dtype", norm.TYPES)
@pytest.mark.parametrize("rows,width", SUMS)
def test_norm_sums_by_their_depth(rows, width, dtype):
    """dweight and dbias, as tight as the order of their additions allows: a block has at least rows / 140 rows less one, then come 4 warps of a block, 20 blocks of a
    run and 32 runs, each addition half a step of 2^-23; (x - mean) * rstd is two roundings more, and its product with dy is fused"""
    s = norm.make(rows, width, dtype, "layer", seed=9)
    y, mean, rstd = norm.forward(s, "layer", dtype)
    dx, dw, db = norm.backward(s, "layer", dtype, mean, rstd)
    dy, n = s["dy"].double(), (s["x"].double() - mean.double()[:, None]) * rstd.double()[:, None]
    terms = rows / 140 + 1 + 4 + 20 + 32
    assert ((dw.double() - (dy * n).sum(0)).abs() <= (terms + 2) * 2 ** -24 * (dy * n).abs().sum(0)).all()
    assert ((db.double() - dy.sum(0)).abs() <= terms * 2 ** -24 * dy.abs().sum(0)).all()
    assert (terms * 2 ** -24 * dy.abs().sum(0) < dy.abs().mean(0)).all()  # a row that were lost would show


@pytest.mark.parametrize("dtype", norm.TYPES)
@pytest.mark.parametrize("rows,width", SUMS)
def test_norm_sums_of_a_single_row(rows, width, dtype):
    """a gradient that only one row has: nothing else hides it if that row is lost, or counted twice"""
    import torch
    s = norm.make(rows, width, dtype, "layer", seed=10)
    y, mean, rstd = norm.forward(s, "layer", dtype)
    all_dy = s["dy"].clone()
    for r in sorted({0, 1, 3, 130, rows // 2, rows - 2, rows - 1} | {x for x in (147, 148, 443, 444, 591, 592, 593, 1183, 1184, 2367, 2368) if x < rows}):
        s["dy"].zero_()
        s["dy"][r] = all_dy[r]
        dx, dw, db = norm.backward(s, "layer", dtype, mean, rstd)
        want = all_dy[r].double() * (s["x"][r].double() - mean[r].double()) * rstd[r].double()
        assert torch.equal(db, all_dy[r].float()), r
        assert ((dw.double() - want).abs() <= 3 * 2 ** -24 * want.abs() + 1e-38).all(), r
