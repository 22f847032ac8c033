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
