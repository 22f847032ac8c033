"""CPU: what the training operators refuse, before they look for a device. Pointers are numbers that nothing follows."""
import pytest

import tffn

P = 1 << 20  # an aligned address
ODD = P + 2


def refused(code, fn, *args, **kw):
    with pytest.raises(tffn.TffnError) as e:
        fn(*args, **kw)
    assert e.value.code == code, e.value
    return e.value.msg


def no_device(fn, *args, **kw):
    """the arguments are fine: only the device is missing"""
    if tffn.device_count() > 0:
        pytest.skip("a GPU is present")
    refused(-5, fn, *args, **kw)


def norm(kind="rms", dtype="bfloat16", x=P, weight=P, bias=None, rows=3, width=64, eps=1e-6, y=P, mean=None, rstd=P):
    tffn.norm_forward(kind, dtype, x, weight, bias, rows, width, eps, y, mean, rstd)


def norm_back(kind="rms", dtype="bfloat16", dy=P, x=P, weight=P, mean=None, rstd=P, skip=None, rows=3, width=64, dx=P, dweight=P, dbias=None, workspace=P,
              size=1 << 20):
    tffn.norm_backward(kind, dtype, dy, x, weight, mean, rstd, skip, rows, width, dx, dweight, dbias, workspace, size)


@pytest.mark.parametrize("change", [dict(kind="group"), dict(dtype="float16"), dict(x=None), dict(weight=None), dict(y=None), dict(rows=-1), dict(width=0),
                                    dict(eps=-1.0), dict(eps=float("nan")), dict(bias=P), dict(mean=P), dict(kind="layer"), dict(x=P + 1),
                                    dict(dtype="float32", x=ODD), dict(dtype="float32", y=ODD)])
def test_norm_forward_refuses(change):
    refused(-1, norm, **change)


def test_norm_width_limit():
    assert "16384" in refused(-7, norm, width=16385)
    no_device(norm, width=16384)
    no_device(norm, kind="layer", bias=P, mean=P)
    no_device(norm, x=ODD)  # bf16 rows at any element
    refused(-1, tffn.norm_backward_workspace, -1, 64)
    refused(-1, tffn.norm_backward_workspace, 3, 0)
    assert tffn.norm_backward_workspace(0, 64) == 0
    assert tffn.norm_backward_workspace(10, 64) == 10 * 64 * 2 * 4


@pytest.mark.parametrize("change", [dict(dy=None), dict(dx=None), dict(rstd=None), dict(mean=P), dict(dbias=P), dict(kind="layer"), dict(workspace=None),
                                    dict(workspace=P + 4), dict(size=3 * 64 * 8 - 1), dict(skip=P + 1), dict(dtype="float32", skip=ODD)])
def test_norm_backward_refuses(change):
    refused(-1, norm_back, **change)


def test_norm_backward_needs_no_workspace_without_sums():
    no_device(norm_back, dweight=None, workspace=None, size=0)
    no_device(norm_back, size=3 * 64 * 8)


def shape(**change):
    s = dict(n_seqs=2, heads=4, kv_heads=2, head_dim=64, rows_q=10, rows_k=12, max_q=6, max_k=8, q_stride=256, k_stride=128, v_stride=128, out_stride=256, causal=1,
             chunk=0, scale=0.125)
    s.update(change)
    return tffn.AttentionShape(**s)


def attn(cu_q=P, cu_k=P, q=P, k=P, v=P, out=P, lse=P, **change):
    tffn.attention_forward(shape(**change), cu_q, cu_k, q, k, v, out, lse)


def attn_back(cu_q=P, cu_k=P, q=P, k=P, v=P, out=P, lse=P, d_out=P, dq=P, dk=P, dv=P, workspace=P, size=1 << 24, **change):
    tffn.attention_backward(shape(**change), cu_q, cu_k, q, k, v, out, lse, d_out, dq, dk, dv, workspace, size)


BAD_SHAPES = [dict(n_seqs=-1), dict(heads=0), dict(kv_heads=0), dict(heads=3), dict(max_q=-1), dict(max_k=-1), dict(rows_q=-1), dict(scale=0.0), dict(scale=-1.0),
              dict(scale=float("inf")), dict(scale=float("nan")), dict(chunk=-1), dict(chunk=5, causal=0), dict(q_stride=248), dict(k_stride=120), dict(v_stride=127),
              dict(out_stride=260)]


@pytest.mark.parametrize("change", BAD_SHAPES + [dict(cu_q=None), dict(cu_k=None), dict(q=None), dict(k=None), dict(v=None), dict(out=None), dict(q=P + 8), dict(k=P + 2),
                                                 dict(v=P + 4), dict(out=P + 8)])
def test_attention_forward_refuses(change):
    refused(-1, attn, **change)


@pytest.mark.parametrize("change", BAD_SHAPES + [dict(lse=None), dict(d_out=None), dict(dq=None), dict(dk=None), dict(dv=None), dict(dq=P + 8), dict(workspace=None),
                                                 dict(workspace=P + 8), dict(size=16)])
def test_attention_backward_refuses(change):
    refused(-1, attn_back, **change)


@pytest.mark.parametrize("change", [dict(head_dim=60, q_stride=256), dict(head_dim=136, q_stride=544, out_stride=544, k_stride=272, v_stride=272), dict(rows_q=1 << 31)])
def test_attention_unsupported(change):
    refused(-7, attn, **change)
    refused(-7, tffn.attention_backward_workspace, shape(**change))


def test_attention_arguments_that_are_fine():
    no_device(attn)
    no_device(attn, lse=None)
    no_device(attn, rows_q=0, q=None, out=None)
    no_device(attn, rows_k=0, k=None, v=None)
    no_device(attn, chunk=7, q_stride=512)
    no_device(attn_back)
    size = tffn.attention_backward_workspace(shape())
    assert size >= 4 * 10 * 4
    no_device(attn_back, size=size)


def logprob(dtype="float32", logits=P, targets=P, rows=3, vocab=100, out=P, row_stride=0):
    tffn.token_logprobs(dtype, logits, targets, rows, vocab, out, row_stride=row_stride)


def policy(dtype="float32", logits=P, targets=P, old=P, ref=P, advantage=P, weight=P, rows=3, vocab=100, low=0.2, high=0.2, kl_coef=0.1, loss=P, row_loss=P, lp=P, kl=P,
           grad=P, row_stride=0):
    tffn.policy_loss(dtype, logits, targets, old, ref, advantage, weight, rows, vocab, low, high, kl_coef, loss, row_loss, lp, kl, grad, row_stride=row_stride)


@pytest.mark.parametrize("change", [dict(dtype="int8"), dict(logits=None), dict(targets=None), dict(rows=-1), dict(vocab=0), dict(row_stride=99), dict(row_stride=-1),
                                    dict(logits=ODD)])
def test_losses_refuse(change):
    refused(-1, logprob, **change)
    refused(-1, policy, **change)


@pytest.mark.parametrize("change", [dict(old=None), dict(advantage=None), dict(row_loss=None), dict(low=-0.1), dict(low=1.1), dict(high=-0.1),
                                    dict(high=float("inf")), dict(kl_coef=float("nan")), dict(grad=ODD)])
def test_policy_loss_refuses(change):
    refused(-1, policy, **change)


def test_losses_limits():
    refused(-1, logprob, out=None)
    refused(-7, policy, vocab=500000)
    refused(-7, policy, dtype="bfloat16", vocab=1000000)
    no_device(policy, vocab=400000)
    no_device(logprob, vocab=1000000)
    no_device(policy, ref=None, weight=None, loss=None, row_loss=None, lp=None, kl=None, grad=None)
    no_device(tffn.train_status)
