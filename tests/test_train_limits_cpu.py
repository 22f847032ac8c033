"""CPU: limits of the training operators. What a call cannot do is refused before anything is enqueued, and nothing that it can do is."""
import pytest
import tffn
import test_train_cpu as cpu

BIG = dict(heads=28, kv_heads=4, q_stride=28 * 64, k_stride=256, v_stride=256, out_stride=28 * 64)


@pytest.mark.parametrize("n,rows,bound", [(10000, 1 << 20, 1 << 20), (8192, 1 << 20, 2 ** 31 - 1), (1 << 20, 1 << 20, 1), (1, (1 << 31) - 5000, (1 << 31) - 5000)])
def test_loose_bounds_are_no_work(n, rows, bound):
    """what the packed rows hold counts, not sequences times the longest that one may be"""
    s = dict(BIG, n_seqs=n, rows_q=rows, rows_k=rows, max_q=bound, max_k=bound)
    assert tffn.attention_backward_workspace(cpu.shape(**s)) > 0
    cpu.no_device(cpu.attn, **s)
    cpu.no_device(cpu.attn_back, size=1 << 50, **s)


def test_units_that_cannot_be_counted():
    """2^30 blocks of queries, or of keys, are refused by both directions before a launch"""
    many = dict(n_seqs=1 << 26, rows_q=1 << 26, rows_k=1 << 26, heads=16, kv_heads=16, head_dim=8, q_stride=128, k_stride=128, v_stride=128, out_stride=128,
                max_q=1 << 20, max_k=1 << 20)
    assert "2^30" in cpu.refused(-7, cpu.attn, **many)
    cpu.refused(-7, cpu.attn_back, size=1 << 50, **many)
    cpu.refused(-7, tffn.attention_backward_workspace, cpu.shape(**many))
    keys = dict(many, rows_q=100, max_q=100)
    cpu.refused(-7, cpu.attn_back, size=1 << 50, **keys)
    cpu.refused(-7, tffn.attention_backward_workspace, cpu.shape(**keys))
    cpu.no_device(cpu.attn, **keys)  # the forward call deals out blocks of queries only
    cpu.no_device(cpu.attn_back, size=1 << 50, **dict(many, n_seqs=1 << 20))


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_vocabularies_next_to_2_31(dtype):
    """sizes that a sum of a few more overflows: too long for the policy loss, and for log-probabilities where an index past the row does not fit"""
    for vocab in (2 ** 31 - 1, 2 ** 31 - 6, 2 ** 31 - 4000):
        cpu.refused(-7, cpu.policy, dtype=dtype, vocab=vocab)
        cpu.refused(-7, cpu.logprob, dtype=dtype, vocab=vocab)
    cpu.refused(-7, cpu.policy, dtype=dtype, vocab=2 ** 31 - 5000)
    cpu.no_device(cpu.logprob, dtype=dtype, vocab=2 ** 31 - 5000)


@pytest.mark.parametrize("call,names", [
    (cpu.norm, ("rstd",)), (lambda **kw: cpu.norm(kind="layer", bias=cpu.P, **kw), ("mean",)), (cpu.norm_back, ("rstd", "dweight")),
    (lambda **kw: cpu.norm_back(**{**dict(kind="layer", mean=cpu.P, dbias=cpu.P), **kw}), ("mean", "dbias")), (cpu.attn, ("cu_q", "cu_k", "lse")),
    (cpu.attn_back, ("cu_q", "cu_k", "lse")), (cpu.logprob, ("targets", "out")),
    (cpu.policy, ("targets", "old", "ref", "advantage", "weight", "loss", "row_loss", "lp", "kl"))])
def test_statistics_offsets_and_rows_start_on_their_elements(call, names):
    """fp32 and int32 tensors half an element off: a fault on the device"""
    for name in names:
        assert "aligned" in cpu.refused(-1, call, **{name: cpu.ODD}), name
    cpu.no_device(call, **{names[0]: cpu.P + 4})


def test_sequences_next_to_2_31():
    """the walk over the sequences steps 32 ahead: a count next to 2^31 would never be passed"""
    for n in (2 ** 31 - 1, 2 ** 31 - 40):
        cpu.refused(-7, cpu.attn, n_seqs=n)
        cpu.refused(-7, cpu.attn_back, n_seqs=n)
        cpu.refused(-7, tffn.attention_backward_workspace, cpu.shape(n_seqs=n))
    cpu.no_device(cpu.attn, n_seqs=1 << 30)
