"""What the speed of the training operators is measured on: one pass of each case is one call, as a trainer of expert deltas makes
it of a frozen base, with buffers and workspaces that it keeps from step to step.

Norms (RMS and layer), packed causal attention with grouped heads, log-probabilities of sampled tokens and the clipped policy loss
with its KL term, in both directions. Where `own` is false a pass computes them from elementary torch operations in 32 bits (sums
over a vocabulary and a token's ratio in 64); where it is true it calls this repository's entry points. Widths, heads and
vocabularies are those of this repository's models; everything comes from the seed."""
import math
import os
import sys

import torch

own = False

# width, query heads, key/value heads, head width, vocabulary of the shapes in tensor-ffn_b200/synth.py
MODELS = {
    "0.5b": (896, 14, 2, 64, 151936),
    "1.5b": (1536, 12, 2, 128, 151936),
    "3b": (2048, 16, 2, 128, 151936),
    "7b": (3584, 28, 4, 128, 152064),
    "stack": (896, 14, 2, 64, 32768),
}
DTYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}
EPS = 1e-6
CLIP_LOW, CLIP_HIGH, KL = 0.2, 0.28, 0.04


def norm(name, kind, direction, rows, width, dtype, skip=False):
    return {"name": name, "op": "norm", "kind": kind, "direction": direction, "rows": rows, "width": width, "dtype": dtype, "skip": skip}


def attention(name, direction, model, seqs, longest, ragged=False, prefix=0, chunk=0, tail=0):
    return {"name": name, "op": "attention", "direction": direction, "model": model, "seqs": seqs, "longest": longest, "ragged": ragged,
            "prefix": prefix, "chunk": chunk, "tail": tail}


def loss(name, op, rows, vocab, dtype, masked=0.0):
    return {"name": name, "op": op, "rows": rows, "vocab": vocab, "dtype": dtype, "masked": masked}


def listed():
    return [
        # one short answer through a norm of the 0.5B model: latency
        norm("norm_few", "rms", "forward", 7, 896, "bfloat16"),
        # a batch through a norm of the 3B model
        norm("norm_batch", "rms", "forward", 8192, 2048, "bfloat16"),
        # backward of the widest model's norm, with the gradient that passes it by on the residual stream
        norm("norm_back_wide", "rms", "backward", 16384, 3584, "bfloat16", skip=True),
        # a layer norm in 32 bits of an odd width: the checks of a new layer
        norm("norm_back_odd", "layer", "backward", 4099, 1111, "float32"),
        # one short answer, both sides of latency
        attention("attn_few", "forward", "0.5b", 1, 37),
        # a batch of ragged documents on the 128-wide heads
        attention("attn_documents", "forward", "1.5b", 8, 2048, ragged=True),
        # many short ragged answers
        attention("attn_back_answers", "backward", "0.5b", 32, 512, ragged=True, tail=5),
        # one long context of the widest model
        attention("attn_back_long", "backward", "7b", 1, 8192),
        # attention inside chunks, behind keys that were there before
        attention("attn_back_chunks", "backward", "stack", 3, 2777, prefix=300, chunk=1024),
        # log-probabilities of sampled tokens under the policy that sampled them
        loss("logprob_batch", "logprob", 1024, 151936, "float32"),
        # a few tokens of a small vocabulary: latency
        loss("policy_few", "policy", 13, 1000, "float32"),
        # a training batch, prompt tokens masked
        loss("policy_batch", "policy", 2048, 151936, "float32", masked=0.25),
    ]


def draw(rng):
    def size(lo, hi):
        return min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))
    op = rng.choice(["norm", "norm", "attention", "attention", "attention", "logprob", "policy", "policy"])
    if op == "norm":
        width = rng.choice([896, 1536, 2048, 3584, size(64, 8192)])
        dtype = rng.choice(["bfloat16", "bfloat16", "float32"])
        rows = size(1, (1 << 25) // width)
        direction = rng.choice(["forward", "backward"])
        return norm("", rng.choice(["rms", "rms", "layer"]), direction, rows, width, dtype, direction == "backward" and rng.random() < 0.5) | {"name": None}
    if op == "attention":
        model = rng.choice(sorted(MODELS))
        longest = size(1, 6000)
        seqs = size(1, max(1, min(64, 50000000 // (longest * (longest + 1024)))))
        chunk = size(64, 1024) if rng.random() < 0.2 else 0
        return attention("", rng.choice(["forward", "backward"]), model, seqs, longest, seqs > 1 and rng.random() < 0.7,
                         size(1, 1024) if rng.random() < 0.25 else 0, chunk, rng.randrange(9)) | {"name": None}
    vocab = rng.choice([151936, 152064, 32768, size(100, 60000)])
    rows = size(1, (1 << 28) // vocab)
    return loss("", op, rows, vocab, rng.choice(["float32", "float32", "bfloat16"]), rng.choice([0.0, 0.25, 0.6]) if op == "policy" else 0.0) | {"name": None}


def lengths(case):
    """query tokens of each sequence; the longest is there, the others are spread below it"""
    n, longest = case["seqs"], case["longest"]
    if not case["ragged"]:
        return [longest] * n
    return [longest] + [1 + int((longest - 1) * ((i * 0.6180339887) % 1.0)) for i in range(1, n)]


def key_lengths(case):
    return [n + case["prefix"] for n in lengths(case)]


def visible_pairs(case):
    """(query, key) pairs that the mask lets through, of one head"""
    total, chunk = 0, case["chunk"]
    for nq, nk in zip(lengths(case), key_lengths(case)):
        for p in range(nk - nq, nk):
            total += p + 1 - (p // chunk * chunk if chunk else 0)
    return total


def heads_of(case):
    return MODELS[case["model"]][1:4]


def work(case):
    if case["op"] == "norm":
        n, size = case["rows"] * case["width"], DTYPES[case["dtype"]].itemsize
        tensors = 2 if case["direction"] == "forward" else 3 + case["skip"]
        vectors = case["width"] * (size * 2 if case["direction"] == "forward" else size + 8)
        return {"bytes": tensors * n * size + vectors + 8 * case["rows"], "flops": (6 if case["direction"] == "forward" else 12) * n}
    if case["op"] == "attention":
        heads, kv, dim = heads_of(case)
        q, k, pairs = sum(lengths(case)), sum(key_lengths(case)), visible_pairs(case)
        rows = 2 * q * heads * dim + 2 * k * kv * dim  # q, out; k, v
        if case["direction"] == "forward":
            return {"bytes": 2 * rows + 4 * q * heads, "flops": 4 * pairs * heads * dim}
        return {"bytes": 4 * rows + 4 * q * heads, "flops": 10 * pairs * heads * dim}
    size = DTYPES[case["dtype"]].itemsize
    n = case["rows"] * case["vocab"]
    if case["op"] == "logprob":
        return {"bytes": n * size + 12 * case["rows"], "flops": 3 * n}
    # masked rows are not read, their gradient is written
    return {"bytes": (n - masked_rows(case) * case["vocab"] + n) * size + 32 * case["rows"], "flops": 6 * n}


def masked_rows(case):
    return min(case["rows"] - 1, int(case["rows"] * case["masked"]))


# ------------------------------------------------------------------------------------------------------------- inputs
def generator(seed):
    return torch.Generator("cuda").manual_seed(seed)


def normal(g, shape, std=1.0, mean=0.0, dtype=torch.float32):
    return torch.randn(shape, generator=g, device="cuda").mul_(std).add_(mean).to(dtype)


def norm_inputs(case, seed):
    g, dtype, shape = generator(seed), DTYPES[case["dtype"]], (case["rows"], case["width"])
    # the residual stream differs in size from token to token
    x = torch.randn(shape, generator=g, device="cuda")
    x = x.mul_(torch.exp(normal(g, (case["rows"], 1), 0.5))).add_(normal(g, (case["rows"], 1), 0.1)).to(dtype)
    s = {"x": x, "weight": normal(g, case["width"], 0.1, 1.0, dtype), "bias": normal(g, case["width"], 0.1, 0.0, dtype)}
    if case["direction"] == "backward":
        s["dy"] = normal(g, shape, 0.02, 0.0, dtype)
        s["skip"] = normal(g, shape, 0.02, 0.0, dtype) if case["skip"] else None
    return s


def attention_inputs(case, seed):
    g = generator(seed)
    heads, kv, dim = heads_of(case)
    nq, nk = sum(lengths(case)) + case["tail"], sum(key_lengths(case)) + case["tail"]
    s = {"q": normal(g, (nq, heads, dim), 1.2, 0.0, torch.bfloat16), "k": normal(g, (nk, kv, dim), 1.2, 0.0, torch.bfloat16),
         "v": normal(g, (nk, kv, dim), 1.0, 0.0, torch.bfloat16)}
    if case["direction"] == "backward":
        s["dout"] = normal(g, (nq, heads, dim), 0.02, 0.0, torch.bfloat16)
    return s


def loss_inputs(case, seed):
    g, dtype = generator(seed), DTYPES[case["dtype"]]
    rows, vocab = case["rows"], case["vocab"]
    logits = torch.empty(rows, vocab, device="cuda", dtype=dtype)
    for a in range(0, rows, 256):
        logits[a:a + 256] = normal(g, (min(256, rows - a), vocab), 2.0, 0.0, dtype)
    targets = torch.randint(0, vocab, (rows,), generator=g, device="cuda", dtype=torch.int32)
    # sampled tokens are likely ones
    at = (torch.arange(rows, device="cuda"), targets.long())
    logits[at] = (logits[at].float() + normal(g, rows, 3.0, 8.0)).to(dtype)
    s = {"logits": logits, "targets": targets}
    if case["op"] == "policy":
        now = torch.cat([torch.log_softmax(logits[a:a + 256].float(), -1)[torch.arange(len(targets[a:a + 256]), device="cuda"), targets[a:a + 256].long()]
                         for a in range(0, rows, 256)])
        s["old"] = now + normal(g, rows, 0.2)
        s["ref"] = now + normal(g, rows, 0.3)
        s["advantage"] = normal(g, rows)
        weight = torch.full((rows,), 1.0 / (rows - masked_rows(case)), device="cuda")
        weight[torch.randperm(rows, generator=g, device="cuda")[:masked_rows(case)]] = 0.0
        s["weight"] = weight
    return s


def offsets(lens):
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return out


def prepare(case, seed):
    """inputs, and the buffers a trainer keeps for what the calls write"""
    s = {"case": case}
    if case["op"] == "norm":
        s.update(norm_inputs(case, seed))
        x, rows, width = s["x"], case["rows"], case["width"]
        if case["direction"] == "backward":
            # the forward pass has left these
            xf = x.float()
            s["mean"] = xf.mean(-1) if case["kind"] == "layer" else None
            centred = xf - s["mean"][:, None] if case["kind"] == "layer" else xf
            s["rstd"] = torch.rsqrt((centred * centred).mean(-1) + EPS)
            s.update(dx=torch.empty_like(x), dweight=torch.empty(width, device="cuda"), dbias=torch.empty(width, device="cuda") if case["kind"] == "layer" else None)
        else:
            s.update(y=torch.empty_like(x), rstd=torch.empty(rows, device="cuda"), mean=torch.empty(rows, device="cuda") if case["kind"] == "layer" else None)
    elif case["op"] == "attention":
        s.update(attention_inputs(case, seed))
        q, k = s["q"], s["k"]
        s["cu_q"] = torch.tensor(offsets(lengths(case)), dtype=torch.int32, device="cuda")
        s["cu_k"] = torch.tensor(offsets(key_lengths(case)), dtype=torch.int32, device="cuda")
        if case["direction"] == "backward":
            s["out"], s["lse"] = plain_attention_forward(s)  # the forward pass has left these
            s.update(dq=torch.zeros_like(q), dk=torch.zeros_like(k), dv=torch.zeros_like(k))
        else:
            s.update(out=torch.zeros_like(q), lse=torch.zeros(q.shape[1], q.shape[0], device="cuda"))
    else:
        s.update(loss_inputs(case, seed))
        rows = case["rows"]
        s["logprob"] = torch.empty(rows, device="cuda")
        if case["op"] == "policy":
            s.update(dlogits=torch.empty_like(s["logits"]), row_loss=torch.empty(rows, device="cuda"), kl=torch.empty(rows, device="cuda"),
                     loss=torch.empty(1, device="cuda"))
    if own:
        keep(s)
    return s


# ------------------------------------------------------------------------------------------------ the framework's calls
def library():
    folder = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "tensor-ffn_b200")
    if folder not in sys.path:
        sys.path.insert(0, folder)
    import tffn
    return tffn


def pointer(t):
    return None if t is None else t.data_ptr()


def keep(s):
    """what a trainer makes once: descriptions and workspaces"""
    tffn, case = library(), s["case"]
    s["lib"] = tffn
    size = 0
    if case["op"] == "norm" and case["direction"] == "backward":
        size = tffn.norm_backward_workspace(case["rows"], case["width"])
    if case["op"] == "attention":
        heads, kv, dim = heads_of(case)
        s["shape"] = tffn.AttentionShape(n_seqs=case["seqs"], heads=heads, kv_heads=kv, head_dim=dim, rows_q=s["q"].shape[0], rows_k=s["k"].shape[0],
                                         max_q=max(lengths(case)), max_k=max(key_lengths(case)), q_stride=heads * dim, k_stride=kv * dim,
                                         v_stride=kv * dim, out_stride=heads * dim, causal=1, chunk=case["chunk"], scale=dim ** -0.5)
        if case["direction"] == "backward":
            size = tffn.attention_backward_workspace(s["shape"])
    s["workspace"] = torch.empty(max(size, 1), dtype=torch.uint8, device="cuda")
    s["workspace_bytes"] = size


def run_own(s):
    case, tffn, p = s["case"], s["lib"], pointer
    stream = torch.cuda.current_stream().cuda_stream
    if case["op"] == "norm":
        if case["direction"] == "forward":
            bias = s["bias"] if case["kind"] == "layer" else None
            tffn.norm_forward(case["kind"], case["dtype"], p(s["x"]), p(s["weight"]), p(bias), case["rows"], case["width"], EPS, p(s["y"]), p(s["mean"]),
                              p(s["rstd"]), stream=stream)
            return outputs(s)
        tffn.norm_backward(case["kind"], case["dtype"], p(s["dy"]), p(s["x"]), p(s["weight"]), p(s["mean"]), p(s["rstd"]), p(s["skip"]), case["rows"],
                           case["width"], p(s["dx"]), p(s["dweight"]), p(s["dbias"]), p(s["workspace"]), s["workspace_bytes"], stream=stream)
        return outputs(s)
    if case["op"] == "attention":
        if case["direction"] == "forward":
            tffn.attention_forward(s["shape"], p(s["cu_q"]), p(s["cu_k"]), p(s["q"]), p(s["k"]), p(s["v"]), p(s["out"]), p(s["lse"]), stream=stream)
        else:
            tffn.attention_backward(s["shape"], p(s["cu_q"]), p(s["cu_k"]), p(s["q"]), p(s["k"]), p(s["v"]), p(s["out"]), p(s["lse"]), p(s["dout"]),
                                    p(s["dq"]), p(s["dk"]), p(s["dv"]), p(s["workspace"]), s["workspace_bytes"], stream=stream)
        return outputs(s)
    if case["op"] == "logprob":
        tffn.token_logprobs(case["dtype"], p(s["logits"]), p(s["targets"]), case["rows"], case["vocab"], p(s["logprob"]), stream=stream)
        return outputs(s)
    tffn.policy_loss(case["dtype"], p(s["logits"]), p(s["targets"]), p(s["old"]), p(s["ref"]), p(s["advantage"]), p(s["weight"]), case["rows"], case["vocab"],
                     CLIP_LOW, CLIP_HIGH, KL, p(s["loss"]), p(s["row_loss"]), p(s["logprob"]), p(s["kl"]), p(s["dlogits"]), stream=stream)
    return outputs(s)


NAMES = {("norm", "forward"): ("y", "mean", "rstd"), ("norm", "backward"): ("dx", "dweight", "dbias"), ("attention", "forward"): ("out", "lse"),
         ("attention", "backward"): ("dq", "dk", "dv"), ("logprob", None): ("logprob",), ("policy", None): ("loss", "row_loss", "logprob", "kl", "dlogits")}


def outputs(s):
    case = s["case"]
    return {n: s[n] for n in NAMES[case["op"], case.get("direction")] if s[n] is not None}


# --------------------------------------------------------------------------------------------------------- plain forms
def plain_norm(s):
    case = s["case"]
    x, w, dtype = s["x"].float(), s["weight"].float(), s["x"].dtype
    layer = case["kind"] == "layer"
    if case["direction"] == "forward":
        mean = x.mean(-1) if layer else None
        c = x - mean[:, None] if layer else x
        rstd = torch.rsqrt((c * c).mean(-1) + EPS)
        y = c * rstd[:, None] * w
        if layer:
            y = y + s["bias"].float()
        out = {"y": y.to(dtype), "mean": mean, "rstd": rstd}
    else:
        dy, rstd = s["dy"].float(), s["rstd"][:, None]
        n = (x - s["mean"][:, None] if layer else x) * rstd
        g = dy * w
        dx = g - n * (g * n).mean(-1, keepdim=True)
        if layer:
            dx = dx - g.mean(-1, keepdim=True)
        dx = dx * rstd
        if s["skip"] is not None:
            dx = dx + s["skip"].float()
        out = {"dx": dx.to(dtype), "dweight": (dy * n).sum(0, dtype=torch.float64).float(), "dbias": dy.sum(0, dtype=torch.float64).float() if layer else None}
    return {n: t for n, t in out.items() if t is not None}


def allowed(case, nq, nk):
    """which key each query of a sequence sees"""
    at = torch.arange(nk - nq, nk, device="cuda")[:, None]
    key = torch.arange(nk, device="cuda")
    see = key <= at
    if case["chunk"]:
        see = see & (key >= at // case["chunk"] * case["chunk"])
    return see


def sequences(s):
    """per sequence: rows of the queries, rows of the keys, mask"""
    case = s["case"]
    q0 = k0 = 0
    for nq, nk in zip(lengths(case), key_lengths(case)):
        yield slice(q0, q0 + nq), slice(k0, k0 + nk), allowed(case, nq, nk)
        q0, k0 = q0 + nq, k0 + nk


def plain_attention_forward(s):
    heads, kv, dim = heads_of(s["case"])
    out, lse = torch.zeros_like(s["q"]), torch.zeros(heads, s["q"].shape[0], device="cuda")
    for rq, rk, see in sequences(s):
        for g in range(kv):
            of = slice(g * heads // kv, (g + 1) * heads // kv)
            q, k, v = s["q"][rq, of].float().transpose(0, 1), s["k"][rk, g].float(), s["v"][rk, g].float()
            score = torch.where(see, q @ k.T * dim ** -0.5, -math.inf)
            top = score.max(-1, keepdim=True).values
            p = torch.exp(score - top)
            total = p.sum(-1, keepdim=True)
            out[rq, of] = (p @ v / total).transpose(0, 1).to(out.dtype)
            lse[of, rq] = (top + torch.log(total))[..., 0]
    return out, lse


def plain_attention_backward(s):
    heads, kv, dim = heads_of(s["case"])
    dq, dk, dv = torch.zeros_like(s["q"]), torch.zeros_like(s["k"]), torch.zeros_like(s["v"])
    for rq, rk, see in sequences(s):
        for g in range(kv):
            of = slice(g * heads // kv, (g + 1) * heads // kv)
            q, do = s["q"][rq, of].float().transpose(0, 1), s["dout"][rq, of].float().transpose(0, 1)
            k, v = s["k"][rk, g].float(), s["v"][rk, g].float()
            score = torch.where(see, q @ k.T * dim ** -0.5, -math.inf)
            p = torch.exp(score - score.max(-1, keepdim=True).values)
            p = p / p.sum(-1, keepdim=True)
            dp = do @ v.T
            ds = p * (dp - (p * dp).sum(-1, keepdim=True)) * dim ** -0.5
            dq[rq, of] = (ds @ k).transpose(0, 1).to(dq.dtype)
            dk[rk, g] = (ds.flatten(0, 1).T @ q.flatten(0, 1)).to(dk.dtype)
            dv[rk, g] = (p.flatten(0, 1).T @ do.flatten(0, 1)).to(dv.dtype)
    return {"dq": dq, "dk": dk, "dv": dv}


def plain_loss(s):
    case = s["case"]
    rows, targets = case["rows"], s["targets"].long()
    logprob = torch.empty(rows, device="cuda", dtype=torch.float64)
    parts = range(0, rows, 256)
    top, total = torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda", dtype=torch.float64)
    for a in parts:
        x = s["logits"][a:a + 256].float()
        top[a:a + 256] = x.max(-1).values
        total[a:a + 256] = torch.exp(x - top[a:a + 256, None]).sum(-1, dtype=torch.float64)
        logprob[a:a + 256] = x.gather(1, targets[a:a + 256, None])[:, 0].double() - top[a:a + 256].double() - torch.log(total[a:a + 256])
    if case["op"] == "logprob":
        return {"logprob": logprob.float()}
    w, adv = s["weight"].double(), s["advantage"].double()
    ratio = torch.exp(logprob - s["old"].double())
    free, clipped = ratio * adv, ratio.clamp(1 - CLIP_LOW, 1 + CLIP_HIGH) * adv
    away = s["ref"].double() - logprob
    kl = torch.exp(away) - away - 1
    row_loss = w * (KL * kl - torch.minimum(free, clipped))
    slope = w * (torch.where(free <= clipped, -free, 0.0) + KL * (1 - torch.exp(away)))
    live = w != 0
    dlogits = torch.empty_like(s["logits"])
    for a in parts:
        p = torch.exp(s["logits"][a:a + 256].float() - top[a:a + 256, None]) / total[a:a + 256, None].float()
        p = torch.where(torch.arange(case["vocab"], device="cuda") == targets[a:a + 256, None], 1 - p, -p)
        dlogits[a:a + 256] = torch.where(live[a:a + 256, None], p * slope[a:a + 256, None].float(), 0.0).to(dlogits.dtype)
    return {"loss": row_loss.sum().float().reshape(1), "row_loss": row_loss.float(), "logprob": torch.where(live, logprob, 0.0).float(),
            "kl": torch.where(live, kl, 0.0).float(), "dlogits": dlogits}


def run(state):
    if own:
        return run_own(state)
    op = state["case"]["op"]
    if op == "norm":
        return plain_norm(state)
    if op == "attention":
        if state["case"]["direction"] == "backward":
            return plain_attention_backward(state)
        out, lse = plain_attention_forward(state)
        return {"out": out, "lse": lse}
    return plain_loss(state)


# -------------------------------------------------------------------------------- the definitions, in 64 bits, by autograd
def exact(case, seed):
    D = torch.float64
    if case["op"] == "norm":
        s = norm_inputs(case, seed)
        x, w = s["x"].to(D).requires_grad_(), s["weight"].to(D).requires_grad_()
        b = s["bias"].to(D).requires_grad_()
        layer, forward = case["kind"] == "layer", case["direction"] == "forward"
        mean = x.mean(-1, keepdim=True) if layer else torch.zeros_like(x[:, :1])
        rstd = 1 / (((x - mean) ** 2).mean(-1, keepdim=True) + EPS).sqrt()
        y = (x - mean) * rstd * w + (b if layer else 0.0)
        if forward:
            return {"y": y.detach()} | ({"mean": mean.detach()[:, 0]} if layer else {}) | {"rstd": rstd.detach()[:, 0]}
        dx, dw, db = torch.autograd.grad(y, (x, w, b), s["dy"].to(D), allow_unused=True)
        out = {"dx": dx + s["skip"].to(D) if case["skip"] else dx, "dweight": dw}
        return out | {"dbias": db} if layer else out
    if case["op"] == "attention":
        s = attention_inputs(case, seed) | {"case": case}
        heads, kv, dim = heads_of(case)
        if visible_pairs(case) * heads * dim > 4e11:
            return None
        q, k, v = (s[n].to(D) for n in "qkv")
        out, lse = torch.zeros_like(q), torch.zeros(heads, len(q), device="cuda", dtype=D)
        dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
        backward = case["direction"] == "backward"
        for rq, rk, see in sequences(s):
            for h in range(heads):
                g = h * kv // heads
                a, b, c = (t.clone().requires_grad_(backward) for t in (q[rq, h], k[rk, g], v[rk, g]))
                score = (a @ b.T / math.sqrt(dim)).masked_fill(~see, -math.inf)
                y = torch.softmax(score, -1) @ c
                if backward:
                    da, db, dc = torch.autograd.grad(y, (a, b, c), s["dout"][rq, h].to(D))
                    dq[rq, h] = da
                    dk[rk, g] += db
                    dv[rk, g] += dc
                else:
                    out[rq, h], lse[h, rq] = y, torch.logsumexp(score, -1)
        return {"dq": dq, "dk": dk, "dv": dv} if backward else {"out": out, "lse": lse}
    s = loss_inputs(case, seed)
    rows = case["rows"]
    kept = {n: [] for n in ("row_loss", "logprob", "kl", "dlogits")}
    for a in range(0, rows, 128):
        x = s["logits"][a:a + 128].to(D).requires_grad_(case["op"] == "policy")
        lp = torch.log_softmax(x, -1).gather(1, s["targets"][a:a + 128, None].long())[:, 0]
        if case["op"] == "logprob":
            kept["logprob"].append(lp)
            continue
        w, adv, old, ref = (s[n][a:a + 128].to(D) for n in ("weight", "advantage", "old", "ref"))
        ratio = (lp - old).exp()
        kl = torch.expm1(ref - lp) - (ref - lp)
        gain = torch.minimum(ratio * adv, ratio.clamp(1 - CLIP_LOW, 1 + CLIP_HIGH) * adv)
        each = w * (KL * kl - gain)
        kept["dlogits"].append(torch.autograd.grad(each.sum(), x)[0])
        for n, t in (("row_loss", each), ("logprob", torch.where(w != 0, lp, 0.0)), ("kl", torch.where(w != 0, kl, 0.0))):
            kept[n].append(t.detach())
    out = {n: torch.cat(t) for n, t in kept.items() if t}
    return {"loss": out["row_loss"].sum().reshape(1)} | out if case["op"] == "policy" else out
