"""-m gpu: the training operators together around expert_forward, as a step of a trainer of expert deltas uses them: norm, attention, norm,
the expert's delta on the residual stream, logits, policy loss; and back to the input. Each operator is checked on what it was given by
the ones before, with its own test's oracle and tolerance; the step as a whole by a second run, on another stream, and by a captured one, which have to
give the same bits (expert_forward waits for its status and stays out of the capture)."""
import pytest
import test_train_attn_gpu as attn
import test_train_loss_gpu as loss
import test_train_norm_gpu as norm

pytestmark = pytest.mark.gpu
ptr = norm.ptr


class Step:
    """One layer on packed sequences. torch does the matrix products of the frozen base between the operators, in bf16 with fp32 sums."""

    def __init__(self, model, expert, layers, hidden, lens, seed=0):
        import tffn
        import torch
        g = torch.Generator("cuda").manual_seed(seed)
        self.heads, self.kv, self.dim = hidden // 64, 1, 64
        self.tokens, self.vocab, self.hidden, self.layers, self.expert, self.lens = sum(lens), 1003, hidden, layers, expert, lens
        bf = lambda *shape, std: (torch.randn(shape, generator=g, device="cuda") * std).to(torch.bfloat16)  # noqa: E731
        self.x = bf(self.tokens, hidden, std=1.0)
        self.n1, self.n2, self.n3 = ((1 + bf(hidden, std=0.1).float()).to(torch.bfloat16) for _ in range(3))
        self.w_qkv, self.w_o = bf((self.heads + 2 * self.kv) * 64, hidden, std=hidden ** -0.5), bf(hidden, self.heads * 64, std=hidden ** -0.5)
        self.w_head = bf(self.vocab, hidden, std=hidden ** -0.5)
        self.cu = attn.offsets(lens)
        self.y = torch.randint(0, self.vocab, (self.tokens,), generator=g, device="cuda", dtype=torch.int32)
        n = lambda std: torch.randn(self.tokens, generator=g, device="cuda") * std  # noqa: E731
        self.near, self.adv = (n(0.05), n(0.05)), n(1.0)
        self.weight = (torch.rand(self.tokens, generator=g, device="cuda") < 0.7).float() / self.tokens  # prompts are masked
        self.old = self.ref = None
        w = self.w_qkv.shape[0]
        self.shape = tffn.AttentionShape(n_seqs=len(lens), heads=self.heads, kv_heads=self.kv, head_dim=64, rows_q=self.tokens, rows_k=self.tokens, max_q=max(lens),
                                         max_k=max(lens), causal=1, q_stride=w, k_stride=w, v_stride=w, out_stride=self.heads * 64, scale=0.125)
        new = lambda *shape, dtype=torch.bfloat16: torch.zeros(shape, dtype=dtype, device="cuda")  # noqa: E731
        f32 = torch.float32
        self.b = dict(h1=new(self.tokens, hidden), r1=new(self.tokens, dtype=f32), qkv=new(self.tokens, w), o=new(self.tokens, self.heads * 64),
                      lse=new(self.heads, self.tokens, dtype=f32), x2=new(self.tokens, hidden), h2=new(layers, self.tokens, hidden), r2=new(self.tokens, dtype=f32),
                      delta=new(layers, self.tokens, hidden, dtype=f32), x3=new(self.tokens, hidden), h3=new(self.tokens, hidden), r3=new(self.tokens, dtype=f32),
                      logits=new(self.tokens, self.vocab, dtype=f32), loss=new(1, dtype=f32), row_loss=new(self.tokens, dtype=f32), lp=new(self.tokens, dtype=f32),
                      kl=new(self.tokens, dtype=f32), d_logits=new(self.tokens, self.vocab, dtype=f32), dh3=new(self.tokens, hidden), dx3=new(self.tokens, hidden),
                      dn3=new(hidden, dtype=f32), do=new(self.tokens, self.heads * 64), dqkv=new(self.tokens, w), dh1=new(self.tokens, hidden), dx=new(self.tokens, hidden),
                      dn1=new(hidden, dtype=f32), norm_ws=new(tffn.norm_backward_workspace(self.tokens, hidden), dtype=torch.uint8),
                      attn_ws=new(tffn.attention_backward_workspace(self.shape), dtype=torch.uint8))

    def rms(self, x, w, y, r, stream):
        import tffn
        tffn.norm_forward("rms", "bfloat16", ptr(x), ptr(w), None, self.tokens, self.hidden, 1e-6, ptr(y), None, ptr(r), stream=stream)

    def rms_back(self, dy, x, w, r, skip, dx, dw, stream):
        import tffn
        ws = self.b["norm_ws"]
        tffn.norm_backward("rms", "bfloat16", ptr(dy), ptr(x), ptr(w), None, ptr(r), ptr(skip), self.tokens, self.hidden, ptr(dx), ptr(dw), None, ptr(ws), ws.numel(),
                           stream=stream)

    def qkv(self, t):
        return t.split([self.heads * 64, 64, 64], 1)

    def forward(self, stream=0, expert=True):
        import tffn
        import torch
        b, x = self.b, self.x
        self.rms(x, self.n1, b["h1"], b["r1"], stream)
        torch.mm(b["h1"], self.w_qkv.T, out=b["qkv"])
        tffn.attention_forward(self.shape, ptr(self.cu), ptr(self.cu), *(ptr(t) for t in self.qkv(b["qkv"])), ptr(b["o"]), ptr(b["lse"]), stream=stream)
        b["x2"].copy_(x + b["o"] @ self.w_o.T)
        self.rms(b["x2"], self.n2, b["h2"][0], b["r2"], stream)
        if expert:
            self.expert.expert_forward(ptr(b["h2"]), ptr(b["delta"]), self.tokens, stream)
        b["x3"].copy_(b["x2"] + b["delta"][0])
        self.rms(b["x3"], self.n3, b["h3"], b["r3"], stream)
        b["logits"].copy_(b["h3"] @ self.w_head.T)

    def objective(self, stream=0, grad=True):
        import tffn
        b = self.b
        tffn.policy_loss("float32", ptr(b["logits"]), ptr(self.y), ptr(self.old), ptr(self.ref), ptr(self.adv), ptr(self.weight), self.tokens, self.vocab, 0.2, 0.28, 0.1,
                         ptr(b["loss"]), ptr(b["row_loss"]), ptr(b["lp"]), ptr(b["kl"]), ptr(b["d_logits"]) if grad else None, stream=stream)

    def backward(self, stream=0):
        """to the gradient of x through the attention and the residual stream (the expert's own gradient is its delta's, dx3)"""
        import tffn
        import torch
        b = self.b
        b["dh3"].copy_(b["d_logits"].to(torch.bfloat16) @ self.w_head)
        self.rms_back(b["dh3"], b["x3"], self.n3, b["r3"], None, b["dx3"], b["dn3"], stream)
        torch.mm(b["dx3"], self.w_o, out=b["do"])
        tffn.attention_backward(self.shape, ptr(self.cu), ptr(self.cu), *(ptr(t) for t in self.qkv(b["qkv"])), ptr(b["o"]), ptr(b["lse"]), ptr(b["do"]),
                                *(ptr(t) for t in self.qkv(b["dqkv"])), ptr(b["attn_ws"]), b["attn_ws"].numel(), stream=stream)
        torch.mm(b["dqkv"], self.w_qkv, out=b["dh1"])
        self.rms_back(b["dh1"], self.x, self.n1, b["r1"], b["dx3"], b["dx"], b["dn1"], stream)

    def sample(self):
        """the policy that sampled the tokens, a little away from this one"""
        import tffn
        import torch
        self.forward()
        now = torch.empty(self.tokens, device="cuda")
        tffn.token_logprobs("float32", ptr(self.b["logits"]), ptr(self.y), self.tokens, self.vocab, ptr(now))
        self.old, self.ref = now + self.near[0], now + self.near[1]


RESULTS = ("h1", "o", "lse", "delta", "h3", "loss", "lp", "d_logits", "dx3", "dn3", "dqkv", "dx", "dn1")


@pytest.mark.parametrize("name,lens", [("mini05", [130, 1, 257, 64]), ("tiny", [5, 40])])
def test_step(model_dirs, name, lens):
    import tffn
    import torch
    d, ep, cfg = model_dirs[name]
    hidden = cfg["hidden_size"]
    assert hidden % 64 == 0
    model = tffn.qwen_load(d)
    expert = tffn.checkpoint_load(ep, model, 0.1)
    s = Step(model, expert, cfg["num_hidden_layers"], hidden, lens)
    s.sample()

    def run(stream=0, expert=True):
        s.forward(stream, expert)
        s.objective(stream)
        s.backward(stream)
    run()
    b = s.b
    # each operator on what it was given
    for x, w, y, r in ((s.x, s.n1, b["h1"], b["r1"]), (b["x2"], s.n2, b["h2"][0], b["r2"]), (b["x3"], s.n3, b["h3"], b["r3"])):
        norm.check_forward(dict(x=x, weight=w, bias=None), "rms", "bfloat16", y, None, r)
    head = lambda t, h: t.unflatten(1, (h, 64))  # noqa: E731
    q, k, v = (head(t, h) for t, h in zip(s.qkv(b["qkv"]), (s.heads, 1, 1)))
    dq, dk, dv = (head(t, h) for t, h in zip(s.qkv(b["dqkv"]), (s.heads, 1, 1)))
    attn.check(dict(q=q, k=k, v=v, dout=head(b["do"], s.heads), out=head(b["o"], s.heads), lse=b["lse"], dq=dq, dk=dk, dv=dv, lens=(lens, lens), shape=s.shape))
    loss.check(dict(x=b["logits"], y=s.y, old=s.old, ref=s.ref, adv=s.adv, weight=s.weight, dtype="float32"), dict(lp=b["lp"], kl=b["kl"], row_loss=b["row_loss"],
               loss=b["loss"], grad=b["d_logits"]), beta=0.1)
    norm.check_backward(dict(x=b["x3"], dy=b["dh3"], weight=s.n3), "rms", "bfloat16", None, b["r3"], b["dx3"], b["dn3"], None, skip=False)
    norm.check_backward(dict(x=s.x, dy=b["dh1"], weight=s.n1, skip=b["dx3"]), "rms", "bfloat16", None, b["r1"], b["dx"], b["dn1"], None)
    # the same bits on a second run, and from a graph
    first = {n: b[n].clone() for n in RESULTS}
    run()
    for n, t in first.items():
        assert torch.equal(t, b[n]), n
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        run(stream.cuda_stream)
    stream.synchronize()
    for n, t in first.items():
        assert torch.equal(t, b[n]), n
    with torch.cuda.graph(graph, stream=stream):
        run(stream.cuda_stream, expert=False)
    for n in RESULTS:
        if n != "delta":
            b[n].zero_()
    graph.replay()
    torch.cuda.synchronize()
    for n, t in first.items():
        assert torch.equal(t, b[n]), n
    assert tffn.train_status() == 0
