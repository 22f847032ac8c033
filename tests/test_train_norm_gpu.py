"""-m gpu: RMS and layer norm of training rows, both directions, against the formulas in 64 bits.

Tolerances. One rounding to the stored type: finfo.eps / 2 of the value. In fp32 a row's sums run over at most 64 terms of a thread and
a tree of 10, then the mean over the row: (64 + 10) 2^-24 = 4.4e-6 of the sum of magnitudes, half of that in rstd; FP = 1e-5 covers it and the
few products behind it, relative to the magnitudes that are added (so it holds where they cancel). dweight and dbias add rows / blocks
terms in a thread, then at most 4 warps, 40 blocks of a run and 16 runs: that many 2^-24 of the sum of magnitudes."""
import pytest

pytestmark = pytest.mark.gpu
FP = 1e-5
TYPES = ["bfloat16", "float32"]


def half_step(t):
    import torch
    return torch.finfo(t).eps / 2


def make(rows, width, dtype, kind, seed=0, offset=0):
    """inputs as views `offset` elements into their buffers"""
    import torch
    g = torch.Generator("cuda").manual_seed(seed)
    t = getattr(torch, dtype)

    def tensor(*shape, std=1.0, mean=0.0):
        n = 1
        for s in shape:
            n *= s
        flat = torch.empty(n + offset, dtype=t, device="cuda")
        out = flat[offset:].view(shape)
        out.copy_(torch.randn(shape, generator=g, device="cuda") * std + mean)
        return out
    return dict(x=tensor(rows, width, std=2.0, mean=0.5), weight=tensor(width, std=0.3, mean=1.0), bias=tensor(width) if kind == "layer" else None,
                dy=tensor(rows, width), skip=tensor(rows, width), new=lambda *s: torch.full(s, float("nan"), device="cuda", dtype=t))


def ptr(t):
    return None if t is None else t.data_ptr()


def forward(s, kind, dtype, eps=1e-6, y=None, stream=0):
    import tffn
    import torch
    rows, width = s["x"].shape
    y = torch.empty_like(s["x"]) if y is None else y
    mean = torch.empty(rows, device="cuda") if kind == "layer" else None
    rstd = torch.empty(rows, device="cuda")
    tffn.norm_forward(kind, dtype, ptr(s["x"]), ptr(s["weight"]), ptr(s["bias"]), rows, width, eps, ptr(y), ptr(mean), ptr(rstd), stream=stream)
    return y, mean, rstd


def backward(s, kind, dtype, mean, rstd, skip=True, dx=None, sums=True, stream=0):
    import tffn
    import torch
    rows, width = s["x"].shape
    dx = torch.empty_like(s["x"]) if dx is None else dx
    dw = torch.full((width,), float("nan"), device="cuda") if sums else None
    db = torch.full((width,), float("nan"), device="cuda") if sums and kind == "layer" else None
    size = tffn.norm_backward_workspace(rows, width)
    ws = torch.empty(max(size, 16), dtype=torch.uint8, device="cuda")
    tffn.norm_backward(kind, dtype, ptr(s["dy"]), ptr(s["x"]), ptr(s["weight"]), ptr(mean), ptr(rstd), ptr(s["skip"]) if skip else None, rows, width, ptr(dx), ptr(dw),
                       ptr(db), ptr(ws) if sums else None, size if sums else 0, stream=stream)
    return dx, dw, db


def check_forward(s, kind, dtype, y, mean, rstd, eps=1e-6, x=None):
    import torch
    x = (s["x"] if x is None else x).double()
    w, b = s["weight"].double(), s["bias"].double() if kind == "layer" else 0.0
    m = x.mean(-1, keepdim=True) if kind == "layer" else torch.zeros_like(x[:, :1])
    r = 1 / (((x - m) ** 2).mean(-1, keepdim=True) + eps).sqrt()
    want = (x - m) * r * w + b
    size = (x.abs() + m.abs()) * r * w.abs() + (b.abs() if kind == "layer" else 0.0)
    tol = half_step(y.dtype) * want.abs() + FP * size + 1e-30
    assert ((y.double() - want).abs() <= tol).all()
    assert ((rstd.double() - r[:, 0]).abs() <= FP * r[:, 0] * (1 + (m[:, 0] * r[:, 0]) ** 2 * 1e-2)).all()
    if kind == "layer":
        assert ((mean.double() - m[:, 0]).abs() <= FP * x.abs().mean(-1)).all()


def check_backward(s, kind, dtype, mean, rstd, dx, dw, db, skip=True, x=None, dy=None, passed=None):
    """with the statistics that the call was given"""
    import torch
    x, dy = (s["x"] if x is None else x).double(), (s["dy"] if dy is None else dy).double()
    w, r = s["weight"].double(), rstd.double()[:, None]
    m = mean.double()[:, None] if kind == "layer" else 0.0
    n, g = (x - m) * r, dy * w
    want = g - n * (g * n).mean(-1, keepdim=True)
    size = g.abs() + n.abs() * (g * n).abs().mean(-1, keepdim=True)
    if kind == "layer":
        want, size = want - g.mean(-1, keepdim=True), size + g.abs().mean(-1, keepdim=True)
    want, size = want * r, size * r
    if skip:
        passed = (s["skip"] if passed is None else passed).double()
        want, size = want + passed, size + passed.abs()
    if kind == "layer":
        size = size + size * 2 * (m.abs() * r)  # x - mean where the mean is the larger
    tol = half_step(dx.dtype) * want.abs() + FP * size + 1e-30
    assert ((dx.double() - want).abs() <= tol).all()
    terms = len(x) / 1 + 4 + 40 + 16
    if dw is not None:
        size = (dy * n).abs().sum(0)
        if kind == "layer":
            size = size + (dy * m * r).abs().sum(0)
        assert ((dw.double() - (dy * n).sum(0)).abs() <= (terms * 2 ** -24 + FP) * size + 1e-30).all()
    if db is not None:
        assert ((db.double() - dy.sum(0)).abs() <= terms * 2 ** -24 * dy.abs().sum(0) + 1e-30).all()


WIDTHS = [1, 2, 7, 8, 64, 100, 512, 896, 1024, 1032, 1111, 1536, 2048, 2056, 3584, 4095, 4097, 8192, 8200, 16383, 16384]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("width", WIDTHS)
def test_norm(width, kind, dtype):
    for rows in (1, 5, 131):
        s = make(rows, width, dtype, kind, seed=rows)
        y, mean, rstd = forward(s, kind, dtype)
        check_forward(s, kind, dtype, y, mean, rstd)
        dx, dw, db = backward(s, kind, dtype, mean, rstd)
        check_backward(s, kind, dtype, mean, rstd, dx, dw, db)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("rows,width", [(5000, 64), (3001, 896), (1300, 3584)])
def test_norm_many_rows(rows, width, kind, dtype):
    """more rows than blocks; twice the same bits"""
    import torch
    s = make(rows, width, dtype, kind, seed=3)
    y, mean, rstd = forward(s, kind, dtype)
    check_forward(s, kind, dtype, y, mean, rstd)
    a = backward(s, kind, dtype, mean, rstd, skip=False)
    check_backward(s, kind, dtype, mean, rstd, *a, skip=False)
    b = backward(s, kind, dtype, mean, rstd, skip=False)
    assert all(torch.equal(p, q) for p, q in zip(a, b) if p is not None)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("offset", [1, 3])
def test_norm_unaligned(offset, dtype):
    for kind, width in (("rms", 896), ("layer", 64), ("layer", 6000)):
        s = make(9, width, dtype, kind, seed=5, offset=offset)
        y, mean, rstd = forward(s, kind, dtype)
        check_forward(s, kind, dtype, y, mean, rstd)
        check_backward(s, kind, dtype, mean, rstd, *backward(s, kind, dtype, mean, rstd))


@pytest.mark.parametrize("over", ["dy", "x", "skip"])
def test_norm_in_place(over):
    for kind, dtype, width in (("rms", "bfloat16", 896), ("layer", "float32", 1111), ("layer", "bfloat16", 3584)):
        s = make(700, width, dtype, kind, seed=7)
        x = s["x"].clone()
        kept = s["x"].clone()
        y, mean, rstd = forward(dict(s, x=x), kind, dtype, y=x)
        check_forward(s, kind, dtype, y, mean, rstd, x=kept)
        old = {n: s[n].clone() for n in ("x", "dy", "skip")}
        dx, dw, db = backward(s, kind, dtype, mean, rstd, dx=s[over])
        check_backward(s, kind, dtype, mean, rstd, dx, dw, db, x=old["x"], dy=old["dy"], passed=old["skip"])


def test_norm_rows_that_are_missing_and_neighbours():
    """no rows: zero sums; rows behind the last one stay; a frozen norm has no sums"""
    import tffn
    import torch
    dw, db = torch.ones(64, device="cuda"), torch.ones(64, device="cuda")
    w = torch.ones(64, device="cuda")
    tffn.norm_forward("rms", "float32", None, ptr(w), None, 0, 64, 1e-6, None, None, None)
    tffn.norm_backward("layer", "float32", None, None, ptr(w), None, None, None, 0, 64, None, ptr(dw), ptr(db), None, 0)
    assert not dw.any() and not db.any()
    s = make(8, 896, "bfloat16", "rms")
    y = s["new"](8, 896)
    s5 = dict(s, x=s["x"][:5], dy=s["dy"][:5], skip=s["skip"][:5])
    _, mean, rstd = forward(s5, "rms", "bfloat16", y=y[:5])
    dx = s["new"](8, 896)
    out = backward(s5, "rms", "bfloat16", mean, rstd, dx=dx[:5], sums=False)
    check_forward(s5, "rms", "bfloat16", y[:5], mean, rstd)
    check_backward(s5, "rms", "bfloat16", mean, rstd, dx[:5], out[1], out[2])
    assert y[5:].isnan().all() and dx[5:].isnan().all()


def test_norm_large_mean_and_gradient_by_differences():
    """a mean a thousand times the deviation: the variance is taken about it; and dx, dweight, dbias against differences of the formula in 64 bits"""
    import torch
    g = torch.Generator("cuda").manual_seed(1)
    rows, width = 4, 320
    x = (torch.randn(rows, width, generator=g, device="cuda") + 1000.0)
    s = dict(make(rows, width, "float32", "layer", seed=2), x=x)
    y, mean, rstd = forward(s, "layer", "float32")
    d = x.double() - x.double().mean(-1, keepdim=True)
    want = 1 / ((d ** 2).mean(-1) + 1e-6).sqrt()
    assert ((rstd.double() - want).abs() <= 1e-5 * want + 2 * 1000 * 2 ** -24 * want ** 2).all()
    s = make(rows, width, "float32", "layer", seed=4)
    y, mean, rstd = forward(s, "layer", "float32")
    dx, dw, db = backward(s, "layer", "float32", mean, rstd, skip=False)

    def loss(x, w, b):
        m = x.mean(-1, keepdim=True)
        n = (x - m) / (((x - m) ** 2).mean(-1, keepdim=True) + 1e-6).sqrt()
        return ((n * w + b) * s["dy"].double()).sum()
    args = [s[n].double() for n in ("x", "weight", "bias")]
    for i, grad in enumerate((dx, dw, db)):
        way = torch.randn(args[i].shape, generator=g, device="cuda", dtype=torch.float64)
        h = 1e-5
        up, down = ([a + (h * k * way if j == i else 0.0) for j, a in enumerate(args)] for k in (1, -1))
        slope = (loss(*up) - loss(*down)) / (2 * h)
        # differences of a smooth function are off by h^2; the gradient by FP of the magnitudes
        assert abs((grad.double() * way).sum() - slope) <= 1e-4 * (grad.double() * way).abs().sum()


def test_norm_streams_and_graph():
    """another stream, and a captured pair of calls replayed on new inputs"""
    import torch
    s = make(300, 896, "bfloat16", "layer", seed=9)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    y, mean, rstd = forward(s, "layer", "bfloat16", stream=st.cuda_stream)
    st.synchronize()
    check_forward(s, "layer", "bfloat16", y, mean, rstd)
    backward(s, "layer", "bfloat16", mean, rstd, stream=st.cuda_stream)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        y, mean, rstd = forward(s, "layer", "bfloat16", stream=st.cuda_stream)
        out = backward(s, "layer", "bfloat16", mean, rstd, stream=st.cuda_stream)
    for seed in (10, 11):
        new = make(300, 896, "bfloat16", "layer", seed=seed)
        for n in ("x", "weight", "bias", "dy", "skip"):
            s[n].copy_(new[n])
        graph.replay()
        torch.cuda.synchronize()
        check_forward(s, "layer", "bfloat16", y, mean, rstd)
        check_backward(s, "layer", "bfloat16", mean, rstd, *out)
