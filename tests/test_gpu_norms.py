"""Layer norm and RMS norm against their formulas in 64 bits.

Bounds, with u the unit roundoff of the output's type (2^-8 bf16, 2^-11 fp16, 2^-24
fp32) and e = 2^-24: an elementwise output is off by its own rounding, u |ref|, and
by the fp32 evaluation, 1e-5 of the largest value, plus the mean's error, at most
(cols / 256 + 13) e of the mean magnitude of the row (serial sums of cols / 256
terms and a tree), times rstd.  A column sum of n terms is off by u |ref| and
(8 + sqrt(n)) e of the sum of its terms' magnitudes.
"""

import pytest
import torch

from dorafactors_b200 import norms

pytestmark = pytest.mark.gpu

U = {torch.float32: 2.0**-24, torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}
TINY = {torch.float32: 0.0, torch.float16: 2.0**-25, torch.bfloat16: 0.0}
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(autouse=True)
def _device_error_stays_clear():
    from dorafactors_b200 import _native

    yield
    assert _native.device_error(reset=True) == 0


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _rows(g, rows, cols, dtype, gap, shift=0.0):
    wide = torch.full((rows, cols + gap), float("nan"), device="cuda", dtype=dtype)
    wide[:, :cols] = torch.randn(rows, cols, device="cuda", generator=g) * 1.5 + shift
    return wide[:, :cols]


def _reference(x, w, b, eps, rms, dy=None):
    x = x.double()
    one = torch.ones(x.shape[-1], device="cuda", dtype=torch.float64)
    w = one if w is None else w.double()
    mean = torch.zeros_like(x[..., :1]) if rms else x.mean(-1, keepdim=True)
    rstd = 1 / torch.sqrt(((x - mean) ** 2).mean(-1, keepdim=True) + eps)
    xh = (x - mean) * rstd
    out = {"y": xh * w + (0 if b is None else b.double()), "mean": mean[..., 0], "rstd": rstd[..., 0]}
    if dy is not None:
        d = dy.double()
        a = d * w
        out["dx"] = rstd * (a - (0 if rms else a.mean(-1, keepdim=True)) - xh * (a * xh).mean(-1, keepdim=True))
        lead = tuple(range(x.ndim - 1))
        out["dw"], out["db"] = (d * xh).sum(lead), d.sum(lead)
        out["dw_abs"], out["db_abs"] = (d * xh).abs().sum(lead), d.abs().sum(lead)
    return out


def _close(got, ref, extra, what):
    bound = U[got.dtype] * ref.abs() + TINY[got.dtype] + extra
    off = (got.double() - ref).abs()
    assert torch.isfinite(got).all() and (off <= bound).all(), (what, float((off / bound.clamp_min(1e-300)).max()))


def _check(x, w, b, dy, rms, eps=1e-5):
    ref = _reference(x, w, b, eps, rms, dy)
    cols, rows = x.shape[-1], x.shape[:-1].numel()
    e = 2.0**-24
    of_mean = 0 if rms else (cols / 256 + 13) * e * x.double().abs().mean(-1)
    if rms:
        y, rstd = norms.rms_norm_forward(x, w, eps)
        dx, dw = norms.rms_norm_backward(dy, x, w, rstd)
        db = None
    else:
        y, mean, rstd = norms.layer_norm_forward(x, w, b, eps)
        assert ((mean.double() - ref["mean"]).abs() <= of_mean + 1e-30).all()
        dx, dw, db = norms.layer_norm_backward(dy, x, w, mean, rstd)
    wmax = 1 if w is None else float(w.abs().max())
    slack = (of_mean * ref["rstd"])[..., None] * wmax if not rms else 0
    _close(rstd, ref["rstd"], 1e-5 * ref["rstd"] + (0 if rms else of_mean**2 * ref["rstd"] ** 3), "rstd")
    _close(y, ref["y"], 1e-5 * ref["y"].abs().max() + slack, "y")
    assert y.dtype is x.dtype and y.shape == x.shape
    _close(dx, ref["dx"], 1e-5 * ref["dx"].abs().max() + slack * ref["dx"].abs().max(), "dx")
    n = (8 + rows**0.5) * e
    of_mean_w = 0 if rms else (of_mean * ref["rstd"]).max() * ref["db_abs"]
    _close(dw, ref["dw"], n * ref["dw_abs"] + 1e-6 * ref["dw_abs"] + of_mean_w, "dw")
    assert dw.dtype is (x.dtype if w is None else w.dtype)
    if db is not None:
        _close(db, ref["db"], n * ref["db_abs"], "db")
    return y, dx, dw, db


@pytest.mark.parametrize("rms", [False, True], ids=["layer", "rms"])
@pytest.mark.parametrize("rows,cols,dtype,wdtype,gap", [
    (1, 1, F32, F32, 0), (3, 2, BF16, BF16, 0), (1, 8, BF16, F32, 0), (5, 31, F16, F16, 3), (17, 64, BF16, BF16, 0),
    (33, 100, F32, F32, 0), (7, 256, BF16, F32, 8), (130, 512, F16, F32, 0), (9, 1000, BF16, BF16, 0),
    (64, 1024, BF16, BF16, 0), (3, 1025, BF16, BF16, 0), (11, 2048, F32, F32, 4), (513, 2056, BF16, BF16, 0),
    (2, 4096, BF16, BF16, 0), (300, 4096, BF16, F32, 0), (31, 4104, F16, F16, 8), (70, 5003, F32, F32, 0),
    (29, 8192, BF16, BF16, 0), (1000, 8192, F32, F32, 0), (5, 8200, BF16, F32, 5), (6, 14336, F16, F16, 0),
    (4, 16384, BF16, BF16, 0), (3, 16392, BF16, BF16, 0), (5, 28672, BF16, BF16, 0), (2, 28672, F32, F32, 0),
    (2, 40001, BF16, F32, 0), (4099, 72, BF16, BF16, 0), (20000, 136, BF16, F32, 0), (700, 768, F16, F16, 16),
])
def test_norm_forward_and_backward(rows, cols, dtype, wdtype, gap, rms):
    g = _gen(rows * 31 + cols)
    x, dy = _rows(g, rows, cols, dtype, gap, 0.4), _rows(g, rows, cols, dtype, 2 * gap)
    w = (1 + 0.3 * torch.randn(cols, device="cuda", generator=g)).to(wdtype)
    b = None if rms else (0.2 * torch.randn(cols, device="cuda", generator=g)).to(wdtype)
    # A row of two equal numbers has variance 0, one of a single number always.
    _check(x, w, b, dy, rms, eps=1e-5 if cols > 2 else 0.5)


@pytest.mark.parametrize("rms", [False, True], ids=["layer", "rms"])
def test_norm_without_weight_and_constant_rows(rms):
    g = _gen(5)
    x, dy = _rows(g, 40, 640, BF16, 0), _rows(g, 40, 640, BF16, 0)
    x[3] = 2.0  # variance 0: only eps is under the root
    x[4] = 0.0
    _check(x, None, None, dy, rms, eps=0.1)


def test_mean_far_from_zero():
    """The variance is taken around the mean, not as a difference of large squares."""
    g = _gen(6)
    for cols in (64, 1000, 4096, 8192, 20000):
        x, dy = _rows(g, 6, cols, F32, 0, shift=1000.0), _rows(g, 6, cols, F32, 0)
        _check(x, torch.ones(cols, device="cuda"), None, dy, False)


def test_alignment_and_layouts():
    """Misaligned bases and rows, 3-D and transposed inputs give the values of an aligned copy."""
    g = _gen(7)
    flat = torch.randn(7 * 1032 + 9, device="cuda", generator=g).bfloat16()
    w = torch.randn(1032 + 1, device="cuda", generator=g).bfloat16()
    x = flat[1: 1 + 7 * 1032].view(7, 1032)
    _check(x, w[1:], w[:-1], flat[9:].view(7, 1032), False)
    x3 = torch.randn(2, 3, 264, device="cuda", generator=g).bfloat16()
    y, mean, rstd = norms.layer_norm_forward(x3)
    assert y.shape == x3.shape and mean.shape == rstd.shape == (2, 3)
    part = torch.randn(2, 3, 400, device="cuda", generator=g)[:, :, 8:272]
    t = torch.randn(264, 6, device="cuda", generator=g).t()
    e = torch.randn(264, device="cuda", generator=g).expand(4, 264)
    for v in (part, t, e, x3.transpose(0, 1)):
        a, b = norms.rms_norm_forward(v)[0], norms.rms_norm_forward(v.contiguous())[0]
        assert torch.equal(a, b)


@pytest.mark.parametrize("rms", [False, True], ids=["layer", "rms"])
def test_empty_and_non_finite(rms):
    f = norms.rms_norm if rms else norms.layer_norm
    x = torch.randn(0, 512, device="cuda", requires_grad=True)
    w = torch.ones(512, device="cuda", requires_grad=True)
    f(x, w).sum().backward()
    assert x.grad.shape == (0, 512) and torch.count_nonzero(w.grad) == 0
    assert f(torch.randn(4, 0, device="cuda")).shape == (4, 0)
    # A NaN or an infinity stays in its row.
    for cols in (100, 1024, 8192):
        x = torch.randn(6, cols, device="cuda")
        x[1, 3], x[4, 7] = float("nan"), float("inf")
        y = f(x)
        assert y[1].isnan().all() and y[4].isnan().any()
        assert torch.equal(y[[0, 2, 3, 5]], f(x[[0, 2, 3, 5]]))


def test_rows_beyond_32_bit_offsets():
    ld = (1 << 30) + 8
    x = torch.empty(2 * ld + 264, device="cuda", dtype=BF16).as_strided((3, 264), (ld, 1))
    dy = torch.empty(2 * ld + 264, device="cuda", dtype=BF16).as_strided((3, 264), (ld, 1))
    g = _gen(8)
    for t in (x, dy):
        t.copy_(torch.randn(3, 264, device="cuda", generator=g))
    _check(x, torch.ones(264, device="cuda"), None, dy, False)


@pytest.mark.parametrize("rms", [False, True], ids=["layer", "rms"])
@pytest.mark.parametrize("cols", [72, 1000, 4096])
def test_gradient_against_differences(cols, rms):
    """Central differences of the fp32 forward along a random direction.  h = 2^-7: their
    error is h^2 / 6 times third derivatives of order one (6e-5 of the gradient) and
    the forward's rounding over 2 h, 2^-23 sqrt(n) / 2^-6; 2e-3 of the gradient covers both."""
    g = _gen(9)
    args = [torch.randn(4, cols, device="cuda", generator=g), 1 + 0.3 * torch.randn(cols, device="cuda", generator=g)]
    if not rms:
        args.append(torch.randn(cols, device="cuda", generator=g))
    f = norms.rms_norm if rms else norms.layer_norm
    dy = torch.randn(4, cols, device="cuda", generator=g)
    grads = torch.autograd.grad(f(*[a.requires_grad_() for a in args]), args, dy)
    for i, grad in enumerate(grads):
        way = torch.randn(args[i].shape, device="cuda", generator=g)
        h = 2.0**-7
        with torch.no_grad():
            ends = [f(*[a + s * h * way if j == i else a for j, a in enumerate(args)]).double() for s in (1, -1)]
        slope = float(((ends[0] - ends[1]) * dy.double()).sum() / (2 * h))
        size = float(grad.double().norm() * way.double().norm()) / grad.numel() ** 0.5
        assert abs(slope - float((grad.double() * way.double()).sum())) <= 2e-3 * size


def test_autograd_matches_passes_and_repeats():
    """The module's gradients are the backward pass's, the same from call to call and on another stream."""
    g = _gen(10)
    x = torch.randn(3, 700, 1096, device="cuda", generator=g).bfloat16().requires_grad_()
    m = norms.LayerNorm(1096, device="cuda")
    with torch.no_grad():
        m.weight.normal_(), m.bias.normal_()
    dy = torch.randn(3, 700, 1096, device="cuda", generator=g).bfloat16()
    first = torch.autograd.grad(m(x), (x, m.weight, m.bias), dy)
    _, mean, rstd = norms.layer_norm_forward(x.detach(), m.weight, m.bias)
    passes = norms.layer_norm_backward(dy, x.detach(), m.weight, mean, rstd)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = torch.autograd.grad(m(x), (x, m.weight, m.bias), dy)
    torch.cuda.current_stream().wait_stream(side)
    for a, b, c in zip(first, again, passes):
        assert torch.equal(a, b) and torch.equal(a, c.view(a.shape))
    only = norms.layer_norm_backward(dy, x.detach(), m.weight, mean, rstd, need=(False, True, False))
    assert only[0] is None and only[2] is None and torch.equal(only[1], passes[1])
    # Parameters of a third type: computed in fp32, gradients back in theirs.
    r = norms.RMSNorm(1096, device="cuda", dtype=torch.float16)
    gx, gw = torch.autograd.grad(r(x), (x, r.weight), dy)
    assert gx.dtype is torch.bfloat16 and gw.dtype is torch.float16
    # In a graph.
    xs = x.detach()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = norms.layer_norm_backward(dy, xs, m.weight, mean, rstd)
    graph.replay()
    assert all(torch.equal(a, b.view(a.shape)) for a, b in zip(out, passes))


def test_refusals():
    x = torch.randn(4, 16, device="cuda")
    w = torch.ones(16, device="cuda")
    with pytest.raises(ValueError, match="weight"):
        norms.layer_norm(x, torch.ones(8, device="cuda"))
    with pytest.raises(ValueError, match="bias"):
        norms.layer_norm(x, w, torch.ones(1, 16, device="cuda"))
    with pytest.raises(ValueError, match="dtype"):
        norms.rms_norm(x.double(), w)
    with pytest.raises(ValueError, match="eps"):
        norms.rms_norm(x, w, -1.0)
    with pytest.raises(RuntimeError, match="CUDA"):
        norms.rms_norm(x, w.cpu())
    _, mean, rstd = norms.layer_norm_forward(x, w)
    with pytest.raises(ValueError, match="shape"):
        norms.layer_norm_backward(x[:2], x, w, mean, rstd)
    with pytest.raises(ValueError, match="mean"):
        norms.layer_norm_backward(x, x, w, mean[:2], rstd)
    with pytest.raises(ValueError, match="rstd"):
        norms.rms_norm_backward(x, x, w, rstd.double())
