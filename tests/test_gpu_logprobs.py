"""Token log probabilities, entropy, alternatives and their gradient against 64 bits.

Bounds, with e = 2^-24: a log probability is a difference of two fp32 logarithms, each
rounded a few times (8 e of its size), plus the sum's relative error: each term 2^-22
(the base-2 exponential) and sqrt(vocab / 256) additions a thread.  So
4 e (8 + sqrt(vocab / 256)) + 8 e |value|; the entropy, a mean of such terms, four times
that.  A gradient is off by its own rounding and by 1e-5 of the row's largest.
"""

import math

import pytest
import torch

from dorafactors_b200 import _native
from dorafactors_b200.logprobs import token_logprobs, token_logprobs_backward

pytestmark = pytest.mark.gpu

U = {torch.float32: 2.0**-24, torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
INF = math.inf


@pytest.fixture(autouse=True)
def _device_error_stays_clear():
    yield
    assert _native.device_error(reset=True) == 0


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _logits(g, rows, vocab, dtype, gap=0, scale=3.0):
    wide = torch.full((rows, vocab + gap), float("nan"), device="cuda", dtype=dtype)
    wide[:, :vocab] = torch.randn(rows, vocab, device="cuda", generator=g) * scale
    return wide[:, :vocab]


def _reference(x, t, temperature, k=0, gl=None, ge=None, gs=None, ignore=-100):
    x = x.double() / temperature
    used = t != ignore
    at = torch.where(used, t, 0)[:, None]
    lse = torch.logsumexp(x, 1)
    logp = torch.log_softmax(x, 1)  # not x - lse: where all logits are the type's lowest, 64 bits absorb the sum
    p = logp.exp()
    plogp = torch.special.xlogy(p, p)
    h = -plogp.sum(1)
    zero = torch.zeros((), device="cuda", dtype=torch.float64)
    out = {"logprobs": torch.where(used, logp.gather(1, at)[:, 0], zero), "logsumexp": torch.where(used, lse, zero),
           "entropy": torch.where(used, h, zero)}
    if k:
        _, index = x.sort(dim=1, descending=True, stable=True)
        out["top"] = torch.where(used[:, None], logp.gather(1, index[:, :k]), zero)
        out["index"] = torch.where(used[:, None], index[:, :k], -1)
    if gl is not None:
        d = -gl.double()[:, None] * p - ge.double()[:, None] * (plogp + p * h[:, None]) + gs.double()[:, None] * p
        d.scatter_add_(1, at, gl.double()[:, None])
        out["grad"] = torch.where(used[:, None], d / temperature, zero)
    return out


def _close(got, ref, vocab, what, times=1.0):
    e = 2.0**-24
    same = (got.double() == ref) | ((got.double() - ref).abs() <= times * (4 * e * (8 + (vocab / 256) ** 0.5) + 8 * e * ref.abs()))
    assert same.all(), (what, got[~same][:4], ref[~same][:4])


@pytest.mark.parametrize("rows,vocab,dtype,k,gap,temperature", [
    (1, 1, F32, 1, 0, 1.0), (3, 2, BF16, 2, 0, 1.0), (2, 7, F16, 7, 1, 0.5), (5, 64, BF16, 64, 0, 1.0),
    (4, 100, F32, 20, 0, 2.0), (33, 1000, BF16, 5, 0, 1.0), (7, 1001, BF16, 20, 0, 1.0), (6, 4099, F32, 64, 5, 0.7),
    (1, 32003, F32, 20, 0, 1.0), (300, 8191, F16, 0, 1, 1.0), (9, 32000, BF16, 1, 64, 1.3), (48, 32003, BF16, 5, 0, 1.0),
    (2, 128256, F32, 20, 0, 1.0), (1, 128256, BF16, 64, 0, 1.0), (20, 128256, F16, 0, 0, 1.0),
    (160, 128257, BF16, 3, 0, 1.0), (700, 50000, BF16, 0, 0, 0.3), (1, 1000003, F32, 10, 0, 1.0),
])
def test_forward_and_gradient(rows, vocab, dtype, k, gap, temperature):
    g = _gen(rows + vocab)
    x = _logits(g, rows, vocab, dtype, gap)
    t = torch.randint(0, vocab, (rows,), device="cuda", generator=g)
    if rows > 4:
        t[1], t[rows - 1] = -100, vocab - 1
    gl, ge, gs = (torch.randn(rows, device="cuda", generator=g) for _ in range(3))
    ref = _reference(x, t, temperature, k, gl, ge, gs)
    leaf = x.detach().requires_grad_()
    r = token_logprobs(leaf, t, temperature=temperature, entropy=True, top_k=k)
    _close(r.logprobs.detach(), ref["logprobs"], vocab, "logprobs")
    _close(r.logsumexp.detach(), ref["logsumexp"], vocab, "logsumexp")
    _close(r.entropy.detach(), ref["entropy"], vocab, "entropy", 4)
    if k:
        assert torch.equal(r.top_indices, ref["index"])
        _close(r.top_logprobs, ref["top"], vocab, "top")
    bare = token_logprobs(x, t, temperature=temperature)
    assert bare.entropy is None and bare.top_logprobs is None
    _close(bare.logprobs, ref["logprobs"], vocab, "logprobs alone")
    (grad,) = torch.autograd.grad((r.logprobs, r.entropy, r.logsumexp), leaf, (gl, ge, gs))
    assert grad.dtype is dtype and grad.shape == x.shape
    tiny = 2.0**-25 if dtype is F16 else 0.0
    off = (grad.double() - ref["grad"]).abs()
    most = ref["grad"].abs().amax(1, keepdim=True)
    assert (off <= U[dtype] * ref["grad"].abs() + 1e-5 * most + tiny).all()
    assert torch.count_nonzero(grad[t == -100]) == 0
    # The gradient of log probabilities alone, and in place of the logits.
    lse, ent = r.logsumexp.detach(), r.entropy.detach()
    alone = _reference(x, t, temperature, 0, gl, 0 * ge, 0 * gs)["grad"]
    d = token_logprobs_backward(gl, None, None, x, t, lse, temperature=temperature)
    assert ((d.double() - alone).abs() <= U[dtype] * alone.abs() + 1e-5 * alone.abs().amax(1, keepdim=True) + tiny).all()
    y = x.clone()
    assert token_logprobs_backward(gl, ge, gs, y, t, lse, ent, temperature=temperature, out=y) is y
    assert torch.equal(y, grad)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("vocab", [50, 5000, 40000])
def test_top_ties_and_orders(vocab, dtype):
    """Equal logits go to the lower column, in any order in which the row is met."""
    g = _gen(vocab)
    rows = [torch.zeros(vocab, device="cuda"), torch.randint(0, 3, (vocab,), device="cuda", generator=g).float(),
            torch.arange(vocab, device="cuda").float(), torch.arange(vocab, 0, -1, device="cuda").float(),
            -torch.randint(0, 2, (vocab,), device="cuda", generator=g).float() * 0.0,
            torch.where(torch.arange(vocab, device="cuda") % 7 == 0, 5.0, -5.0)]
    x = torch.stack(rows).to(dtype)
    t = torch.zeros(len(rows), dtype=torch.int64, device="cuda")
    for k in (1, 2, 33, 50):
        r = token_logprobs(x, t, top_k=k)
        ref = _reference(x, t, 1.0, k)
        assert torch.equal(r.top_indices, ref["index"])
        _close(r.top_logprobs, ref["top"], vocab, "top")


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("vocab", [9, 1000, 40001])
def test_masked_logits(vocab, dtype):
    """-inf is a token of probability 0; the type's lowest value likewise; a row may be empty."""
    g = _gen(3)
    x = _logits(g, 6, vocab, dtype)
    low = torch.finfo(dtype).min
    x[0, 1:] = -INF
    x[1, ::2] = -INF
    x[2, ::2] = low
    x[3] = -INF
    x[4] = low
    t = torch.tensor([0, 0, 1, 2, 3, 4], device="cuda")
    gl, ge, gs = (torch.randn(6, device="cuda", generator=g) for _ in range(3))
    leaf = x.detach().requires_grad_()
    r = token_logprobs(leaf, t, entropy=True, top_k=5)
    (grad,) = torch.autograd.grad((r.logprobs, r.entropy, r.logsumexp), leaf, (gl, ge, gs))
    r = r._replace(**{name: getattr(r, name).detach() for name in ("logprobs", "entropy", "logsumexp")})
    ref = _reference(x, t, 1.0, 5, gl, ge, gs)
    keep = [0, 1, 2, 4, 5]
    for name in ("logprobs", "logsumexp", "entropy"):
        _close(getattr(r, name).detach()[keep], ref[name][keep], vocab, name, 4)
    assert torch.equal(r.top_indices[keep], ref["index"][keep])
    _close(r.top_logprobs[keep], ref["top"][keep], vocab, "top")
    most = ref["grad"][keep].abs().amax(1, keepdim=True)
    tiny = 2.0**-25 if dtype is F16 else 0.0
    assert ((grad.double() - ref["grad"])[keep].abs() <= U[dtype] * ref["grad"][keep].abs() + 1e-5 * most + tiny).all()
    assert float(r.logprobs[1]) == -INF  # the target itself is masked
    # The empty row.
    assert float(r.logprobs[3]) == float(r.logsumexp[3]) == -INF and float(r.entropy[3]) == 0
    assert torch.equal(r.top_indices[3], torch.arange(5, device="cuda")) and (r.top_logprobs[3] == -INF).all()
    assert torch.count_nonzero(grad[3]) == 0


@pytest.mark.parametrize("vocab", [40, 3000, 70001])
def test_rows_without_a_distribution(vocab):
    """A NaN or +inf makes its own row NaN; a target outside the vocabulary is reported."""
    x = _logits(_gen(4), 5, vocab, F32)
    t = torch.full((5,), 2, device="cuda")
    clean = token_logprobs(x, t, entropy=True, top_k=4)
    x[1, 7], x[3, vocab - 1] = float("nan"), INF
    r = token_logprobs(x, t, entropy=True, top_k=4)
    for name in ("logprobs", "logsumexp", "entropy", "top_logprobs"):
        got = getattr(r, name)
        assert got[[1, 3]].isnan().all() and torch.equal(got[[0, 2, 4]], getattr(clean, name)[[0, 2, 4]]), name
    assert torch.equal(r.top_indices[1], torch.arange(4, device="cuda"))
    t[0], t[2] = vocab, -7
    r = token_logprobs(x, t, entropy=True)
    assert r.logprobs[[0, 2]].isnan().all() and torch.equal(r.entropy[[0, 2, 4]], clean.entropy[[0, 2, 4]])
    assert _native.device_error(reset=True) == _native.ERR_INVALID_ARGUMENT
    # -7 as the ignored index: nothing is read, nothing reported.
    x[2] = float("nan")
    r = token_logprobs(x[2:3], t[2:3], top_k=2, ignore_index=-7)
    assert float(r.logprobs) == 0 and r.top_indices.tolist() == [[-1, -1]]


def test_peaked_rows_keep_small_differences():
    """log p near 0 is as exact as fp32 allows, whatever the logits' size."""
    x = torch.zeros(4, 1000, device="cuda")
    x[:, 0] = torch.tensor([20.0, 30.0, 60.0, 500.0], device="cuda")
    r = token_logprobs(x, torch.zeros(4, dtype=torch.int64, device="cuda"), entropy=True)
    ref = _reference(x, torch.zeros(4, dtype=torch.int64, device="cuda"), 1.0)
    assert ((r.logprobs.double() - ref["logprobs"]).abs() <= 2.0**-23).all()


def test_layouts_and_offsets():
    g = _gen(5)
    x = torch.randn(2, 3, 520, device="cuda", generator=g)
    t = torch.randint(0, 520, (2, 3), device="cuda", generator=g)
    r = token_logprobs(x, t, entropy=True, top_k=3)
    assert r.logprobs.shape == (2, 3) and r.top_indices.shape == (2, 3, 3)
    for y in (x.transpose(0, 1), x[:, :, :500], x[:, ::2], x[..., ::2]):
        u = torch.zeros(y.shape[:-1], dtype=torch.int64, device="cuda")
        a, b = token_logprobs(y, u, top_k=3), token_logprobs(y.contiguous(), u, top_k=3)
        assert torch.equal(a.top_indices, b.top_indices)
        _close(a.logprobs, b.logprobs.double(), 520, "layout")
    assert token_logprobs(x[:, :0], t[:, :0], top_k=2).top_indices.shape == (2, 0, 2)
    # Rows beyond 32-bit offsets, and one misaligned by an element.
    ld = (1 << 30) + 1
    far = torch.empty(2 * ld + 1000, device="cuda", dtype=BF16).as_strided((3, 1000), (ld, 1))
    far.copy_(torch.randn(3, 1000, device="cuda", generator=g))
    u = torch.tensor([1, 2, 999], device="cuda")
    leaf = far.detach().requires_grad_()
    r = token_logprobs(leaf, u, entropy=True, top_k=9)
    ref = _reference(far, u, 1.0, 9, *(torch.ones(3, device="cuda"),) * 3)
    _close(r.logprobs.detach(), ref["logprobs"], 1000, "far")
    assert torch.equal(r.top_indices, ref["index"])
    (grad,) = torch.autograd.grad(r.logprobs.sum() + r.entropy.sum() + r.logsumexp.sum(), leaf)
    assert ((grad.double() - ref["grad"]).abs() <= U[BF16] * ref["grad"].abs() + 1e-5).all()


def test_gradient_against_differences():
    """Central differences along a random direction; h = 2^-7 and 2e-3 of the gradient as
    for any smooth fp32 function of order one (h^2 / 6 and rounding over 2 h)."""
    g = _gen(6)
    x = torch.randn(8, 200, device="cuda", generator=g) * 2
    t = torch.randint(0, 200, (8,), device="cuda", generator=g)
    for name in ("logprobs", "entropy", "logsumexp"):
        c = torch.randn(8, device="cuda", generator=g)

        def f(y):
            return getattr(token_logprobs(y, t, temperature=0.8, entropy=True), name)

        leaf = x.clone().requires_grad_()
        (grad,) = torch.autograd.grad(f(leaf), leaf, c)
        way = torch.randn(x.shape, device="cuda", generator=g)
        h = 2.0**-7
        slope = float(((f(x + h * way).double() - f(x - h * way).double()) * c).sum() / (2 * h))
        assert abs(slope - float((grad.double() * way).sum())) <= 2e-3 * max(1.0, float(grad.norm()))


def test_streams_graphs_and_repeats():
    g = _gen(7)
    x, t = _logits(g, 70, 9001, BF16), torch.randint(0, 9001, (70,), device="cuda", generator=g)
    first = token_logprobs(x, t, entropy=True, top_k=8)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = token_logprobs(x, t, entropy=True, top_k=8)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = token_logprobs(x, t, entropy=True, top_k=8)
    graph.replay()
    for a, b, c in zip(first, again, kept):
        assert torch.equal(a, b) and torch.equal(a, c)


def test_refusals():
    x, t = torch.randn(4, 16, device="cuda"), torch.zeros(4, dtype=torch.int64, device="cuda")
    for bad in (dict(top_k=17), dict(top_k=-1), dict(temperature=0.0), dict(temperature=float("nan"))):
        with pytest.raises(ValueError):
            token_logprobs(x, t, **bad)
    with pytest.raises(ValueError, match="top_k"):
        token_logprobs(torch.randn(1, 100, device="cuda"), t[:1], top_k=65)
    with pytest.raises(ValueError, match="int64"):
        token_logprobs(x, t.int())
    with pytest.raises(ValueError, match="match"):
        token_logprobs(x, t[:3])
    with pytest.raises(ValueError, match="dtype"):
        token_logprobs(x.double(), t)
    with pytest.raises(RuntimeError, match="CUDA"):
        token_logprobs(x, t.cpu())
    r = token_logprobs(x, t, entropy=True)
    with pytest.raises(ValueError, match="entropy"):
        token_logprobs_backward(r.logprobs, r.entropy, None, x, t, r.logsumexp)
    with pytest.raises(ValueError, match="logsumexp"):
        token_logprobs_backward(r.logprobs, None, None, x, t, r.logsumexp[:2])
    big = torch.randn(5, 16, device="cuda")
    with pytest.raises(ValueError, match="overlaps"):
        token_logprobs_backward(r.logprobs, None, None, big[:4], t, r.logsumexp, out=big[1:])
    with pytest.raises(ValueError, match="type"):
        token_logprobs_backward(r.logprobs, None, None, x, t, r.logsumexp, out=x.half())
