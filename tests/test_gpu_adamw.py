"""AdamW over many tensors: the step in 64 bits, the 8-bit moments bit for bit.

Bounds: fp32 moments are two products and a sum, each rounded once: 3 * 2^-24 of their
terms.  A parameter is its own rounding (u |p|) and the fp32 update, a handful of
roundings: 2^-21 of |p| and of the step lr |m| / denominator.  8-bit moments are held
to a numpy evaluation of their definition in fp32, code by code.
"""

import copy

import numpy as np
import pytest
import torch

from dorafactors_b200 import _native
from dorafactors_b200.optim import AdamW

pytestmark = pytest.mark.gpu

U = {torch.float32: 2.0**-24, torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
SHAPES = [(1,), (7,), (255,), (256,), (257, 1), (3, 100), (4096,), (16, 513), (128, 1000), (8193,), (40, 2048), (300001,)]


@pytest.fixture(autouse=True)
def _device_error_stays_clear():
    yield
    assert _native.device_error(reset=True) == 0


def _params(shapes, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [torch.nn.Parameter((torch.randn(*s, device="cuda", generator=g) * 0.05).to(dtype)) for s in shapes], g


def _grads(params, g, size=1e-3):
    for p in params:
        p.grad = (torch.randn(p.shape, device="cuda", generator=g) * size *
                  torch.exp(torch.randn(p.shape, device="cuda", generator=g))).to(p.dtype)


class _Numpy8:
    """The 8-bit moments of one parameter by their definition, in numpy's fp32."""

    def __init__(self, n, index, seed):
        self.n, self.index, self.seed = n, index, seed
        self.blocks = -(-n // 256)
        self.m = np.zeros(self.blocks * 256, np.float32)
        self.v = np.zeros(self.blocks * 256, np.float32)

    @staticmethod
    def _scaled(x):
        x = x.reshape(-1, 256)
        top = np.abs(x).max(1)
        live = top >= np.float32(2.0**-100)
        inverse = np.where(live, np.float32(1.875) / np.where(live, top, np.float32(1)), np.float32(0)).astype(np.float32)
        scale = np.where(live, top * np.float32(8 / 15), np.float32(0)).astype(np.float32)
        return (np.abs(x) * inverse[:, None]).view(np.int32), scale

    def step(self, g, b1, b2, t):
        f = np.float32
        g = np.concatenate([g, np.zeros(self.blocks * 256 - self.n, np.float32)])
        m = self.m * f(b1) + g * f(1 - b1)
        v = self.v * f(b2) + (g * g) * f(1 - b2)
        y, self.ms = self._scaled(m)
        c = np.clip(((y + (1 << 19)) >> 20) - (112 << 3), 0, 127)
        self.mc = (c + 128 * (m.reshape(-1, 256) < 0)).astype(np.uint8)
        u = np.where(c > 0, ((c + (112 << 3)) << 20).astype(np.int32).view(f), f(0))
        self.m = (np.where(self.mc > 127, -u, u) * self.ms[:, None]).reshape(-1).astype(f)
        y, self.vs = self._scaled(v)
        low = np.uint64(0xFFFFFFFF)
        key = np.uint64((self.seed + t * 0x9E3779B1 + self.index * 0xC2B2AE35) & 0xFFFFFFFF)
        x = (np.arange(self.blocks * 128, dtype=np.uint64) * np.uint64(0x85EBCA77) + key) & low
        x = ((x ^ (x >> np.uint64(15))) * np.uint64(0xA2C79B4D)) & low
        x = ((x ^ (x >> np.uint64(13))) * np.uint64(0x5BD0E6A7)) & low
        x ^= x >> np.uint64(16)
        bits = np.stack([x & np.uint64(0xFFFF), x >> np.uint64(16)], -1).reshape(-1, 256).astype(np.int32)
        c = np.clip(((y + (bits << 4)) >> 20) - (96 << 3), 1, 255)
        c = np.where(v.reshape(-1, 256) > 0, c, 0)
        self.vc = c.astype(np.uint8)
        self.v = (np.where(c > 0, ((c + (96 << 3)) << 20).astype(np.int32).view(f), f(0)) * self.vs[:, None]).reshape(-1)
        return m[: self.n], v[: self.n]


@pytest.mark.parametrize("dtype,master", [(F32, False), (BF16, False), (BF16, True), (F16, False), (F16, True)])
def test_32_bit_steps(dtype, master):
    params, g = _params(SHAPES, dtype)
    lr, betas, eps, wd = 3e-3, (0.9, 0.99), 1e-8, 0.1
    opt = AdamW(params, lr=lr, betas=betas, eps=eps, weight_decay=wd, master_weights=master)
    m = [torch.zeros(p.shape, device="cuda", dtype=torch.float64) for p in params]
    v = [torch.zeros(p.shape, device="cuda", dtype=torch.float64) for p in params]
    for t in range(1, 5):
        _grads(params, g)
        before = [(opt.state[p]["master"] if master else p).detach().double() for p in params]
        opt.step()
        for i, p in enumerate(params):
            grad, st = p.grad.double(), opt.state[p]
            terms = betas[0] * m[i].abs() + (1 - betas[0]) * grad.abs()
            m[i] = betas[0] * m[i] + (1 - betas[0]) * grad
            v[i] = betas[1] * v[i] + (1 - betas[1]) * grad**2
            # fp32 constants are off by 2^-24 too; errors of earlier steps come along.
            assert ((st["exp_avg"].double() - m[i]).abs() <= 5 * t * 2.0**-24 * terms).all()
            assert ((st["exp_avg_sq"].double() - v[i]).abs() <= 5 * t * 2.0**-24 * v[i]).all()
            m[i], v[i] = st["exp_avg"].double(), st["exp_avg_sq"].double()
            step = lr / (1 - betas[0] ** t) * m[i] / (v[i].sqrt() / (1 - betas[1] ** t) ** 0.5 + eps)
            want = before[i] * (1 - lr * wd) - step
            bound = 2.0**-21 * (want.abs() + step.abs())
            if master:
                assert ((st["master"].double() - want).abs() <= bound).all()
                assert torch.equal(p.detach(), st["master"].to(dtype))
            else:
                tiny = 2.0**-25 if dtype is F16 else 0.0
                assert ((p.detach().double() - want).abs() <= U[dtype] * want.abs() * (1 + 1e-3) + bound + tiny).all()
            assert st["step"] == t


def test_agrees_with_torch_adamw():
    params, g = _params(SHAPES, F32, 1)
    others = [torch.nn.Parameter(p.detach().clone()) for p in params]
    a, b = AdamW(params, lr=1e-2, weight_decay=0.05), torch.optim.AdamW(others, lr=1e-2, weight_decay=0.05)
    for _ in range(5):
        _grads(params, g, 1.0)
        for p, q in zip(params, others):
            q.grad = p.grad.clone()
        a.step(), b.step()
    for p, q in zip(params, others):
        torch.testing.assert_close(p, q, rtol=1e-5, atol=1e-6)


@pytest.mark.parametrize("dtype,master", [(F32, False), (BF16, False), (BF16, True), (F16, False)])
def test_8_bit_moments_bit_for_bit(dtype, master):
    params, g = _params(SHAPES, dtype, 2)
    lr, betas, eps, wd = 3e-3, (0.9, 0.999), 1e-8, 0.01
    opt = AdamW(params, lr=lr, betas=betas, eps=eps, weight_decay=wd, state_bits=8, master_weights=master, seed=5)
    plain = [_Numpy8(p.numel(), i, 5) for i, p in enumerate(params)]
    for t in range(1, 5):
        _grads(params, g)
        with torch.no_grad():
            params[-1].grad[:300] = 0  # a block of zeros, and some in the next
            params[-1].grad[600:700] *= 1e-6
        before = [(opt.state[p]["master"] if master else p).detach().double() for p in params]
        opt.step()
        flat_m, flat_v = opt.moments()
        at = 0
        for p, q, p0 in zip(params, plain, before):
            st = opt.state[p]
            m, v = q.step(p.grad.float().cpu().numpy().reshape(-1), *betas, t)
            n = p.numel()
            assert np.array_equal(st["exp_avg_scale"].cpu().numpy(), q.ms)
            assert np.array_equal(st["exp_avg_sq_scale"].cpu().numpy(), q.vs)
            assert np.array_equal(st["exp_avg_codes"].cpu().numpy().reshape(-1), q.mc.reshape(-1)[:n])
            assert np.array_equal(st["exp_avg_sq_codes"].cpu().numpy().reshape(-1), q.vc.reshape(-1)[:n])
            assert np.array_equal(flat_m[at: at + n].cpu().numpy(), q.m[:n])
            assert np.array_equal(flat_v[at: at + n].cpu().numpy(), q.v[:n])
            at += q.blocks * 256
            # The step itself uses the moments before they are rounded.
            m, v = (torch.from_numpy(x.astype(np.float64)).cuda().view(p.shape) for x in (m, v))
            step = lr / (1 - betas[0] ** t) * m / (v.sqrt() / (1 - betas[1] ** t) ** 0.5 + eps)
            want = p0 * (1 - lr * wd) - step
            got, u = (st["master"], U[F32]) if master else (p.detach(), U[dtype])
            tiny = 2.0**-25 if dtype is F16 else 0.0
            assert ((got.double() - want).abs() <= 1.001 * u * want.abs() + 2.0**-21 * (want.abs() + step.abs()) + tiny).all()


def test_8_bit_codes_are_near_and_unbiased():
    """Codes stand for their moments within half a step (first) or one (second), and the second's mean is kept."""
    n = 1 << 20
    p = torch.nn.Parameter(torch.zeros(n, device="cuda"))
    opt = AdamW([p], state_bits=8, betas=(0.0, 0.0), weight_decay=0.0)
    g = torch.Generator(device="cuda").manual_seed(3)
    p.grad = torch.randn(n, device="cuda", generator=g) * torch.exp(2 * torch.randn(n, device="cuda", generator=g))
    opt.step()
    m, v = (x.double() for x in opt.moments())
    x = p.grad.double()
    top = x.abs().view(-1, 256).amax(1, keepdim=True).expand(-1, 256).reshape(-1)
    assert ((m - x).abs() <= x.abs() / 16 * (1 + 1e-6) + top * 2.0**-15).all()
    assert ((v - x**2).abs() <= x**2 / 8 * (1 + 1e-6) + top**2 * 2.0**-30).all()
    # Each ratio has a standard deviation of at most 1/16: the mean's is that over 2^10, taken five times.
    ratio = (v / x**2)[x**2 > top**2 * 2.0**-28]
    assert abs(float(ratio.mean()) - 1) <= 5 / 16 / ratio.numel() ** 0.5


def test_8_bit_second_moment_follows_slow_changes():
    """With b2 = 0.999 the average of v follows a change of scale that no single step could show in 8 bits.

    Half the elements of each block see gradients of 1, half of 1/4; then they swap.  After
    1500 steps the exact v is 1 - 0.999^1500 (1 - 1/16) = 0.79 where it rose; the mean of the
    codes is held to it within 5 %: the codes' noise, about a quarter, over 2^13 elements is 0.3 %."""
    n = 1 << 14
    p = torch.nn.Parameter(torch.zeros(n, device="cuda"))
    opt = AdamW([p], lr=0.0, state_bits=8, betas=(0.9, 0.999), weight_decay=0.0)
    odd = torch.arange(n, device="cuda") % 2 == 1
    st = opt.state[p]
    p.grad = torch.where(odd, 1.0, 0.25)
    exact = None
    for t in range(3000):
        if t == 1500:
            p.grad = torch.where(odd, 0.25, 1.0)
        opt.step()
        e = p.grad[:2].double() ** 2
        exact = 0.001 * e if exact is None else 0.999 * exact + 0.001 * e
    assert st["step"] == 3000
    v = opt.moments()[1].double()
    for k in (0, 1):
        assert abs(float(v[k::2].mean() / exact[k]) - 1) <= 0.05


def test_non_finite_gradients_stay_in_their_block():
    for bits in (32, 8):
        p = torch.nn.Parameter(torch.ones(2000, device="cuda"))
        opt = AdamW([p], state_bits=bits)
        p.grad = torch.full((2000,), 0.5, device="cuda")
        p.grad[300], p.grad[700] = float("nan"), float("inf")
        opt.step()
        m, v = opt.moments()
        bad = torch.zeros(2048, dtype=torch.bool, device="cuda")
        bad[[300, 700]] = True
        if bits == 8:
            bad = bad.view(-1, 256).any(1).repeat_interleave(256)
        live = torch.arange(2048, device="cuda") < 2000
        assert torch.equal(~torch.isfinite(m) & live, bad & live) and torch.equal(~torch.isfinite(v) & live, bad & live)
        assert torch.isfinite(p[:300]).all() and torch.isfinite(p[1000:]).all() and torch.isnan(p[300])


def test_tiny_and_zero_gradients():
    """Moments below the 8-bit scales' range count as zero; nothing becomes NaN."""
    for size in (0.0, 1e-30, 1e-20, 1e-12):
        for bits in (32, 8):
            p = torch.nn.Parameter(torch.ones(1000, device="cuda"))
            opt = AdamW([p], state_bits=bits, lr=1e-3, weight_decay=0.0)
            for _ in range(3):
                p.grad = torch.full((1000,), size, device="cuda")
                opt.step()
            assert torch.isfinite(p).all() and float((p.detach() - 1).abs().max()) <= 4e-3


def test_groups_missing_gradients_and_closure():
    """Groups have their own settings; a parameter without a gradient keeps its value, state and step count."""
    params, g = _params([(50,), (60, 3), (70,), (300, 5)], BF16, 4)
    extra, _ = _params([(33,), (999,)], F32, 5)
    opt = AdamW([{"params": params, "state_bits": 8, "lr": 1e-2}, {"params": extra, "weight_decay": 0.0}], lr=1e-3,
                seed=1)
    _grads(params + extra, g)
    opt.step()
    params[1].grad = None
    kept = params[1].detach().clone(), copy.deepcopy(opt.state[params[1]])
    opt.step()
    assert [opt.state[p]["step"] for p in params] == [2, 1, 2, 2]
    assert torch.equal(params[1], kept[0])
    for name, value in kept[1].items():
        assert value == 1 if name == "step" else torch.equal(opt.state[params[1]][name], value)
    _grads(params + extra, g)
    opt.step()  # 3, 2, 3, 3: two launches
    assert [opt.state[p]["step"] for p in params] == [3, 2, 3, 3]
    single, _ = _params([(60, 3)], BF16, 4)
    loss = opt.step(lambda: torch.tensor(7.0))
    assert float(loss) == 7.0
    for p in params + extra:
        p.grad = None
    before = [p.detach().clone() for p in params]
    opt.step()
    assert all(torch.equal(a, b) for a, b in zip(params, before))
    # torch's schedulers drive it.
    sched = torch.optim.lr_scheduler.LambdaLR(opt, lambda t: 0.5**t)
    _grads(params + extra, g)
    opt.step(), sched.step()
    assert opt.param_groups[0]["lr"] == 5e-3


@pytest.mark.parametrize("bits,master", [(32, False), (8, False), (8, True), (32, True)])
def test_state_dict_continues_the_run(bits, master, tmp_path):
    params, g = _params(SHAPES, BF16, 6)
    opt = AdamW(params, lr=1e-2, state_bits=bits, master_weights=master, seed=9)
    for _ in range(2):
        _grads(params, g)
        opt.step()
    torch.save(opt.state_dict(), tmp_path / "opt.pt")
    twins = [torch.nn.Parameter(p.detach().clone()) for p in params]
    other = AdamW(twins, lr=5.0, state_bits=bits, master_weights=master, seed=9)
    other.load_state_dict(torch.load(tmp_path / "opt.pt"))
    assert other.param_groups[0]["lr"] == 1e-2
    for _ in range(2):
        _grads(params, g)
        for p, q in zip(params, twins):
            q.grad = p.grad.clone()
        opt.step(), other.step()
    for p, q in zip(params, twins):
        assert torch.equal(p, q)
        for name, value in opt.state[p].items():
            assert value == other.state[q][name] if name == "step" else torch.equal(value, other.state[q][name])
    with pytest.raises(ValueError, match="state_bits"):
        AdamW(twins, state_bits=40 - bits, master_weights=master).load_state_dict(opt.state_dict())
    with pytest.raises(ValueError, match="size"):
        AdamW(twins[:3], state_bits=bits, master_weights=master).load_state_dict(opt.state_dict())


def test_many_tensors_misaligned_views_and_layouts():
    """More tensors than one launch holds; views at odd offsets; gradients of other strides."""
    flat = torch.randn(1000 * 130 + 1, device="cuda")
    gflat = torch.randn(1000 * 130 + 3, device="cuda")
    params = [torch.nn.Parameter(flat[1 + 130 * i: 1 + 130 * i + 129]) for i in range(1000)]
    for i, p in enumerate(params):
        p.grad = gflat[3 + 130 * i: 3 + 130 * i + 129]
    want = flat.clone()
    opt = AdamW(params, lr=0.1, weight_decay=0.0)
    opt.step()
    moved = flat != want
    assert not bool(moved[0]) and not moved[1:].view(1000, 130)[:, 129].any()  # between the views nothing is written
    torch.testing.assert_close(flat[1:].view(1000, 130)[:, :129],
                               (want - 0.1 * gflat[2:] / (gflat[2:].abs() + 1e-8))[1:].view(1000, 130)[:, :129], rtol=1e-4, atol=1e-4)
    a, b = (torch.nn.Parameter(torch.ones(64, 96, device="cuda", dtype=BF16)) for _ in range(2))
    grad = torch.randn(96, 64, device="cuda").bfloat16()
    a.grad, b.grad = grad.t(), grad.t().contiguous()
    AdamW([a], state_bits=8).step(), AdamW([b], state_bits=8).step()
    assert torch.equal(a, b)


def test_elements_beyond_32_bit_offsets():
    n = (1 << 31) + 777
    p = torch.nn.Parameter(torch.zeros(n, device="cuda", dtype=BF16))
    p.grad = torch.zeros(n, device="cuda", dtype=BF16)
    p.grad[-1000:] = torch.randn(1000, device="cuda").bfloat16()
    opt = AdamW([p], lr=0.5, state_bits=8, weight_decay=0.0)
    opt.step()
    assert torch.count_nonzero(p[: 1 << 20]) == 0
    want = -0.5 * torch.sign(p.grad[-1000:].float())
    torch.testing.assert_close(p[-1000:].float(), want, rtol=1e-2, atol=1e-2)
    st = opt.state[p]
    last = st["exp_avg_codes"][-777:]
    assert torch.equal(last > 127, p.grad[-777:] < 0) and float(st["exp_avg_scale"][-1]) > 0


def test_other_stream():
    params, g = _params(SHAPES, BF16, 8)
    twins = [torch.nn.Parameter(p.detach().clone()) for p in params]
    a, b = AdamW(params, state_bits=8), AdamW(twins, state_bits=8)
    _grads(params, g)
    for p, q in zip(params, twins):
        q.grad = p.grad.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        b.step()
    torch.cuda.current_stream().wait_stream(side)
    a.step()
    assert all(torch.equal(p, q) for p, q in zip(params, twins))


def test_refusals():
    p = torch.nn.Parameter(torch.zeros(8, 8, device="cuda"))
    for bad in (dict(lr=-1.0), dict(betas=(0.9, 1.0)), dict(eps=-1e-8), dict(weight_decay=float("nan")), dict(state_bits=16)):
        with pytest.raises(ValueError):
            AdamW([p], **bad)
    with pytest.raises(RuntimeError, match="CUDA"):
        AdamW([torch.nn.Parameter(torch.zeros(3))])
    with pytest.raises(ValueError, match="dtype"):
        AdamW([torch.nn.Parameter(torch.zeros(3, device="cuda", dtype=torch.float64))])
    with pytest.raises(ValueError, match="contiguous"):
        AdamW([torch.nn.Parameter(torch.zeros(4, 6, device="cuda").t())])
    with pytest.raises(ValueError, match="one dtype"):
        AdamW([p, torch.nn.Parameter(torch.zeros(3, device="cuda").half())])
    opt = AdamW([p])
    p.grad = torch.ones(8, 8, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="graph"):
        with torch.cuda.graph(graph):
            opt.step()
