"""Norms, token log probabilities and AdamW without a GPU: argument checks of the C
entry points (all return before any CUDA call) and of the Python layer."""

import ctypes

import numpy as np
import pytest
import torch


@pytest.fixture(scope="module")
def lib():
    from dorafactors_b200 import _native
    from dorafactors_b200.build import build

    build()
    return _native.load_library()


vp = ctypes.c_void_p
P = [vp(1 << (12 + i)) for i in range(12)]  # addresses that are never used
N = None


def test_norm_arguments(lib):
    f = lib.dora_layer_norm_fwd
    assert f(P[0], 8, N, N, 2, 1e-5, P[1], N, N, -1, 8, 2, N) == 1
    assert f(P[0], 7, N, N, 2, 1e-5, P[1], N, N, 4, 8, 2, N) == 1  # row stride below the width
    assert f(P[0], 8, N, N, 1, 1e-5, P[1], N, N, 4, 8, 2, N) == 1  # fp16 weight with bf16 rows
    assert f(P[0], 8, N, N, 2, -1.0, P[1], N, N, 4, 8, 2, N) == 1
    assert f(P[0], 8, N, N, 2, float("nan"), P[1], N, N, 4, 8, 2, N) == 1
    assert f(P[0], 8, N, N, 2, 1e-5, P[0], N, N, 4, 8, 2, N) == 1  # in place
    assert f(N, 8, N, N, 2, 1e-5, N, N, N, 0, 8, 2, N) == 0
    assert lib.dora_rms_norm_fwd(N, 8, N, 2, 1e-5, P[1], N, 4, 8, 2, N) == 1
    b = lib.dora_layer_norm_bwd
    assert b(P[0], 8, P[1], 8, N, 2, N, P[3], P[4], N, N, N, 0, 4, 8, 2, N) == 1  # no mean
    assert b(P[0], 8, P[1], 8, N, 2, P[2], P[3], P[0], N, N, N, 0, 4, 8, 2, N) == 1  # dx over dy
    assert b(P[0], 8, P[1], 8, N, 2, P[2], P[3], P[4], P[5], N, N, 0, 4, 8, 2, N) == 3  # no workspace
    assert b(P[0], 8, P[1], 8, N, 2, P[2], P[3], N, N, N, N, 0, 4, 8, 2, N) == 0  # nothing asked for
    assert lib.dora_rms_norm_bwd(P[0], 7, P[1], 8, N, 2, P[3], P[4], N, N, 0, 4, 8, 2, N) == 1
    assert lib.dora_layer_norm_bwd_workspace_size(16384, 8192) > 0
    assert lib.dora_layer_norm_bwd_workspace_size(4, 0) == 0


def test_logprobs_arguments(lib):
    def f(rows=4, vocab=8, ld=8, temperature=1.0, k=0, dtype=2, logits=P[0]):
        return lib.dora_token_logprobs_fwd(logits, ld, P[1], -100, temperature, P[2], P[3], N, k, N, N, rows, vocab, dtype, N)

    assert f(rows=-1) == 1 and f(vocab=0) == 1 and f(ld=7) == 1 and f(dtype=5) == 1 and f(logits=N) == 1
    assert f(temperature=0.0) == 1 and f(temperature=float("nan")) == 1 and f(temperature=float("inf")) == 1
    assert f(k=9) == 1 and f(k=-1) == 1 and f(k=65, vocab=100, ld=100) == 2 and f(k=2) == 1  # no place for the top
    assert f(rows=0, logits=N) == 0

    def b(ldd=8, entropy=N, g_entropy=N, d=P[6]):
        return lib.dora_token_logprobs_bwd(P[0], 8, P[1], -100, 1.0, P[2], entropy, P[3], g_entropy, N, d, ldd, 4, 8, 2, N)

    assert b(ldd=7) == 1 and b(g_entropy=P[4]) == 1 and b(d=N) == 1 and b(ldd=16, d=P[0]) == 1


def test_adamw_arguments(lib):
    from dorafactors_b200 import _native

    t = np.zeros(2, dtype=_native.ADAMW_TENSOR)
    assert t.itemsize == 72
    for name in ("param", "grad", "exp_avg", "exp_avg_sq"):
        t[name] = 4096
    t["numel"] = 8

    def f(count=2, dtype=0, bits=32, lr=1e-3, b1=0.9, b2=0.999, eps=1e-8, wd=0.0, step=1):
        return lib.dora_adamw_step(t.ctypes.data, count, dtype, bits, lr, b1, b2, eps, wd, step, N)

    nan = float("nan")
    for bad in (dict(count=-1), dict(dtype=3), dict(bits=16), dict(lr=-1.0), dict(lr=nan), dict(b1=1.0), dict(b2=-0.1),
                dict(eps=nan), dict(wd=-1.0), dict(step=0)):
        assert f(**bad) == 1, bad
    assert f(count=0) == 0
    assert f(bits=8) == 1  # no scales
    t["master"][0] = 4096
    assert f(dtype=0) == 1 and f(dtype=2) == 1  # a master of fp32; one of two tensors with a master
    t["master"], t["grad"][1] = 0, 0
    assert f() == 1
    t["numel"][1] = -1
    assert f() == 1
    t["numel"] = 0
    assert f() == 0  # empty tensors have nothing to do
    assert lib.dora_adamw_decode(P[0], P[1], P[2], P[3], P[4], P[5], -1, N) == 1
    assert lib.dora_adamw_decode(N, N, N, N, N, N, 0, N) == 0
    assert lib.dora_adamw_decode(P[0], N, P[2], P[3], P[4], P[5], 8, N) == 1


def test_cpu_tensors_fail_loudly():
    from dorafactors_b200.logprobs import token_logprobs, token_logprobs_backward
    from dorafactors_b200.norms import LayerNorm, RMSNorm
    from dorafactors_b200.optim import AdamW

    x, t = torch.randn(4, 16), torch.zeros(4, dtype=torch.int64)
    for f in (LayerNorm(16), RMSNorm(16)):
        with pytest.raises(RuntimeError, match="CUDA"):
            f(x)
    with pytest.raises(RuntimeError, match="CUDA"):
        token_logprobs(x, t)
    with pytest.raises(RuntimeError, match="CUDA"):
        token_logprobs_backward(x[:, 0], None, None, x, t, x[:, 0])
    with pytest.raises(RuntimeError, match="CUDA"):
        AdamW([torch.nn.Parameter(x)])
    with pytest.raises(ValueError):
        AdamW([])


def test_modules_have_torch_parameter_names():
    from dorafactors_b200.norms import LayerNorm, RMSNorm

    assert list(LayerNorm(8).state_dict()) == list(torch.nn.LayerNorm(8).state_dict())
    assert list(LayerNorm(8, bias=False).state_dict()) == ["weight"]
    assert list(RMSNorm(8).state_dict()) == list(torch.nn.RMSNorm(8).state_dict())
    assert not list(RMSNorm(8, elementwise_affine=False).parameters())


def test_rows_of_keeps_rows_of_wider_buffers():
    from dorafactors_b200 import _native

    base = torch.randn(6, 40)
    for x, kept in ((base, True), (base[:, :32], True), (base[::2, 4:20], True), (base.view(2, 3, 40)[..., :8], True),
                    (base.t(), False), (base[:, ::2], False), (base[0].expand(5, 40), False),
                    (base.view(2, 3, 40)[:, :2], False)):
        data, rows, cols, ld = _native.rows_of(x)
        assert (rows, cols) == (x.shape[:-1].numel(), x.shape[-1])
        assert (data.data_ptr() == x.data_ptr() and ld >= cols) is kept
        assert torch.equal(data.as_strided((rows, cols), (ld, 1), data.storage_offset()), x.reshape(rows, cols))
