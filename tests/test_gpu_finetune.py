"""The fine-tuning step on native norms, loss and optimizer against the same model with
torch's: loss and adapter gradients of one step in fp32 (1e-5 relative for the loss, 1e-4
normwise for the gradients, as for the model itself), and training in bf16."""

import copy

import pytest
import torch
from torch import nn

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _device_error_stays_clear():
    from dorafactors_b200 import _native

    yield
    assert _native.device_error(reset=True) == 0


def _model(dtype, vocab=1000):
    from dorafactors_b200.model import add_dora, build_llama, llama_config

    cfg = llama_config(layers=2, hidden=256, ffn=512, heads=4, kv_heads=2, vocab=vocab, max_pos=256)
    cfg._attn_implementation = "eager"
    model = build_llama(cfg, "cuda", dtype=dtype, seed=1)
    return model, add_dora(model, r=8, scaling=2.0, seed=2)


def test_step_matches_torch():
    from dorafactors_b200 import _native
    from dorafactors_b200.finetune import causal_lm_loss, use_native_norms
    from dorafactors_b200.optim import AdamW

    old = torch.backends.cuda.matmul.allow_tf32
    torch.backends.cuda.matmul.allow_tf32 = False
    try:
        model, params = _model(torch.float32)
        ref = copy.deepcopy(model)
        names = [n for n, p in model.named_parameters() if p.requires_grad]
        ref_params = [dict(ref.named_parameters())[n] for n in names]
        params = [dict(model.named_parameters())[n] for n in names]
        assert use_native_norms(model) == 2 * 2 + 1
        ids = torch.randint(0, 1000, (2, 64), device="cuda", generator=torch.Generator("cuda").manual_seed(3))
        labels = ids.clone()
        labels[0, :20] = -100
        launches = _native.launch_count()
        loss, out = causal_lm_loss(model(input_ids=ids).logits, labels, top_k=3)
        loss.backward()
        assert _native.launch_count() > launches
        ref_loss = ref(input_ids=ids, labels=labels).loss
        ref_loss.backward()
        torch.testing.assert_close(loss, ref_loss, rtol=1e-5, atol=0)
        assert out.top_indices.shape == (2, 64, 3) and torch.count_nonzero(out.logprobs[0, :19]) == 0
        for n, p, q in zip(names, params, ref_params):
            num, den = (p.grad.double() - q.grad.double()).norm(), q.grad.double().norm().clamp_min(1e-30)
            assert float(num / den) <= 1e-4, (n, float(num / den))
        # The optimizers on the same gradients.
        for p, q in zip(params, ref_params):
            q.grad.copy_(p.grad)
        AdamW(params, lr=1e-3, weight_decay=0.1).step()
        torch.optim.AdamW(ref_params, lr=1e-3, weight_decay=0.1).step()
        for p, q in zip(params, ref_params):
            torch.testing.assert_close(p, q, rtol=1e-5, atol=1e-7)
    finally:
        torch.backends.cuda.matmul.allow_tf32 = old


@pytest.mark.parametrize("bits,master", [(32, True), (8, True), (8, False)])
def test_training_learns_a_batch(bits, master):
    """A repeated batch: its loss falls from about ln 1000 by a third within 60 steps, as with 32-bit moments."""
    from dorafactors_b200.finetune import train_step, use_native_norms
    from dorafactors_b200.optim import AdamW

    model, params = _model(torch.bfloat16)
    use_native_norms(model)
    opt = AdamW(params, lr=5e-3, state_bits=bits, master_weights=master, weight_decay=0.0)
    ids = torch.randint(0, 1000, (2, 64), device="cuda", generator=torch.Generator("cuda").manual_seed(4))
    losses = [float(train_step(model, ids, opt)[0]) for _ in range(60)]
    assert losses[-1] < losses[0] * 2 / 3, losses[::10]


def test_native_norms_replace_layer_norms_too():
    from dorafactors_b200.finetune import use_native_norms
    from dorafactors_b200.norms import LayerNorm

    net = nn.Sequential(nn.Linear(64, 96), nn.LayerNorm(96), nn.Sequential(nn.LayerNorm(96, bias=False))).cuda()
    x = torch.randn(5, 64, device="cuda")
    before, keys = net(x), list(net.state_dict())
    assert use_native_norms(net) == 2 and isinstance(net[1], LayerNorm) and list(net.state_dict()) == keys
    torch.testing.assert_close(net(x), before, rtol=1e-5, atol=1e-5)
    assert use_native_norms(net) == 0


def test_entropy_term():
    """d(-mean lp - w mean H) against autograd through log_softmax in 64 bits."""
    from dorafactors_b200.finetune import causal_lm_loss

    g = torch.Generator("cuda").manual_seed(5)
    logits = torch.randn(2, 9, 50, device="cuda", generator=g).requires_grad_()
    labels = torch.randint(0, 50, (2, 9), device="cuda", generator=g)
    loss, _ = causal_lm_loss(logits, labels, entropy_weight=0.3)
    (grad,) = torch.autograd.grad(loss, logits)
    d = logits.detach().double().requires_grad_()
    logp = torch.log_softmax(d, -1)
    lp = logp[:, :-1].gather(-1, labels[:, 1:, None])[..., 0]
    h = -(logp.exp() * logp).sum(-1)[:, :-1]
    ref = -(lp.sum() + 0.3 * h.sum()) / 16
    (ref_grad,) = torch.autograd.grad(ref, d)
    torch.testing.assert_close(loss.double(), ref, rtol=1e-5, atol=1e-6)
    torch.testing.assert_close(grad.double(), ref_grad, rtol=1e-4, atol=1e-6)
