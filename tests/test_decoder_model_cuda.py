"""A decoder's training step on the package's operators, on the GPU: loss, norms and 8-bit activations together."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def _models(**config):
    from soap_tp_b200.models.llama_tp import LlamaConfig, LlamaTP

    cfg = LlamaConfig.tiny(vocab_size=1000, hidden_size=256, intermediate_size=680, num_heads=4, num_kv_heads=2, max_seq_len=64, **config)
    model = LlamaTP(cfg, dtype=torch.bfloat16, device="cuda", seed=1)
    exact = LlamaTP(cfg, dtype=torch.float64, device="cuda", seed=1)
    with torch.no_grad():
        for p, q in zip(model.parameters(), exact.parameters()):
            q.copy_(p)
    return model, exact


def _gradients(model, tokens, **switches):
    for name, value in switches.items():
        setattr(model, name, value)
    loss = model(tokens[:, :-1], tokens[:, 1:])
    return float(loss), torch.autograd.grad(loss, list(model.parameters()))


def _error(grads, exact):
    return max(float((a.double() - b.double()).norm() / b.double().norm()) for a, b in zip(grads, exact))


@pytest.mark.parametrize("config", [dict(), dict(norm_after=True, gated_residual=True, residual_scale=0.5)])
@pytest.mark.parametrize("checkpointed", [False, True])
def test_fused_step_is_as_near_to_64_bits_as_the_eager_one(config, checkpointed):
    from soap_tp_b200.engine import kernels

    model, exact = _models(**config)
    tokens = torch.randint(0, 1000, (3, 65), generator=torch.Generator("cuda").manual_seed(2), device="cuda")
    loss, grads = _gradients(exact, tokens)
    _, eager = _gradients(model, tokens)
    fused_loss, fused = _gradients(model, tokens, fused_loss=True, fused_norms=True, checkpoint_activations=checkpointed)
    kernels.check_status()
    # the products' roundings are common to both; the operators round less often than the eager formulas that they replace
    assert _error(fused, grads) <= 1.5 * _error(eager, grads) + 2.0 ** -8
    assert abs(fused_loss - loss) <= 2.0 ** -8 * loss


def test_eight_bit_activations_leave_the_loss_and_nearly_the_gradients():
    from soap_tp_b200.engine import kernels

    model, exact = _models()
    tokens = torch.randint(0, 1000, (3, 65), generator=torch.Generator("cuda").manual_seed(2), device="cuda")
    _, grads = _gradients(exact, tokens)
    loss, fused = _gradients(model, tokens, fused_loss=True, fused_norms=True)
    kept_loss, kept = _gradients(model, tokens, checkpoint_activations=True, checkpoint_bits=8, mlp_bits=8)
    kernels.check_status()
    assert abs(kept_loss - loss) <= 2.0 ** -8 * loss
    # a kept value is off by half a step, 1 / 254 of its group's largest; two layers keep three tensors each, and a group's largest is some
    # three times its root mean square: 6 * 3 / 254 if all of it added up
    assert _error(kept, grads) <= 1.5 * _error(fused, grads) + 18 / 254


def test_training_on_the_operators():
    from soap_tp_b200 import train as train_module
    from soap_tp_b200.engine import kernels

    args = train_module.parse_args(["--preset", "tiny", "--steps", "6", "--precondition-frequency", "3", "--global-batch", "4", "--block-size", "16",
                                    "--lr", "1e-2", "--fused-loss", "--fused-norms", "--checkpoint-activations", "--checkpoint-bits", "8",
                                    "--mlp-bits", "8"])
    summary = train_module.train(args)
    kernels.check_status()
    assert len(summary["losses"]) == 6 and all(math.isfinite(v) for v in summary["losses"])
    assert abs(summary["losses"][0] - math.log(64)) < 0.5
