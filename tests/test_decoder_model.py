"""The decoder on the package's operators against the decoder in eager torch, on CPU tensors and gloo ranks."""
import pytest
import torch
import torch.distributed as dist

from distributed_helpers import run_distributed
from soap_tp_b200 import ops
from soap_tp_b200.models.llama_tp import LlamaConfig, LlamaTP
from soap_tp_b200.train import parse_args, train

SWITCHES = dict(fused_loss=True, fused_norms=True)


def _model(seed=3, **config):
    model = LlamaTP(LlamaConfig.tiny(**config), dtype=torch.float32, device="cpu", seed=seed)
    generator = torch.Generator().manual_seed(seed)
    with torch.no_grad():      # norms and gates that do something
        for name, p in model.named_parameters():
            if p.ndim == 1:
                p.add_(0.1 * torch.randn(p.shape, generator=generator))
    return model


def _tokens(vocabulary=64):
    tokens = torch.randint(0, vocabulary, (2, 9), generator=torch.Generator().manual_seed(1))
    return tokens[:, :-1], tokens[:, 1:]


def _loss_and_gradients(model, **switches):
    for name, value in switches.items():
        setattr(model, name, value)
    loss = model(*_tokens())
    return loss.detach(), torch.autograd.grad(loss, list(model.parameters()))


CONFIGS = [dict(), dict(norm_after=True, gated_residual=True, residual_scale=0.5), dict(gated_residual=True)]


@pytest.mark.parametrize("config", CONFIGS)
@pytest.mark.parametrize("checkpointed", [False, True])
def test_fused_norms_and_loss_change_roundings_only(config, checkpointed):
    # fp32 against fp32: sums of up to 64 terms in another order through two layers, a few hundred half steps of 2^-24
    loss, grads = _loss_and_gradients(_model(**config))
    fused_loss, fused_grads = _loss_and_gradients(_model(**config), checkpoint_activations=checkpointed, **SWITCHES)
    assert abs(float(loss - fused_loss)) <= 400 * 2.0 ** -24 * float(loss)
    for a, b in zip(grads, fused_grads):
        assert float((a - b).norm()) <= 400 * 2.0 ** -24 * float(a.norm())


@pytest.mark.parametrize("fused", [False, True])
def test_eight_bits_change_the_backward_pass_only(fused):
    switches = SWITCHES if fused else {}
    loss, _ = _loss_and_gradients(_model(), **switches)
    kept, grads = _loss_and_gradients(_model(), checkpoint_activations=True, checkpoint_bits=8, mlp_bits=8, **switches)
    assert abs(float(loss - kept)) <= 400 * 2.0 ** -24 * float(loss)
    assert all(bool(torch.isfinite(g).all()) and bool(g.any()) for g in grads)


def test_gradients_of_a_checkpointed_block_are_those_at_its_kept_input():
    model = _model(norm_after=True, gated_residual=True)
    block = model.blocks[0]
    x = torch.randn(2, 8, 32, generator=torch.Generator().manual_seed(5)).requires_grad_()
    from soap_tp_b200.models.llama_tp import rope_tables

    cos, sin = rope_tables(8, 8, 10000.0, "cpu")
    grad = torch.randn(2, 8, 32, generator=torch.Generator().manual_seed(6))
    parameters = list(block.parameters())
    got = torch.autograd.grad(ops.checkpoint8(block.fused_from_sum, x, cos, sin, parameters=parameters), [x, *parameters], grad)
    kept = ops.unpack8(ops.pack8(x)).requires_grad_()
    expected = torch.autograd.grad(block.fused_from_sum(kept, cos, sin), [kept, *parameters], grad)
    for a, b in zip(got, expected):
        assert torch.equal(a, b)


def test_switches_are_checked():
    model = _model()
    with pytest.raises(ValueError):
        model.mlp_bits = 4
    model.checkpoint_bits = 4
    with pytest.raises(ValueError):
        model(*_tokens())
    with pytest.raises(SystemExit):
        parse_args(["--checkpoint-bits", "8"])


def _ranks_case(rank, world):
    for config in CONFIGS[:2]:
        loss, grads = _loss_and_gradients(_model(**config))
        fused_loss, fused_grads = _loss_and_gradients(_model(**config), **SWITCHES)
        values = [torch.zeros(()) for _ in range(world)]
        dist.all_gather(values, fused_loss)
        assert all(torch.allclose(values[0], v, rtol=1e-6) for v in values)
        assert abs(float(loss - fused_loss)) <= 400 * 2.0 ** -24 * float(loss)
        for a, b in zip(grads, fused_grads):
            assert float((a - b).norm()) <= 400 * 2.0 ** -24 * float(a.norm())
    summary = train(parse_args(["--preset", "tiny", "--device", "cpu", "--steps", "3", "--global-batch", "2", "--block-size", "8",
                                "--precondition-frequency", "2", "--basis-implementation", "eigh", "--fused-loss", "--fused-norms",
                                "--checkpoint-activations", "--checkpoint-bits", "8", "--mlp-bits", "8"]))
    assert all(loss == loss for loss in summary["losses"])


def test_fused_decoder_on_two_ranks():
    run_distributed(_ranks_case, 2)
