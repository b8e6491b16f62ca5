"""Operators of a decoder's training step on CPU tensors: definitions, gradients against differences, refusals, several ranks."""
import pytest
import torch
import torch.distributed as dist

from decoder_bounds import IGNORED
from distributed_helpers import run_distributed
from soap_tp_b200 import ops

D = torch.float64


def _rand(*shape, seed=0, dtype=D):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed), dtype=D).to(dtype)


@pytest.mark.parametrize("reduction", ["none", "sum", "mean"])
def test_cross_entropy_against_logits(reduction):
    hidden, weight = _rand(3, 5, 7).requires_grad_(), _rand(11, 7, seed=1).requires_grad_()
    targets = torch.randint(0, 11, (3, 5), generator=torch.Generator().manual_seed(2))
    targets[1, 2:] = IGNORED
    loss = ops.linear_cross_entropy(hidden, weight, targets, reduction=reduction)
    expected = torch.nn.functional.cross_entropy((hidden @ weight.t()).flatten(0, 1), targets.flatten(), reduction=reduction)
    if reduction == "none":
        expected = expected.view(3, 5)
    assert loss.shape == expected.shape and torch.allclose(loss, expected, rtol=0, atol=1e-13)
    up = torch.rand_like(loss)
    for a, b in zip(torch.autograd.grad(loss, (hidden, weight), up), torch.autograd.grad(expected, (hidden, weight), up)):
        assert torch.allclose(a, b, rtol=0, atol=1e-13)


def test_cross_entropy_gradients_against_differences():
    hidden, weight = _rand(4, 3).requires_grad_(), _rand(6, 3, seed=1).requires_grad_()
    targets = torch.tensor([5, IGNORED, 0, 0])
    for reduction in ("none", "mean"):
        assert torch.autograd.gradcheck(lambda a, b: ops.linear_cross_entropy(a, b, targets, reduction=reduction), (hidden, weight))


def test_cross_entropy_without_counted_tokens():
    hidden, weight = _rand(2, 3).requires_grad_(), _rand(4, 3, seed=1).requires_grad_()
    loss = ops.linear_cross_entropy(hidden, weight, torch.full((2,), IGNORED))
    assert float(loss) == 0.0 and all(not g.any() for g in torch.autograd.grad(loss, (hidden, weight)))
    empty = ops.linear_cross_entropy(hidden[:0], weight, torch.zeros(0, dtype=torch.int64))
    assert float(empty) == 0.0 and all(not g.any() for g in torch.autograd.grad(empty, (hidden, weight)))
    assert ops.linear_cross_entropy(hidden[:0], weight, torch.zeros(0, dtype=torch.int64), reduction="none").shape == (0,)


@pytest.mark.parametrize("change,error", [
    (dict(reduction="max"), ValueError), (dict(targets=torch.zeros(3, dtype=torch.int64)), ValueError),
    (dict(targets=torch.zeros(2)), TypeError), (dict(weight=_rand(4, 5)), ValueError), (dict(weight=_rand(4, 3).float()), TypeError),
    (dict(weight=_rand(0, 3)), ValueError), (dict(weight=_rand(3)), ValueError), (dict(workspace_bytes=0), ValueError),
    (dict(targets=torch.tensor([0, 4])), IndexError), (dict(targets=torch.tensor([0, -1])), IndexError),
    (dict(hidden=torch.zeros(2, 3, dtype=torch.int64), weight=torch.zeros(4, 3, dtype=torch.int64)), TypeError)])
def test_cross_entropy_refusals(change, error):
    arguments = dict(hidden=_rand(2, 3), weight=_rand(4, 3), targets=torch.tensor([0, 1])) | change
    with pytest.raises(error):
        ops.linear_cross_entropy(arguments.pop("hidden"), arguments.pop("weight"), arguments.pop("targets"), **arguments)


def _sharded_case(rank, world):
    hidden = _rand(5, 7).requires_grad_()
    full = _rand(6, 7, seed=1)
    targets = torch.tensor([0, 5, IGNORED, 3, 2])
    whole = full.clone().requires_grad_()
    expected = ops.linear_cross_entropy(hidden, whole, targets)
    g_hidden, g_weight = torch.autograd.grad(expected, (hidden, whole))
    per_rank = 6 // world
    mine = full[rank * per_rank:(rank + 1) * per_rank].clone().requires_grad_()
    loss = ops.linear_cross_entropy(hidden, mine, targets, group=dist.group.WORLD)
    assert torch.allclose(loss, expected, rtol=0, atol=1e-13)
    d_hidden, d_weight = torch.autograd.grad(loss, (hidden, mine))
    assert torch.allclose(d_hidden, g_hidden, rtol=0, atol=1e-13)
    assert torch.allclose(d_weight, g_weight[rank * per_rank:(rank + 1) * per_rank], rtol=0, atol=1e-13)


def test_cross_entropy_over_two_ranks():
    run_distributed(_sharded_case, 2)


@pytest.mark.parametrize("after,gated,normed", [(a, g, n) for a in (0, 1) for g in (0, 1) for n in (0, 1)])
def test_residual_norm_gradients_against_differences(after, gated, normed):
    x, b = _rand(3, 5).requires_grad_(), _rand(3, 5, seed=1).requires_grad_()
    vectors = [(1 + 0.1 * _rand(5, seed=2 + i)).requires_grad_() if on else None for i, on in enumerate((normed, after, gated))]

    def f(x, b, *_):
        return tuple(t for t in ops.residual_norm(x, b, vectors[0], branch_weight=vectors[1], gate=vectors[2], scale=0.7) if t is not None)

    assert torch.autograd.gradcheck(f, (x, b, *(v for v in vectors if v is not None)))


def test_rms_norm_definition():
    x, w = _rand(4, 9), _rand(9, seed=1)
    assert torch.allclose(ops.rms_norm(x, w, eps=1e-3), x / (x.square().mean(-1, keepdim=True) + 1e-3).sqrt() * w, rtol=1e-14, atol=0)
    assert ops.rms_norm(x[:0], w).shape == (0, 9)


@pytest.mark.parametrize("change,error", [
    (dict(branch=_rand(3, 4)), ValueError), (dict(branch=_rand(3, 5).float()), ValueError), (dict(branch=None), ValueError),
    (dict(weight=_rand(4)), ValueError), (dict(weight=_rand(5, dtype=torch.float16)), TypeError), (dict(eps=-1.0), ValueError),
    (dict(weight=_rand(5), gate=_rand(5, dtype=torch.float32)), TypeError), (dict(scale=float("nan")), ValueError),
    (dict(x=torch.zeros(3, 5, dtype=torch.int32)), TypeError), (dict(x=_rand(3, 0), branch=_rand(3, 0)), ValueError)])
def test_residual_norm_refusals(change, error):
    arguments = dict(x=_rand(3, 5), branch=_rand(3, 5)) | change
    with pytest.raises(error):
        ops.residual_norm(arguments.pop("x"), arguments.pop("branch"), arguments.pop("weight", None), **arguments)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [1, 63, 64, 65, 200])
def test_pack8_is_off_by_half_a_step_at_most(dtype, dim):
    x = (_rand(2, 3, dim) * 10).to(dtype)
    packed = ops.pack8(x)
    back = ops.unpack8(packed)
    assert back.shape == x.shape and back.dtype == dtype and packed.values.dtype == torch.int8
    step = packed.scales.repeat_interleave(64, dim=1)[:, :dim].view(x.shape).double()
    # half a step; the quotient and the product have 127 * 2^-23 of a step of rounding; the result is rounded to its type
    bound = step * (0.5 + 2.0 ** -15) + torch.finfo(dtype).eps / 2 * (x.double().abs() + step)
    assert bool(((back.double() - x.double()).abs() <= bound).all())


def test_pack8_of_special_values():
    x = torch.zeros(4, 130)
    x[1, 3], x[2, 70], x[3, 129] = float("inf"), float("nan"), 2.0 ** -140
    back = ops.unpack8(ops.pack8(x))
    assert not back[0].any() and bool(back[1, :64].isnan().all()) and not back[1, 64:].any()
    assert bool(back[2, 64:128].isnan().all()) and not back[2, :64].any() and float(back[3, 129]) == 0.0
    assert ops.unpack8(ops.pack8(x[:0])).shape == (0, 130)


def test_pack8_refusals():
    packed = ops.pack8(torch.randn(2, 70))
    for change in (dict(shape=torch.Size((2, 71 + 8))), dict(shape=torch.Size((3, 70))), dict(scales=packed.scales[:, :1])):
        with pytest.raises(ValueError):
            ops.unpack8(packed._replace(**change))
    for change in (dict(dtype=torch.int32), dict(values=packed.values.to(torch.int32))):
        with pytest.raises(TypeError):
            ops.unpack8(packed._replace(**change))
    with pytest.raises(TypeError):
        ops.pack8(torch.zeros(3, dtype=torch.int32))
    with pytest.raises(ValueError):
        ops.pack8(torch.zeros(()))


def test_swiglu8_uses_the_kept_values():
    gate, up = _rand(3, 70, dtype=torch.float32).requires_grad_(), _rand(3, 70, seed=1, dtype=torch.float32).requires_grad_()
    y = ops.swiglu8(gate, up)
    assert torch.allclose(y, torch.nn.functional.silu(gate) * up, rtol=1e-6, atol=0)
    up_grad = _rand(3, 70, seed=2, dtype=torch.float32)
    got = torch.autograd.grad(y, (gate, up), up_grad)
    g, u = ops.unpack8(ops.pack8(gate.detach())).requires_grad_(), ops.unpack8(ops.pack8(up.detach())).requires_grad_()
    for a, b in zip(got, torch.autograd.grad(torch.nn.functional.silu(g) * u, (g, u), up_grad)):
        assert torch.allclose(a, b, rtol=1e-5, atol=1e-6)
    weight = _rand(4, 70, seed=3, dtype=torch.float32).requires_grad_()
    out = ops.swiglu_linear8(gate, up, weight)
    assert torch.allclose(out, y @ weight.t(), rtol=1e-5, atol=1e-5)
    grad = _rand(3, 4, seed=4, dtype=torch.float32)
    got = torch.autograd.grad(out, (gate, up, weight), grad)
    for a, b in zip(got, torch.autograd.grad((torch.nn.functional.silu(g) * u) @ weight.t(), (g, u, weight), grad)):
        assert torch.allclose(a, b, rtol=1e-4, atol=1e-5)
    with pytest.raises(ValueError):
        ops.swiglu8(gate, up[:2])
    with pytest.raises(TypeError):
        ops.swiglu8(gate.double(), up.double())
    with pytest.raises(ValueError):
        ops.swiglu_linear8(gate, up, weight[:, :3])


def test_checkpoint8_runs_again_from_the_kept_input():
    layer = torch.nn.Sequential(torch.nn.Linear(70, 9), torch.nn.Tanh())
    x = _rand(2, 3, 70, dtype=torch.float32).requires_grad_()
    shift = _rand(9, seed=5, dtype=torch.float32).requires_grad_()

    class Block(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.layer = layer

        def forward(self, x, shift, factor):
            return self.layer(x) + shift, factor * x

    block = Block()
    out, scaled = ops.checkpoint8(block, x, shift, 2.0)
    plain, plain_scaled = block(x, shift, 2.0)
    assert torch.equal(out, plain) and torch.equal(scaled, plain_scaled)
    wanted = (x, shift, *block.parameters())
    grads = (_rand(2, 3, 9, seed=6, dtype=torch.float32), _rand(2, 3, 70, seed=7, dtype=torch.float32))
    got = torch.autograd.grad((out, scaled), wanted, grads)
    kept = ops.unpack8(ops.pack8(x)).requires_grad_()
    expected = torch.autograd.grad(block(kept, shift, 2.0), (kept, *wanted[1:]), grads)
    for a, b in zip(got, expected):
        assert torch.equal(a, b)
    # one output unused, an input without gradients, no gradients at all
    out, _ = ops.checkpoint8(block, x.detach(), shift, 2.0)
    out.sum().backward()
    assert shift.grad is not None and layer[0].weight.grad is not None
    with torch.no_grad():
        assert not ops.checkpoint8(block, x, shift, 2.0)[0].requires_grad
    with pytest.raises(TypeError):
        ops.checkpoint8(block, torch.zeros(3, dtype=torch.int64))


# ---- under autocast -----------------------------------------------------------------------------------------------------
def test_checkpoint8_runs_again_under_the_autocast_of_the_first_run():
    torch.manual_seed(4)
    layer, x = torch.nn.Linear(70, 40), torch.randn(12, 70)
    direction = torch.randn(12, 40).bfloat16()
    kept = ops.unpack8(ops.pack8(x)).requires_grad_()
    with torch.autocast("cpu", dtype=torch.bfloat16):
        wanted = torch.autograd.grad(layer(kept), [kept, *layer.parameters()], direction)
        y = ops.checkpoint8(layer, x.requires_grad_())
        expected = layer(x)
    assert y.dtype == torch.bfloat16 and torch.equal(y, expected)
    for a, b in zip(torch.autograd.grad(y, [x, *layer.parameters()], direction), wanted):
        assert torch.equal(a, b)


def test_checkpoint8_under_autocast_around_the_backward_pass_alone():
    """What the plain block gives at the kept input.  (Not what it gives without autocast: torch's own products of a backward pass are rounded by
    the autocast around it, those of the plain block as well.)"""
    torch.manual_seed(4)
    layer, x = torch.nn.Linear(70, 40), torch.randn(12, 70, requires_grad=True)
    deep = torch.nn.Sequential(layer, torch.nn.Tanh(), torch.nn.Linear(40, 30))     # where the second run's own roundings would show
    for block in (layer, deep):
        kept = ops.unpack8(ops.pack8(x)).requires_grad_()
        plain, loss = block(kept).sum(), ops.checkpoint8(block, x).sum()
        with torch.autocast("cpu", dtype=torch.bfloat16):
            wanted = torch.autograd.grad(plain, [kept, *block.parameters()])
            inside = torch.autograd.grad(loss, [x, *block.parameters()])
        for a, b in zip(inside, wanted):
            assert torch.equal(a, b)


def test_swiglu_linear8_keeps_its_type_under_autocast():
    torch.manual_seed(5)
    gate, up, weight = (torch.randn(*shape, requires_grad=True) for shape in ((9, 70), (9, 70), (33, 70)))
    plain = ops.swiglu_linear8(gate, up, weight)
    wanted = torch.autograd.grad(plain.sum(), (gate, up, weight))
    with torch.autocast("cpu", dtype=torch.bfloat16):
        y = ops.swiglu_linear8(gate, up, weight)
        gradients = torch.autograd.grad(y.sum(), (gate, up, weight))
    for a, b in zip((y, *gradients), (plain, *wanted)):
        assert a.dtype == torch.float32 and torch.equal(a, b)


def test_cross_entropy_keeps_its_accuracy_under_autocast():
    torch.manual_seed(6)
    hidden, weight = torch.randn(9, 70, requires_grad=True), torch.randn(50, 70, requires_grad=True)
    targets = torch.randint(0, 50, (9,))
    plain = ops.linear_cross_entropy(hidden, weight, targets)
    wanted = torch.autograd.grad(plain, (hidden, weight))
    with torch.autocast("cpu", dtype=torch.bfloat16):
        loss = ops.linear_cross_entropy(hidden, weight, targets)
        gradients = torch.autograd.grad(loss, (hidden, weight))
    for a, b in zip((loss, *gradients), (plain, *wanted)):
        assert a.dtype == torch.float32 and torch.equal(a, b)


# ---- the plain product of the native library ----------------------------------------------------------------------------
def _product(**change):
    from soap_tp_b200 import _decoder

    bf16 = torch.bfloat16
    given = dict(a=torch.zeros(16, 24, dtype=bf16), b=torch.zeros(24, 32, dtype=bf16), out=torch.zeros(16, 32, dtype=bf16), turned=False, status=0)
    given.update(change)
    return _decoder.gemm16(**given)


@pytest.mark.parametrize("change,error", [
    (dict(), ValueError),                                                              # not on CUDA
    (dict(out=torch.zeros(16, 24, dtype=torch.bfloat16)), ValueError),
    (dict(out=torch.zeros(8, 32, dtype=torch.bfloat16)), ValueError),
    (dict(b=torch.zeros(16, 32, dtype=torch.bfloat16)), ValueError),
    (dict(turned=True), ValueError),
    (dict(out=torch.zeros(32, 16, dtype=torch.bfloat16).t()), ValueError),
    (dict(a=torch.zeros(24, dtype=torch.bfloat16)), ValueError),
    (dict(out=torch.zeros(16, 32)), TypeError),
    (dict(b=torch.zeros(24, 32, dtype=torch.float16)), TypeError),
    (dict(split_parts=torch.zeros(4)), ValueError),
    (dict(split_parts=torch.zeros(4), split_counters=torch.zeros(4, dtype=torch.int32)), ValueError),
])
def test_native_product_refusals(change, error):
    with pytest.raises(error):
        _product(**change)
