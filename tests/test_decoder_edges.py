"""Operators of a decoder's training step on CPU tensors, at the edges of what they accept: see also ``test_decoder_ops.py``."""
import functools
import math

import pytest
import torch

from decoder_bounds import F32, IGNORED, half_step, within
from soap_tp_b200 import ops


# ---- the largest numbers ------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_largest_values_stay_finite_in_eight_bits(dtype):
    x = torch.zeros(2, 130, dtype=dtype)
    x[0, 3], x[1, 70], x[1, 129] = torch.finfo(dtype).max, torch.finfo(dtype).min, torch.finfo(dtype).min
    back = ops.unpack8(ops.pack8(x))
    # the scale is rounded once or a step below that, the product once, the result once
    within(back, (x.double(), (half_step(dtype) + 4 * F32) * x.double().abs()))
    x[0, 5] = float("inf")
    assert bool(ops.unpack8(ops.pack8(x))[0, :64].isnan().all())


# ---- padding ------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("held", [float("nan"), float("inf"), -1e30])
@pytest.mark.parametrize("dtype", [torch.float64, torch.float32, torch.bfloat16])
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_cross_entropy_leaves_padding_out(reduction, dtype, held):
    generator = torch.Generator().manual_seed(3)
    hidden, weight = torch.randn(7, 12, generator=generator).to(dtype), torch.randn(20, 12, generator=generator).to(dtype).requires_grad_()
    targets = torch.randint(0, 20, (7,), generator=generator)
    targets[2], targets[6] = IGNORED, IGNORED
    up = torch.rand(7 if reduction == "none" else (), generator=generator, dtype=torch.float64 if dtype == torch.float64 else torch.float32)

    def results(hidden):
        loss = ops.linear_cross_entropy(hidden, weight, targets, reduction=reduction)
        return (loss, *torch.autograd.grad(loss, (hidden, weight), up))

    expected = results(hidden.clone().requires_grad_())
    hidden[targets == IGNORED] = held
    for a, b in zip(results(hidden.requires_grad_()), expected):
        assert torch.equal(a, b)
    assert not expected[1][targets == IGNORED].any()


# ---- losses of any size -------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("loss", [1e-30, 1e-12, 0.5, 5.0, 19.0, 20.5, 21.0, 25.0, 40.0, 300.0])
def test_cross_entropy_of_64_bits_has_64_bits(loss):
    # 64 words of equal logits, 0, and the target's: log(1 + 64 exp(-t)) = loss
    t = math.log(64) - math.log(math.expm1(loss))
    hidden = torch.tensor([[t]], dtype=torch.float64, requires_grad=True)
    weight = torch.zeros(65, 1, dtype=torch.float64)
    weight[7] = 1.0
    got = ops.linear_cross_entropy(hidden, weight, torch.tensor([7]))
    # log 64, t and their difference are rounded to 2^-53 of at most 300 + 2 log 64, and the loss to 2^-53 of itself
    exact = math.log1p(64 * math.exp(-t))
    assert abs(float(got.detach()) - exact) <= 8 * 2.0 ** -53 * max(1.0, abs(t)) * exact
    # the gradient is p - 1 = expm1(-loss), from exp(l - lse) - 1: off by the rounding of lse and of one
    assert abs(float(torch.autograd.grad(got, hidden)[0]) - math.expm1(-exact)) <= 8 * 2.0 ** -53 * max(1.0, abs(t))


def test_cross_entropy_of_words_that_cannot_be():
    weight = torch.zeros(4, 1, dtype=torch.float64)
    weight[0], weight[1:] = 1.0, float("-inf")
    assert float(ops.linear_cross_entropy(torch.ones(1, 1, dtype=torch.float64), weight, torch.tensor([0]))) == 0.0
    assert float(ops.linear_cross_entropy(torch.ones(1, 1, dtype=torch.float64), weight, torch.tensor([2]))) == float("inf")


# ---- what a checkpointed function returns -------------------------------------------------------------------------------
def test_checkpoint8_leaves_tensors_alone_that_the_function_returns():
    module, x = torch.nn.Linear(70, 9), torch.randn(4, 70, requires_grad=True)
    constant = torch.randn(9)
    module.register_buffer("buffer", constant)

    class Returns(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.inner = module

        def forward(self, t):
            return self.inner(t), self.inner.weight, self.inner.buffer, t

    y, weight, buffer, same = ops.checkpoint8(Returns(), x)
    assert module.weight.is_leaf and module.weight.grad_fn is None and not constant.requires_grad and x.is_leaf
    assert torch.equal(weight, module.weight) and torch.equal(buffer, constant) and torch.equal(same, x)
    (y.sum() + 2 * weight.sum() + 3 * same.sum()).backward()
    kept = ops.unpack8(ops.pack8(x))
    assert torch.allclose(module.weight.grad, kept.sum(0).expand(9, 70) + 2, rtol=1e-6)
    assert torch.allclose(x.grad, module.weight.detach().sum(0).expand(4, 70) + 3, rtol=1e-6)


def test_checkpoint8_of_lists_and_refusals_of_other_containers():
    module, x = torch.nn.Linear(70, 9), torch.randn(4, 70, requires_grad=True)

    class Returns(torch.nn.Module):
        def __init__(self, container):
            super().__init__()
            self.inner, self.container = module, container

        def forward(self, t):
            return self.container(self.inner(t))

    a, b = ops.checkpoint8(Returns(lambda y: [y, 2 * y]), x)
    (a + b).sum().backward()
    assert torch.allclose(x.grad, 3 * module.weight.detach().sum(0).expand(4, 70), rtol=1e-6, atol=1e-6)
    with pytest.raises(TypeError, match="tuple"):
        ops.checkpoint8(Returns(lambda y: {"y": y}), x)


def test_checkpoint8_refuses_tensors_inside_its_outputs():
    class Returns(torch.nn.Linear):
        def __init__(self, form):
            super().__init__(70, 9)
            self.form = form

        def forward(self, t):
            return self.form(super().forward(t))

    x = torch.randn(4, 70, requires_grad=True)
    for form in (lambda y: (y, (2 * y, 3 * y)), lambda y: [y, {"twice": [2 * y]}]):
        with pytest.raises(TypeError, match="containers"):
            ops.checkpoint8(Returns(form), x)
    y, shape, nothing = ops.checkpoint8(Returns(lambda y: (y, y.shape, None)), x)
    assert y.requires_grad and shape == (4, 9) and nothing is None


# ---- what a checkpointed function uses ----------------------------------------------------------------------------------
class _Scaled(torch.nn.Module):
    def __init__(self):
        super().__init__()
        self.layer = torch.nn.Linear(70, 9)

    def forward(self, x, factor=1.0):
        return self.layer(x).tanh() * factor

    def other(self, x, factor=1.0):
        return self.layer(x).sigmoid() * factor


@pytest.mark.parametrize("form", ["forward", "other", "partial"])
def test_checkpoint8_of_a_method_reaches_its_modules_parameters(form):
    torch.manual_seed(1)
    module, x = _Scaled(), torch.randn(4, 70, requires_grad=True)
    function = {"forward": module.forward, "other": module.other, "partial": functools.partial(module, factor=3.0)}[form]
    kept = ops.unpack8(ops.pack8(x)).requires_grad_()
    direction = torch.randn(4, 9)
    wanted = torch.autograd.grad(function(kept), (kept, *module.parameters()), direction)
    got = torch.autograd.grad(ops.checkpoint8(function, x), (x, *module.parameters()), direction)
    for a, b in zip(got, wanted):
        assert torch.equal(a, b)
    # x without gradients, as a first block's input: kept in 8 bits for the parameters all the same
    for a, b in zip(torch.autograd.grad(ops.checkpoint8(function, x.detach()), tuple(module.parameters()), direction), wanted[1:]):
        assert torch.equal(a, b)


def test_checkpoint8_refuses_to_lose_gradients():
    torch.manual_seed(2)
    module, x, shift = _Scaled(), torch.randn(4, 70, requires_grad=True), torch.randn(9, requires_grad=True)
    made = shift * 2
    for function, args in ((lambda t: module(t), ()), (lambda t: t + x, ()), (lambda t: module.layer.weight, ()), (lambda t: module(t) + made, ()),
                           (lambda t, pair: t[:, :9] * pair[0], ((shift,),)), (lambda t: (t, shift), ())):
        y = ops.checkpoint8(function, x, *args)
        with pytest.raises(RuntimeError, match="checkpoint8"):
            (y if isinstance(y, torch.Tensor) else y[0]).sum().backward()
    assert x.grad is None and shift.grad is None and module.layer.weight.grad is None
    # said in so many words, in `parameters`, or with nothing to lose
    ops.checkpoint8(lambda t: module(t), x, parameters=module.parameters()).sum().backward()
    assert module.layer.weight.grad is not None and x.grad is not None
    module.zero_grad()
    ops.checkpoint8(lambda t: module(t), x, parameters=()).sum().backward()
    assert module.layer.weight.grad is None
    ops.checkpoint8(lambda t, s: t[:, :9] * s, x, shift).sum().backward()
    assert shift.grad is not None
    module.requires_grad_(False)
    ops.checkpoint8(lambda t: module(t), x).sum().backward()
    ops.checkpoint8(module.requires_grad_(True), x).sum().backward()
    assert module.layer.weight.grad is not None


@pytest.mark.parametrize("hooks", [lambda: torch.autograd.graph.saved_tensors_hooks(torch.clone, lambda t: t), torch.autograd.graph.save_on_cpu])
def test_checkpoint8_under_hooks_on_saved_tensors(hooks):
    torch.manual_seed(3)
    module, x, direction = _Scaled(), torch.randn(4, 70, requires_grad=True), torch.randn(4, 9)
    wanted = torch.autograd.grad(ops.checkpoint8(module, x), (x, *module.parameters()), direction)
    for function, options in ((module, {}), (lambda t: module(t), dict(parameters=module.parameters()))):
        with hooks():
            y = ops.checkpoint8(function, x, **options)
        for a, b in zip(torch.autograd.grad(y, (x, *module.parameters()), direction, allow_unused=True), wanted):
            assert a is not None and torch.equal(a, b)
    y = ops.checkpoint8(module, x)
    with torch.no_grad():
        module.layer.weight.add_(1.0)
    with pytest.raises(RuntimeError, match="modified"):
        y.sum().backward()


# ---- the plain product of the native library ----------------------------------------------------------------------------
BF16, FP16 = torch.bfloat16, torch.float16


@pytest.mark.parametrize("change,error,message", [
    (dict(), ValueError, "of one CUDA device"),
    (dict(out=torch.zeros(16, 24, dtype=BF16)), ValueError, "sizes do not match"),
    (dict(out=torch.zeros(8, 32, dtype=BF16)), ValueError, "sizes do not match"),
    (dict(b=torch.zeros(16, 32, dtype=BF16)), ValueError, "sizes do not match"),
    (dict(turned=True), ValueError, "sizes do not match"),
    (dict(out=torch.zeros(32, 16, dtype=BF16).t()), ValueError, "rows lie in memory"),
    (dict(out=torch.zeros(512, dtype=BF16).as_strided((16, 32), (8, 1))), ValueError, "rows lie in memory"),
    (dict(a=torch.zeros(24, dtype=BF16)), ValueError, "rows lie in memory"),
    (dict(a=torch.zeros(16, 0, dtype=BF16), b=torch.zeros(0, 32, dtype=BF16)), ValueError, "rows lie in memory"),
    (dict(out=torch.zeros(16, 32)), TypeError, "all of one type"),
    (dict(b=torch.zeros(24, 32, dtype=FP16)), TypeError, "all of one type"),
    (dict(a=torch.zeros(16, 24), b=torch.zeros(24, 32), out=torch.zeros(16, 32)), TypeError, "bfloat16 or float16"),
    (dict(split_parts=torch.zeros(4)), ValueError, "go together"),
    (dict(split_counters=torch.zeros(4, dtype=torch.int32)), ValueError, "go together"),
    (dict(split_parts=torch.zeros(4), split_counters=torch.zeros(4, dtype=torch.int32)), ValueError, "too small"),
    (dict(split_parts=torch.zeros(4), split_counters=torch.zeros(4)), TypeError, "split_counters int32"),
    (dict(split_parts=torch.zeros(4, dtype=BF16), split_counters=torch.zeros(4, dtype=torch.int32)), TypeError, "split_parts are float32"),
])
def test_what_the_native_product_says_it_refuses(change, error, message):
    native = pytest.importorskip("soap_tp_b200._decoder")
    given = dict(a=torch.zeros(16, 24, dtype=BF16), b=torch.zeros(24, 32, dtype=BF16), out=torch.zeros(16, 32, dtype=BF16), turned=False, status=0)
    with pytest.raises(error, match=message):
        native.gemm16(**given | change)
