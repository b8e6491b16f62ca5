"""Operators of a decoder's training step on the GPU, at the edges of what they accept: see also ``test_decoder_ops_cuda.py``."""
import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from decoder_bounds import IGNORED, F32, half_step, head_exact, smallest, within
from test_decoder_ops_cuda import BF16, FP16, FP32, _check_head, _check_norm, _head, _no_timeouts, _rand  # noqa: F401

pytestmark = pytest.mark.gpu


# ---- forward mode -------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("which", [0, 1, 2])
@pytest.mark.parametrize("grad_mode", [True, False])
def test_forward_mode_is_refused(which, grad_mode):
    from soap_tp_b200 import ops

    plain = [_rand(4, 64, seed=i, dtype=BF16) for i in range(2)] + [_rand(8, 64, seed=2, dtype=BF16)]
    with torch.set_grad_enabled(grad_mode), forward_ad.dual_level():
        gate, up, weight = (forward_ad.make_dual(t, torch.ones_like(t)) if i == which else t for i, t in enumerate(plain))
        with pytest.raises(RuntimeError, match="jvp"):
            ops.swiglu_linear8(gate, up, weight)
        if which < 2:
            with pytest.raises(RuntimeError, match="jvp"):
                ops.swiglu8(gate, up)
            with pytest.raises(RuntimeError, match="jvp"):
                ops.residual_norm(gate, up, torch.ones(64, device="cuda"))
            with pytest.raises(RuntimeError, match="jvp"):
                ops.linear_cross_entropy(gate if which == 0 else up, weight, torch.zeros(4, dtype=torch.int64, device="cuda"))


# ---- gates far below zero -----------------------------------------------------------------------------------------------
def _exp_error(dtype, gate):
    """Relative error of silu for gates of -20 and below, in 16 bits in units of 2^-23: the exponent, at most |g| log2 e, is rounded (0.5 |g|) and
    multiplied by a rounded log2 e (0.2 |g|), the power and the reciprocal are off by two and one, products by half a unit each.  fp32: the
    accurate functions' two units."""
    return (8 + 1.173 * gate.abs()) * 2.0 ** -23 if dtype != FP32 else torch.full_like(gate, 16 * F32)


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
def test_swiglu8_of_gates_far_below_zero(dtype):
    """exp(g) down to 2^-149 counts: 1e37 silu(-88) is -0.5.  Below 2^-126 it is a multiple of 2^-149, and so is its quotient."""
    from soap_tp_b200.ops import pack8, swiglu8

    gate = torch.linspace(-96.0, -20.0, 64 * 40, device="cuda").view(40, 64).to(dtype).requires_grad_()
    large = 1e37 if dtype != FP16 else 4e4
    up = (_rand(40, 64, seed=1).sign() * (0.5 + _rand(40, 64, seed=2).abs().clamp(max=1.0)) * large).to(dtype).requires_grad_()
    grad = _rand(40, 64, seed=3, dtype=dtype)
    y = swiglu8(gate, up)
    g, v, u = gate.detach().double(), up.detach().double(), half_step(dtype)
    exact = g * torch.sigmoid(g) * v
    within(y, (exact, (u + _exp_error(dtype, g)) * exact.abs() + 2.0 ** -148 * (g * v).abs() + smallest(dtype)))

    def kept(t):
        packed = pack8(t.detach())
        return packed.values.double() * packed.scales.double().repeat_interleave(64, dim=1)

    got = torch.autograd.grad(y, (gate, up), grad)
    g, v, d = kept(gate), kept(up), grad.double()
    # (a kept value is a product rounded to fp32, off by |g| 2^-24: that much of its exponential)
    s, c = torch.sigmoid(g), _exp_error(dtype, g) + g.abs() * F32
    d_up, d_gate = d * g * s, d * v * s * (1 + g * (1 - s))
    within(got[1], (d_up, (u + c) * d_up.abs() + 2.0 ** -148 * (d * g).abs() + smallest(dtype)))
    within(got[0], (d_gate, u * d_gate.abs() + (d * v).abs() * (1 + g.abs()) * (c * s + 2.0 ** -147) + smallest(dtype)))


# ---- the largest numbers ------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
def test_largest_values_stay_finite_in_eight_bits(dtype):
    from soap_tp_b200.ops import pack8, unpack8

    x = torch.zeros(2, 130, dtype=dtype, device="cuda")
    x[0, 3], x[1, 70], x[1, 129] = torch.finfo(dtype).max, torch.finfo(dtype).min, torch.finfo(dtype).min
    back = unpack8(pack8(x))
    assert bool(torch.isfinite(back).all())
    within(back, (x.double(), (half_step(dtype) + 4 * F32) * x.double().abs()))


# ---- padding ------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("counted", [1, 64])
def test_loss_of_a_token_does_not_depend_on_padding(dtype, counted):
    from soap_tp_b200.ops import linear_cross_entropy

    hidden, weight, targets = _head(counted, 4200, 700, dtype)
    padded, padded_targets = torch.cat((hidden.detach(), _rand(300, 4200, seed=7, dtype=dtype))), torch.full((counted + 300,), IGNORED, device="cuda")
    padded_targets[:counted] = targets
    for reduction in ("none", "mean"):
        alone = linear_cross_entropy(hidden, weight, targets, reduction=reduction)
        among = linear_cross_entropy(padded.requires_grad_(), weight, padded_targets, reduction=reduction)
        assert torch.equal(alone, among[:counted] if reduction == "none" else among)


# ---- nothing to do ------------------------------------------------------------------------------------------------------
def test_empty_swiglu_linear8_keeps_its_type_under_autocast():
    from soap_tp_b200.ops import swiglu_linear8

    gate, weight = torch.zeros(0, 64, dtype=BF16, device="cuda", requires_grad=True), _rand(5, 64, dtype=BF16).requires_grad_()
    with torch.autocast("cuda", dtype=FP16):
        y = swiglu_linear8(gate, gate, weight)
        grads = torch.autograd.grad(y.sum(), (gate, weight))
    assert y.dtype == BF16 and y.shape == (0, 5) and all(g.dtype == BF16 for g in grads) and not grads[1].any()


# ---- paths that small sizes do not take ---------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("reduction", ["mean", "none"])
# logits drained twice and three times, in tiles that pairs of thread blocks take one and several of; every 256 of K for a few tokens
@pytest.mark.parametrize("tokens,depth,words", [(300, 2112, 700), (300, 4200, 700), (300, 4200, 10000), (600, 6000, 5000), (40, 1000, 300), (64, 2100, 20000)])
def test_cross_entropy_of_deep_hidden_states(tokens, depth, words, reduction, dtype):
    _check_head(*_head(tokens, depth, words, dtype, ignored=0.1), reduction)


# more rows than the blocks' rings hold at once, off 16-byte boundaries and on them
@pytest.mark.parametrize("rows,dim,dtype", [(4000, 3001, BF16), (4000, 3000, FP16), (40000, 67, BF16), (40000, 72, FP16), (6000, 1001, FP32), (3000, 5001, BF16),
                                            (3000, 5120, BF16)])
@pytest.mark.parametrize("after,gated", [(False, False), (True, True)])
def test_residual_norm_of_many_rows(rows, dim, dtype, after, gated):
    _check_norm(rows, dim, dtype, after, gated)


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_cross_entropy_by_token_in_a_graph(dtype):
    from soap_tp_b200.ops import linear_cross_entropy

    def step(hidden, weight, targets, up):
        loss = linear_cross_entropy(hidden, weight, targets, reduction="none", workspace_bytes=1)
        return (loss, *torch.autograd.grad(loss, (hidden, weight), up))

    def inputs(seed):
        up = torch.rand(300, generator=torch.Generator("cuda").manual_seed(seed + 9), device="cuda") - 0.3
        return [*_head(300, 72, 400, dtype, seed=seed, ignored=0.2 + 0.0005 * seed), up]

    held = inputs(0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*held)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outputs = step(*held)
    for seed in (100, 1000):
        with torch.no_grad():
            for old, new in zip(held, inputs(seed)):
                old.copy_(new)
        for _ in range(2):
            graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(outputs, step(*inputs(seed))):
            assert torch.equal(a, b)


# ---- saved tensors that travel, several threads, a second backward pass -------------------------------------------------
def _operators():
    from soap_tp_b200 import ops

    hidden, weight, targets = _head(300, 72, 400, BF16, ignored=0.2)
    x, b, gate, up = (_rand(40, 136, seed=10 + i, dtype=BF16).requires_grad_() for i in range(4))
    norm, down = (1 + _rand(136, seed=20, scale=0.1)).to(BF16).requires_grad_(), _rand(24, 136, seed=21, dtype=BF16).requires_grad_()
    per_token = torch.rand(300, generator=torch.Generator("cuda").manual_seed(9), device="cuda")
    return [
        (lambda: ops.linear_cross_entropy(hidden, weight, targets), (hidden, weight), None),
        (lambda: ops.linear_cross_entropy(hidden, weight, targets, reduction="none"), (hidden, weight), per_token),
        (lambda: ops.residual_norm(x, b, norm, branch_weight=norm, gate=norm, scale=0.5), (x, b, norm), (_rand(40, 136, seed=30, dtype=BF16),) * 2),
        (lambda: ops.rms_norm(x, norm), (x, norm), _rand(40, 136, seed=31, dtype=BF16)),
        (lambda: ops.swiglu8(gate, up), (gate, up), _rand(40, 136, seed=32, dtype=BF16)),
        (lambda: ops.swiglu_linear8(gate, up, down), (gate, up, down), _rand(40, 24, seed=33, dtype=BF16)),
        (lambda: ops.checkpoint8(lambda t, w: torch.nn.functional.linear(t, w), x, down), (x, down), _rand(40, 24, seed=34, dtype=BF16))]


@pytest.mark.parametrize("which", range(7))
def test_operators_under_hooks_on_saved_tensors(which):
    call, leaves, up = _operators()[which]
    wanted = torch.autograd.grad(call(), leaves, up)
    with torch.autograd.graph.save_on_cpu():
        outputs = call()
    for a, b in zip(torch.autograd.grad(outputs, leaves, up), wanted):
        assert torch.equal(a, b)


@pytest.mark.parametrize("which", range(7))
def test_a_second_backward_pass_gives_the_same(which):
    call, leaves, up = _operators()[which]
    outputs = call()
    first = [g.clone() for g in torch.autograd.grad(outputs, leaves, up, retain_graph=True)]
    second, third = torch.autograd.grad(outputs, leaves, up, retain_graph=True), torch.autograd.grad(outputs, leaves, up)
    for a, b, c in zip(first, second, third):
        assert torch.equal(b, c)
        # (a reduced loss makes its gradients with its value, and again from logits computed anew: of bf16's roundings apart)
        assert torch.equal(a, b) or which == 0 and float((a.double() - b.double()).norm()) <= 2.0 ** -7 * float(b.double().norm())


def test_operators_from_several_threads():
    import threading

    calls = _operators()
    wanted = [torch.autograd.grad(call(), leaves, up) for call, leaves, up in calls]
    torch.cuda.synchronize()
    results, errors = {}, []

    def work(number):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for _ in range(3):
                    results[number] = [torch.autograd.grad(call(), leaves, up) for call, leaves, up in calls]
            stream.synchronize()
        except Exception as error:      # pragma: no cover - shown by the assertion below
            errors.append(error)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(3)]
    for thread in threads:
        thread.start()
    for thread in threads:
        thread.join()
    assert not errors and len(results) == 3
    for got in results.values():
        for one, expected in zip(got, wanted):
            for a, b in zip(one, expected):
                assert torch.equal(a, b)
