"""Operators of a decoder's training step on the GPU, against their definitions in 64 bits and bounds derived in ``decoder_bounds.py``."""
import pytest
import torch

from decoder_bounds import IGNORED, F32, half_step, head_exact, norm_exact, smallest, within

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def _rand(*shape, seed=0, dtype=FP32, scale=1.0):
    return (scale * torch.randn(*shape, generator=torch.Generator("cuda").manual_seed(seed), device="cuda")).to(dtype)


@pytest.fixture(autouse=True)
def _no_timeouts():
    yield
    from soap_tp_b200.engine import kernels

    kernels.check_status()


# ---- products on 16-bit operands ----------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("k_major", [True, False])
@pytest.mark.parametrize("split", [False, True])
@pytest.mark.parametrize("m,n,k", [(1, 8, 1), (128, 256, 64), (256, 256, 128), (130, 72, 200), (513, 300, 65), (300, 1000, 2000), (2600, 2300, 1096),
                                   (100, 700, 30000)])
def test_gemm16(m, n, k, k_major, dtype, split):
    from soap_tp_b200.engine import decoder, kernels

    native = decoder.native

    def padded(rows, cols, seed):
        return _rand(rows, kernels.round_up(cols, 8), seed=seed, dtype=dtype)[:, :cols]

    a = padded(m, k, 1) if k_major else padded(k, m, 1)
    b = padded(k, n, 2)
    c = torch.full((m + 1, n + 3), 7.0, dtype=dtype, device="cuda")
    parts = torch.full((native.SPLIT_SCRATCH,), float("nan"), device="cuda") if split else None
    counters = torch.zeros(native.SPLIT_COUNTERS, dtype=torch.int32, device="cuda") if split else None
    native.gemm16(a, b, c, not k_major, decoder.status(a.device), parts, counters)
    x = a.double() if k_major else a.double().t()
    exact = x @ b.double()
    bound = half_step(dtype) * exact.abs() + (k // 16 + 2) * 2.0 ** -23 * (x.abs() @ b.double().abs()) + smallest(dtype)
    within(c[:m, :n], (exact, bound))
    assert bool((c[m] == 7).all()) and bool((c[:, n:] == 7).all()) and (counters is None or not counters.any())


# ---- cross entropy ------------------------------------------------------------------------------------------------------
def _head(tokens, depth, words, dtype, seed=0, ignored=0.0):
    weight = _rand(words, depth, seed=seed, dtype=dtype, scale=1.5 / depth ** 0.5)
    targets = torch.randint(0, words, (tokens,), generator=torch.Generator("cuda").manual_seed(seed + 1), device="cuda")
    known = 12.0 * torch.rand(tokens, 1, generator=torch.Generator("cuda").manual_seed(seed + 2), device="cuda")
    hidden = (_rand(tokens, depth, seed=seed + 3) + known / 2.25 * weight[targets].float()).to(dtype)
    targets[torch.rand(tokens, generator=torch.Generator("cuda").manual_seed(seed + 4), device="cuda") < ignored] = IGNORED
    return hidden.requires_grad_(), weight.requires_grad_(), targets


def _check_head(hidden, weight, targets, reduction="mean", upstream=None, **options):
    from soap_tp_b200.ops import linear_cross_entropy

    loss = linear_cross_entropy(hidden, weight, targets, reduction=reduction, **options)
    assert loss.dtype == FP32
    if reduction == "none" and upstream is None:
        upstream = torch.rand(loss.shape, generator=torch.Generator("cuda").manual_seed(9), device="cuda") - 0.3
    grads = torch.autograd.grad(loss, (hidden, weight), upstream)
    flat = hidden.detach().reshape(-1, hidden.shape[-1])
    losses, d_hidden, d_weight = head_exact(flat, weight, targets.reshape(-1), reduction, None if upstream is None else upstream.reshape(-1) if
                                            reduction == "none" else upstream)
    within(loss, losses)
    assert grads[0].shape == hidden.shape and grads[0].dtype == hidden.dtype and grads[1].shape == weight.shape
    within(grads[0], d_hidden)
    within(grads[1], d_weight)
    return loss, grads


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("tokens,depth,words", [(1, 8, 1), (1, 64, 300), (3, 100, 129), (128, 32, 64), (257, 40, 513), (300, 520, 1000),
                                                (33, 33, 77), (700, 256, 2500)])
@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_cross_entropy(tokens, depth, words, dtype, reduction):
    _check_head(*_head(tokens, depth, words, dtype, ignored=0.3 if tokens > 30 else 0.0), reduction)


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_cross_entropy_in_several_turns(reduction):
    # 700 tokens, 256 at a time: the weight's gradient is summed in fp32
    _check_head(*_head(700, 72, 1100, BF16, ignored=0.2), reduction, workspace_bytes=256 * 2 * 1152)


def test_cross_entropy_with_a_scaled_loss():
    _check_head(*_head(200, 64, 300, FP16), "mean", upstream=torch.tensor(1024.0, device="cuda"))
    _check_head(*_head(200, 64, 300, BF16), "sum", upstream=torch.tensor(-0.3, device="cuda"))


def test_cross_entropy_forward_alone_gives_the_same_loss():
    from soap_tp_b200.ops import linear_cross_entropy

    hidden, weight, targets = _head(300, 72, 1100, BF16, ignored=0.2)
    for reduction in ("none", "sum", "mean"):
        with torch.no_grad():
            alone = linear_cross_entropy(hidden, weight, targets, reduction=reduction)
        within(alone, head_exact(hidden, weight, targets, reduction)[0])


def test_cross_entropy_of_other_strides_and_types():
    hidden, weight, targets = _head(60, 48, 200, BF16)
    wide = torch.zeros(60, 100, dtype=BF16, device="cuda")
    wide[:, 3:51] = hidden.detach()
    _check_head(wide[:, 3:51].requires_grad_(), weight, targets)                                     # rows not on 16 bytes
    _check_head(hidden, weight.detach().t().contiguous().t().requires_grad_(), targets)              # weight stored the other way
    _check_head(hidden.detach()[:1].expand(60, 48).requires_grad_(), weight, targets)               # one row for all tokens
    _check_head(hidden.detach().view(4, 15, 48).transpose(0, 1).requires_grad_(), weight, targets.view(4, 15).t().to(torch.int32))


def test_cross_entropy_gradients_one_at_a_time_and_twice():
    from soap_tp_b200.ops import linear_cross_entropy

    hidden, weight, targets = _head(100, 64, 300, BF16)
    loss = linear_cross_entropy(hidden, weight, targets)
    first = torch.autograd.grad(loss, (hidden, weight), retain_graph=True)
    for _ in range(2):
        again = torch.autograd.grad(loss, (hidden, weight), retain_graph=True)
        exact = head_exact(hidden, weight, targets, "mean")
        within(again[0], exact[1])
        within(again[1], exact[2])
    within(first[0], exact[1])
    within(first[1], exact[2])
    for h, w in ((hidden, weight.detach()), (hidden.detach(), weight)):
        loss = linear_cross_entropy(h, w, targets)
        leaf = h if h.requires_grad else w
        within(torch.autograd.grad(loss, leaf)[0], exact[1 if leaf is h else 2])


def test_cross_entropy_of_unusual_targets():
    from soap_tp_b200.ops import linear_cross_entropy

    hidden, weight, targets = _head(40, 64, 300, BF16)
    for reduction in ("none", "sum", "mean"):
        loss = linear_cross_entropy(hidden, weight, torch.full_like(targets, IGNORED), reduction=reduction)
        assert not loss.any() and not any(g.any() for g in torch.autograd.grad(loss.sum(), (hidden, weight)))
    for wrong in (-1, 300, 2 ** 40):
        bad = targets.clone()
        bad[7] = wrong
        losses = linear_cross_entropy(hidden, weight, bad, reduction="none")
        assert bool(losses[7].isnan()) and int(losses.isnan().sum()) == 1
        loss = linear_cross_entropy(hidden, weight, bad)
        assert bool(loss.isnan()) and bool(torch.autograd.grad(loss, hidden)[0][7].isnan().all())
    _check_head(hidden, weight, torch.full_like(targets, 299))


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("ignored", [0.02, 0.9, 0.99])
def test_cross_entropy_leaves_padding_out(dtype, ignored):
    from soap_tp_b200.ops import linear_cross_entropy

    hidden, weight, targets = _head(700, 60, 500, dtype, ignored=ignored)
    targets[3], targets[5] = 17, IGNORED
    spoilt = hidden.detach().clone()
    spoilt[targets == IGNORED] = float("nan")
    for reduction in ("mean", "none"):
        _, expected = _check_head(hidden, weight, targets, reduction, workspace_bytes=1)
        up = torch.rand(700, generator=torch.Generator("cuda").manual_seed(9), device="cuda") - 0.3 if reduction == "none" else None
        leaf = spoilt.clone().requires_grad_()
        loss = linear_cross_entropy(leaf, weight, targets, reduction=reduction, workspace_bytes=1)
        for got, want in zip(torch.autograd.grad(loss, (leaf, weight), up), expected):
            assert torch.equal(got, want)
        assert not expected[0][targets == IGNORED].any()


def test_cross_entropy_backward_pass_captured_alone():
    from soap_tp_b200.ops import linear_cross_entropy

    hidden, weight, targets = _head(100, 64, 300, BF16)
    up = torch.tensor(0.5, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(linear_cross_entropy(hidden, weight, targets), (hidden, weight), up)
        loss = linear_cross_entropy(hidden, weight, targets)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        grads = torch.autograd.grad(loss, (hidden, weight), up)
    exact = head_exact(hidden, weight, targets, "mean", up)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        within(grads[0], exact[1])
        within(grads[1], exact[2])


def test_cross_entropy_of_captured_forward_and_backward_graphs():
    # two graphs: the backward one is replayed on its own too
    from soap_tp_b200.ops import linear_cross_entropy

    hidden, weight, targets = _head(100, 64, 300, BF16)
    up = torch.tensor(0.5, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(linear_cross_entropy(hidden, weight, targets), (hidden, weight), up)
    torch.cuda.current_stream().wait_stream(side)
    pool = torch.cuda.graph_pool_handle()
    forward, backward = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(forward, pool=pool, stream=side):
        loss = linear_cross_entropy(hidden, weight, targets)
    with torch.cuda.graph(backward, pool=pool, stream=side):
        grads = torch.autograd.grad(loss, (hidden, weight), up)
    exact = head_exact(hidden, weight, targets, "mean", up)
    for graph in (forward, backward, backward, forward, backward):
        graph.replay()
        torch.cuda.synchronize()
        within(loss, exact[0]) if graph is forward else (within(grads[0], exact[1]), within(grads[1], exact[2]))


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_cross_entropy_of_many_tokens(dtype):
    # more tokens than are counted at a time, and than the statistics of one turn hold
    hidden, weight, targets = _head(20001, 16, 130, dtype, ignored=0.3)
    for reduction in ("mean", "none"):
        _check_head(hidden, weight, targets, reduction, workspace_bytes=4096 * 24)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("reduction", ["sum", "none"])
def test_cross_entropy_of_known_words(dtype, reduction):
    # targets far ahead of all others: losses from 1 down to 1e-30, each to its own size
    from soap_tp_b200.ops import linear_cross_entropy

    weight = torch.eye(128, 64, device="cuda", dtype=dtype) * 4
    targets = torch.arange(60, device="cuda")
    hidden = torch.zeros(60, 64, device="cuda", dtype=dtype)
    hidden[targets, targets] = torch.linspace(1.0, 16.0, 60, device="cuda").to(dtype)
    hidden, weight = hidden.requires_grad_(), weight.requires_grad_()
    losses = linear_cross_entropy(hidden, weight, targets, reduction="none")
    exact = (127 * torch.exp(-4.0 * hidden.detach().double()[targets, targets])).log1p()
    # exact logits here: exp, log and sums of 127 equal terms in fp32
    within(losses, (exact, 2.0 ** -18 * exact))
    grads = torch.autograd.grad(linear_cross_entropy(hidden, weight, targets, reduction=reduction), hidden,
                                torch.ones(60, device="cuda") if reduction == "none" else None)[0]
    exact = 4 * torch.expm1(-exact)                      # by the target's word alone
    within(grads[targets, targets], (exact, (2 * half_step(dtype) + 2.0 ** -17) * exact.abs() + (2.0 ** -24 if dtype == FP16 else 0.0)))


def test_cross_entropy_of_large_logits():
    hidden, weight, targets = _head(64, 64, 300, BF16)
    big = (hidden.detach() * 40).requires_grad_()
    _check_head(big, weight, targets, "sum")


def test_cross_entropy_refuses_fp32_on_cuda():
    from soap_tp_b200.ops import linear_cross_entropy

    with pytest.raises(TypeError):
        linear_cross_entropy(_rand(2, 8), _rand(4, 8), torch.zeros(2, dtype=torch.int64, device="cuda"))


def _sharded_case(rank, world):
    # two ranks on one GPU, whose collectives go over the host; nothing on the device waits for the other rank
    import torch.distributed as dist
    from soap_tp_b200.ops import linear_cross_entropy

    for dtype, reduction, workspace in ((BF16, "mean", 1), (BF16, "sum", 2**31), (FP16, "none", 1), (BF16, "none", 2**31)):
        hidden, weight, targets = _head(600, 72, 640, dtype, ignored=0.2)
        per_rank = 640 // world
        mine = weight.detach()[rank * per_rank:(rank + 1) * per_rank].clone().requires_grad_()
        loss = linear_cross_entropy(hidden, mine, targets, reduction=reduction, group=dist.group.WORLD, workspace_bytes=workspace)
        up = torch.rand(600, generator=torch.Generator("cuda").manual_seed(9), device="cuda") if reduction == "none" else None
        d_hidden, d_weight = torch.autograd.grad(loss, (hidden, mine), up)
        losses, exact_hidden, exact_weight = head_exact(hidden, weight, targets, reduction, up)
        within(loss, losses)
        # each of the two ranks' parts of the hidden states' gradient is rounded before they are added: by half a step of the sums' magnitudes,
        # or half of the smallest subnormal number
        p = torch.softmax(hidden.detach().double() @ weight.detach().double().t(), dim=1)
        sizes = (p @ weight.detach().double().abs() + weight.detach().double()[targets.clamp(min=0)].abs()) * (targets != IGNORED).unsqueeze(1)
        sizes = sizes * (up.unsqueeze(1) if up is not None else 1.0 if reduction == "sum" else 1.0 / int((targets != IGNORED).sum()))
        within(d_hidden, (exact_hidden[0], exact_hidden[1] + 2 * half_step(dtype) * sizes + 2 * smallest(dtype)))
        within(d_weight, (exact_weight[0][rank * per_rank:(rank + 1) * per_rank], exact_weight[1][rank * per_rank:(rank + 1) * per_rank]))


def test_cross_entropy_over_two_ranks():
    from distributed_helpers import run_distributed

    run_distributed(_sharded_case, 2)


def test_cross_entropy_beyond_32_bits():
    # the softmax of one turn has more than 2^31 elements
    from soap_tp_b200.ops import linear_cross_entropy

    tokens, depth, words = 17000, 16, 128256
    hidden, weight, targets = _head(tokens, depth, words, BF16)
    loss = linear_cross_entropy(hidden, weight, targets, reduction="none", workspace_bytes=5 * 2 ** 30)
    up = torch.zeros(tokens, device="cuda")
    up[-50:] = 1.0
    grads = torch.autograd.grad(loss, (hidden, weight), up)
    exact = head_exact(hidden.detach()[-50:], weight, targets[-50:], "sum", tokens=tokens)
    within(loss[-50:].sum(), (exact[0][0], exact[0][1] + 64 * F32 * exact[0][0]))
    within(grads[0][-50:], exact[1])
    assert not grads[0][:-50].any()
    within(grads[1], exact[2])


# ---- norms --------------------------------------------------------------------------------------------------------------
def _check_norm(rows, dim, dtype, after, gated, normed=True, vector_dtype=None, scale=0.7, with_grad_h=True, with_grad_y=True, seed=0,
                eps=1e-5, pitch=None):
    from soap_tp_b200.ops import residual_norm

    vector_dtype = vector_dtype or dtype
    pitch = pitch or dim
    x, b, gh, gy = (_rand(rows, pitch, seed=seed + i, dtype=dtype)[:, :dim] for i in range(4))
    x, b = x.requires_grad_(), b.requires_grad_()
    w, wb, g = ((1 + 0.2 * _rand(dim, seed=seed + 5 + i)).to(vector_dtype).requires_grad_() if on else None
                for i, on in enumerate((normed, after, gated)))
    h, y = residual_norm(x, b, w, branch_weight=wb, gate=g, scale=scale, eps=eps)
    leaves = {k: v for k, v in dict(x=x, branch=b, weight=w, branch_weight=wb, gate=g).items() if v is not None}
    outputs = [(o, up) for o, up, on in ((h, gh, with_grad_h), (y, gy, with_grad_y)) if o is not None and on]
    grads = torch.autograd.grad([o for o, _ in outputs], list(leaves.values()), [up for _, up in outputs], allow_unused=True)
    exact = norm_exact(x, b, w, wb, g, scale, eps, gh if with_grad_h else None, gy if with_grad_y else None)
    within(h, exact["h"])
    if normed:
        within(y, exact["y"])
    for (name, leaf), grad in zip(leaves.items(), grads):
        if name == "weight" and not with_grad_y:
            assert grad is None
            continue
        assert grad.dtype == leaf.dtype and grad.shape == leaf.shape
        within(grad, exact[name])


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("rows,dim", [(1, 1), (3, 7), (20, 32), (300, 256), (7, 257), (33, 1000), (400, 1032), (9, 3001), (1000, 4096), (5, 5000), (4, 8200),
                                      (20, 4099), (7, 8191), (600, 33)])
@pytest.mark.parametrize("after,gated", [(False, False), (True, True)])
def test_residual_norm(rows, dim, dtype, after, gated):
    _check_norm(rows, dim, dtype, after, gated)


@pytest.mark.parametrize("dim", [9001, 16384, 16391, 20000, 32768])
def test_residual_norm_of_long_rows(dim):
    _check_norm(3, dim, BF16, True, True)


@pytest.mark.parametrize("options", [
    dict(after=True, gated=False), dict(after=False, gated=True), dict(after=False, gated=False, scale=1.0), dict(after=True, gated=True, normed=False),
    dict(after=False, gated=False, normed=False, scale=1.0), dict(after=True, gated=True, with_grad_h=False), dict(after=True, gated=True, with_grad_y=False),
    dict(after=False, gated=False, with_grad_y=False), dict(after=True, gated=True, vector_dtype=FP32), dict(after=True, gated=True, pitch=80),
    dict(after=True, gated=True, pitch=77)])
def test_residual_norm_forms(options):
    for dim in (72, 67):
        _check_norm(50, dim, BF16, **{"pitch": None, **options})


def test_residual_norm_of_zeros_and_large_values():
    from soap_tp_b200.ops import residual_norm, rms_norm

    x = torch.zeros(3, 64, device="cuda", dtype=BF16, requires_grad=True)
    b = torch.zeros(3, 64, device="cuda", dtype=BF16, requires_grad=True)
    w = torch.ones(64, device="cuda", dtype=BF16, requires_grad=True)
    h, y = residual_norm(x, b, w, branch_weight=w)
    assert not h.any() and not y.any()
    assert all(bool(torch.isfinite(g).all()) for g in torch.autograd.grad((h, y), (x, b, w), (torch.ones_like(h), torch.ones_like(y))))
    row = _rand(4, 512, seed=1)
    row[2] *= 1e15
    y = rms_norm(row, torch.ones(512, device="cuda"))
    exact = row.double() / (row.double().square().mean(-1, keepdim=True) + 1e-5).sqrt()
    within(y, (exact, 100 * F32 * exact.abs()))
    row[1, 3] = float("nan")
    y = rms_norm(row, torch.ones(512, device="cuda"))
    assert bool(y[1].isnan().all()) and int(y.isnan().sum()) == 512


def test_rms_norm_gradients():
    from soap_tp_b200.ops import rms_norm

    x, w = _rand(3, 5, 200, dtype=BF16).requires_grad_(), (1 + _rand(200, seed=1, scale=0.1)).to(BF16).requires_grad_()
    gy = _rand(3, 5, 200, seed=2, dtype=BF16)
    dx, dw = torch.autograd.grad(rms_norm(x, w), (x, w), gy)
    flat = x.detach().reshape(15, 200)
    exact = norm_exact(flat, torch.zeros_like(flat), w, None, None, 1.0, 1e-5, None, gy.reshape(15, 200))
    within(dx, exact["x"])
    within(dw, exact["weight"])


def test_residual_norm_gradients_do_not_share_memory_between_leaves():
    from soap_tp_b200.ops import residual_norm

    x, b = _rand(4, 64, dtype=BF16).requires_grad_(), _rand(4, 64, seed=1, dtype=BF16).requires_grad_()
    w = torch.ones(64, device="cuda", dtype=BF16)
    for _ in range(2):
        h, y = residual_norm(x.view(2, 2, 64), b.view(2, 2, 64), w)
        (h.float().sum() + y.float().square().sum()).backward()
    assert x.grad.data_ptr() != b.grad.data_ptr() and torch.equal(x.grad, b.grad)


# ---- activations in 8 bits ----------------------------------------------------------------------------------------------
SHAPES8 = [(1, 1), (2, 7), (3, 64), (5, 65), (600, 9), (70, 127), (41, 3001), (128, 32), (33, 200), (300, 1000), (77, 1792), (4, 14336)]


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("rows,dim", SHAPES8)
def test_pack8(rows, dim, dtype):
    from soap_tp_b200.ops import pack8, unpack8

    x = _rand(rows, dim, dtype=dtype, scale=3.0)
    packed = pack8(x)
    groups = -(-dim // 64)
    padded = torch.nn.functional.pad(x.double(), (0, groups * 64 - dim)).view(rows, groups, 64)
    scales = padded.abs().amax(-1) / 127
    assert bool(((packed.scales.double() - scales).abs() <= F32 * scales).all())           # one rounding
    step = packed.scales.double().repeat_interleave(64, dim=1)[:, :dim]
    # a quotient is moved onto a tie from up to 2^-16 + 127 * 2^-24 away (2^-16 = 256 * 2^-24), and the kept scale is rounded, 127 * 2^-24
    # more: half a step and (256 + 127 + 127) * 2^-24; fp32's three roundings make 127 * 3 * 2^-24
    assert bool(((packed.values[:, :dim].double() * step - x.double()).abs() <= step * (0.5 + 511 * F32)).all())
    exact = packed.values[:, :dim].double() * step
    within(unpack8(packed), (exact, (half_step(dtype) + F32) * exact.abs() + smallest(dtype)))


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_pack8_rounds_ties_to_even(dtype):
    """127 x / max in 64 bits (127 x is exact): what is a tie is rounded as one, and no other value leaves the definition unless it is near one."""
    from soap_tp_b200.ops import pack8

    x = _rand(4000, 64, dtype=dtype, scale=3.0)
    x[0, :] = x[0].abs().amax() / 2                                  # max / 2: the tie 63.5, of both signs
    x[0, :20] *= -1
    x[0, 0] = 2 * x[0, 1]
    quotient = 127 * x.double() / x.double().abs().amax(dim=1, keepdim=True)
    wanted, kept = quotient.round(), pack8(x).values.double()
    off = ((quotient - quotient.floor()) - 0.5).abs()                # distance from a tie
    assert int((off == 0).sum()) > 100
    assert torch.equal(kept[off == 0], wanted[off == 0])
    assert bool((off[kept != wanted] <= 2.0 ** -16 + 127 * F32).all())


def test_pack8_of_strided_rows_and_special_values():
    from soap_tp_b200.ops import pack8, unpack8

    wide = _rand(6, 300, dtype=BF16)
    for view in (wide[:, 5:205], wide[:, 8:208], wide.t()[:200], wide[:1].expand(6, 300)):
        assert torch.equal(unpack8(pack8(view)), unpack8(pack8(view.contiguous())))
    x = torch.zeros(4, 130, device="cuda")
    x[1, 3], x[2, 70], x[3, 129] = float("inf"), float("nan"), 2.0 ** -140
    back = unpack8(pack8(x))
    assert not back[0].any() and bool(back[1, :64].isnan().all()) and not back[1, 64:].any()
    assert bool(back[2, 64:128].isnan().all()) and not back[2, :64].any() and float(back[3, 129]) == 0.0
    assert unpack8(pack8(x[:0])).shape == (0, 130)
    tiny = torch.full((1, 64), 2.0 ** -120, device="cuda")
    assert torch.allclose(unpack8(pack8(tiny)), tiny, rtol=2.0 ** -7)


def test_pack8_beyond_32_bits():
    from soap_tp_b200.ops import pack8, unpack8

    x = torch.zeros(2 ** 17 + 3, 2 ** 15 + 8, dtype=FP16, device="cuda")      # more than 2^32 values
    x[-1] = _rand(2 ** 15 + 8, dtype=FP16)
    packed = pack8(x)
    last = pack8(x[-1:])
    assert torch.equal(packed.values[-1:], last.values) and torch.equal(packed.scales[-1:], last.scales)
    del x
    assert torch.equal(unpack8(packed)[-1:], unpack8(last))


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("dim", [5, 8, 61, 64, 200, 1001])
def test_rows_at_every_offset_from_a_boundary(dim, dtype):
    from soap_tp_b200.ops import pack8, swiglu8, unpack8

    for offset in range(8):
        for pitch in (dim, dim + 3):
            flat = _rand(40 * pitch + 16, seed=offset, dtype=dtype)
            x = flat[offset:].as_strided((33, dim), (pitch, 1))
            assert torch.equal(unpack8(pack8(x)), unpack8(pack8(x.clone())))
            assert torch.equal(swiglu8(x, x), swiglu8(x.clone(), x.clone()))


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("rows,dim", SHAPES8)
def test_swiglu8(rows, dim, dtype):
    from soap_tp_b200.ops import pack8, swiglu8, swiglu_linear8

    both = _rand(rows, 2 * dim, dtype=dtype, scale=2.0).requires_grad_()
    gate, up = both[:, :dim], both[:, dim:]            # halves of one projection
    y = swiglu8(gate, up)
    grad = _rand(rows, dim, seed=3, dtype=dtype)
    got = torch.autograd.grad(y, both, grad)[0]
    u = half_step(dtype)
    # exp to 2^-20 of itself and a quotient in the 16-bit forms; fp32 has the accurate ones
    c = 2.0 ** -18 if dtype != FP32 else 16 * F32 * (1 + 2.0 * gate.detach().double().abs())
    g, v = gate.detach().double(), up.detach().double()
    exact = torch.nn.functional.silu(g) * v
    within(y, (exact, (u + c) * exact.abs() + smallest(dtype)))

    def kept(t):
        packed = pack8(t.detach())
        return packed.values[:, :dim].double() * packed.scales.double().repeat_interleave(64, dim=1)[:, :dim]

    g, v, d = kept(gate), kept(up), grad.double()
    s = torch.sigmoid(g)
    c = 2.0 ** -18 if dtype != FP32 else 16 * F32 * (1 + 2.0 * g.abs())
    d_up, d_gate = d * g * s, d * v * s * (1 + g * (1 - s))
    within(got[:, dim:], (d_up, (u + c) * d_up.abs() + smallest(dtype)))
    within(got[:, :dim], (d_gate, u * d_gate.abs() + c * (d * v).abs() * s * (1 + g.abs()) + smallest(dtype)))
    # with the linear layer behind it: the same gradients from grad @ weight, and the kept activation for the weight's
    weight = _rand(5, dim, seed=4, dtype=dtype, scale=dim ** -0.5).requires_grad_()
    out_grad = _rand(rows, 5, seed=5, dtype=dtype)
    out = swiglu_linear8(gate, up, weight)
    assert torch.equal(out, torch.nn.functional.linear(y, weight))
    d_both, d_weight = torch.autograd.grad(out, (both, weight), out_grad)
    expected = torch.autograd.grad(swiglu8(gate, up), both, out_grad @ weight.detach())[0]
    assert torch.equal(d_both, expected)
    kept_y = g * s * v
    exact = out_grad.double().t() @ kept_y
    e = (u + c) * 1.01 * kept_y.abs()
    within(d_weight, (exact, u * exact.abs() + out_grad.double().abs().t() @ (e + rows * 2.0 ** -23 * kept_y.abs()) + smallest(dtype)))


def test_operators_are_differentiable_once():
    from soap_tp_b200 import ops

    x, b, gate, up = (_rand(4, 64, seed=i, dtype=BF16).requires_grad_() for i in range(4))
    hidden, weight, targets = _head(30, 64, 300, BF16)
    h, y = ops.residual_norm(x, b, torch.ones(64, device="cuda", dtype=BF16))
    outputs = [(h.float() * y.float()).sum(), ops.swiglu8(gate, up).float().sum(), ops.linear_cross_entropy(hidden, weight, targets),
               ops.swiglu_linear8(gate, up, x).float().sum()]
    for output, leaf in zip(outputs, (x, gate, hidden, up)):
        grad = torch.autograd.grad(output, leaf, create_graph=True)[0]
        assert grad.requires_grad
        with pytest.raises(RuntimeError, match="once"):
            grad.float().sum().backward()


# ---- streams, graphs, several at once -----------------------------------------------------------------------------------
def _step(hidden, weight, targets, x, branch, norm, gate, up):
    from soap_tp_b200 import ops

    h, y = ops.residual_norm(x, branch, norm, scale=0.5)
    act = ops.swiglu8(gate, up)
    loss = ops.linear_cross_entropy(hidden, weight, targets, workspace_bytes=1)
    total = loss + (h.float() * y.float()).mean() + act.float().mean()
    return (loss, h, y, act) + torch.autograd.grad(total, (hidden, weight, x, branch, norm, gate, up))


def _step_inputs(seed):
    hidden, weight, targets = _head(300, 72, 400, BF16, seed=seed, ignored=0.2)
    x, branch, gate, up = (_rand(40, 136, seed=seed + 10 + i, dtype=BF16).requires_grad_() for i in range(4))
    norm = (1 + _rand(136, seed=seed + 20, scale=0.1)).to(BF16).requires_grad_()
    return [hidden, weight, targets, x, branch, norm, gate, up]


def test_graph_replays_with_new_inputs_and_other_graphs_between():
    graphs = []
    for seed in (0, 100):
        inputs = _step_inputs(seed)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            for _ in range(2):
                _step(*inputs)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outputs = _step(*inputs)
        graphs.append((graph, inputs, outputs))
    for seed in (200, 300):
        for graph, inputs, _ in graphs:
            with torch.no_grad():
                for old, new in zip(inputs, _step_inputs(seed)):
                    old.copy_(new)
        for graph, _, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        expected = _step(*_step_inputs(seed))
        for _, _, outputs in graphs:
            for a, b in zip(outputs, expected):
                assert torch.equal(a, b)


def test_results_are_the_same_on_every_stream_and_run():
    inputs = _step_inputs(7)
    expected = _step(*inputs)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    results = []
    for _ in range(3):
        for stream in streams:
            stream.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(stream):
                results.append(_step(*inputs))
    torch.cuda.synchronize()
    for result in results:
        for a, b in zip(result, expected):
            assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_operators_under_autocast(dtype):
    """swiglu_linear8 and checkpoint8 are what they are without it, or with it around both runs."""
    from soap_tp_b200.ops import checkpoint8, pack8, swiglu_linear8, unpack8

    gate, up, weight = (_rand(*shape, dtype=dtype).requires_grad_() for shape in ((40, 136), (40, 136), (72, 136)))
    direction = _rand(40, 72, dtype=dtype)
    plain = swiglu_linear8(gate, up, weight)
    wanted = torch.autograd.grad(plain, (gate, up, weight), direction)
    with torch.autocast("cuda", dtype=FP16):
        y = swiglu_linear8(gate, up, weight)
    for a, b in zip((y, *torch.autograd.grad(y, (gate, up, weight), direction)), (plain, *wanted)):
        assert a.dtype == dtype and torch.equal(a, b)
    with torch.no_grad(), torch.autocast("cuda", dtype=FP16):
        assert torch.equal(swiglu_linear8(gate, up, weight), plain)

    kept, direction = unpack8(pack8(gate)).requires_grad_(), direction.half()
    with torch.autocast("cuda", dtype=FP16):
        wanted = torch.autograd.grad(torch.nn.functional.linear(kept, weight), (kept, weight), direction)
        y = checkpoint8(lambda x, w: torch.nn.functional.linear(x, w), gate, weight)
    for a, b in zip(torch.autograd.grad(y, (gate, weight), direction), wanted):
        assert y.dtype == FP16 and torch.equal(a, b)
