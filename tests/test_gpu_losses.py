"""Cross entropy of a linear head without its logits against the formula in 64 bits.

Bounds.  A logit: the products of 16-bit numbers are exact in fp32, sixteen of them are added and cut off once at 2^-23 of
the running sum, so it is off by at most e = (d / 16 + 4) 2^-23 times the largest sum of its terms' magnitudes in the row.  A loss is
off by 2 e (the maximum and the sum of exponentials move with the logits), and by 2^-20 of log(v) and of itself.
A probability is off by (2 e + 2^-19) of itself; its gradient is rounded to 16 bits (u = 2^-8 or 2^-11), the products add a
term of (terms / 16 + 4) 2^-23 of the sum of magnitudes for each piece, and the result is rounded to 16 bits once more."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
B, H = torch.bfloat16, torch.float16
UNIT = {B: 2.0 ** -8, H: 2.0 ** -11}
LEAST = {B: 2.0 ** -133, H: 2.0 ** -24}


def _make(rows, d, v, dtype, seed=0, ignore=-100, share=0.2):
    g = torch.Generator(device="cuda").manual_seed(seed)
    weight = (torch.randn(v, d, generator=g, device="cuda") * 2 / math.sqrt(d)).to(dtype)
    target = torch.randint(0, v, (rows,), generator=g, device="cuda")
    hidden = (torch.randn(rows, d, generator=g, device="cuda") + torch.rand(rows, 1, generator=g, device="cuda") * weight[target].float()).to(dtype)
    if rows > 1:
        target[torch.rand(rows, generator=g, device="cuda") < share] = ignore
    return hidden, weight, target


def _formula(hidden, weight, target, ignore=-100):
    h, w = hidden.double(), weight.double()
    z = h @ w.T
    size = (h.abs() @ w.abs().T).max(1).values
    lse = torch.logsumexp(z, 1)
    live = target != ignore
    at = torch.where(live, target, torch.zeros_like(target))
    each = torch.where(live, lse - z.gather(1, at[:, None])[:, 0], torch.zeros_like(lse))
    p = torch.exp(z - lse[:, None])
    e = (h.size(1) / 16 + 4) * 2.0 ** -23 * size
    return each, live, at, p, e


def _check_each(got, hidden, weight, target, ignore=-100):
    each, live, at, p, e = _formula(hidden, weight, target, ignore)
    assert got.dtype == torch.float32
    limit = 2 * e + 2.0 ** -20 * (each.abs() + math.log(weight.size(0)) + 1)
    assert bool(((got.double() - each).abs() <= limit).all()), float(((got.double() - each).abs() / limit).max())
    assert float(got[~live].abs().sum()) == 0


def _check_gradients(dh, dw, hidden, weight, target, row_grad, ignore=-100, pieces=1):
    """row_grad: gradient of each row's loss, in 64 bits."""
    each, live, at, p, e = _formula(hidden, weight, target, ignore)
    unit, least = UNIT[hidden.dtype], LEAST[hidden.dtype]
    g = p.clone()
    g[torch.arange(len(at), device=at.device), at] -= 1
    factor = (live.double() * row_grad)[:, None]
    # numbers so small that 16 bits cannot hold them keep an absolute error: the least one, of a largest weight of 1 or 2^15
    most = float(row_grad.abs().max()) * (1.0 if hidden.dtype == B else 2.0 ** -15)
    off = (unit * g.abs() + p * (2 * e[:, None] + 2.0 ** -19)) * factor.abs() + least * most
    g = g * factor
    for got, a, b, terms in ((dh, g, weight.double(), weight.size(0)), (dw, g.T, hidden.double(), len(at))):
        ref = a @ b
        slack = (off if got is dh else off.T) @ b.abs() + pieces * (terms / 16 + 4) * 2.0 ** -23 * (a.abs() @ b.abs())
        limit = slack * 1.01 + unit * ref.abs() + least
        d = (got.double() - ref).abs()
        assert bool((d <= limit).all()), float((d / limit).max())
        if float(ref.norm()) and hidden.dtype == B:   # roundings are independent: in the 2-norm they add up as squares
            assert float(d.norm() / ref.norm()) <= 1.5 * unit


SHAPES = [(1, 8, 1), (1, 64, 100), (2, 16, 2), (5, 9, 33), (16, 512, 1000), (127, 72, 129), (128, 64, 128), (129, 64, 257), (200, 520, 999),
          (257, 136, 2049), (300, 1, 300), (513, 100, 512), (777, 264, 3001), (40, 2048, 5000), (1000, 33, 130)]


@pytest.mark.parametrize("dtype", [B, H], ids=["bf16", "f16"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_loss_and_gradients(cuda_device, shape, dtype, reduction):
    from deepshift_b200 import losses
    hidden, weight, target = _make(*shape, dtype, seed=sum(shape))
    live = target != -100
    each = losses.linear_cross_entropy(hidden, weight, target, reduction="none")
    _check_each(each, hidden, weight, target)
    leaves = hidden.clone().requires_grad_(True), weight.clone().requires_grad_(True)
    loss = losses.linear_cross_entropy(*leaves, target, reduction=reduction)
    count = int(live.sum())
    if reduction == "none":
        assert torch.equal(loss, each)
        grad = torch.randn(len(target), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)) * 3
        row_grad = grad.double()
    else:
        want = float(each.double().sum()) / (count if reduction == "mean" else 1)
        assert abs(float(loss.detach()) - want) <= 2.0 ** -23 * abs(want)
        grad = torch.tensor(0.7, device="cuda")
        row_grad = torch.full((len(target),), float(grad) / (count if reduction == "mean" else 1), device="cuda", dtype=torch.float64)
    dh, dw = torch.autograd.grad(loss, leaves, grad)
    assert dh.dtype == dtype and dw.dtype == dtype
    _check_gradients(dh, dw, hidden, weight, target, row_grad)
    assert float(dh[~live].abs().sum()) == 0
    again = torch.autograd.grad(losses.linear_cross_entropy(*leaves, target, reduction=reduction), leaves, grad)
    assert torch.equal(again[0], dh) and torch.equal(again[1], dw)


def test_several_pieces_of_the_vocabulary(cuda_device):
    from deepshift_b200 import _ffi, losses
    rows, d, v = 20000, 72, 14001
    hidden, weight, target = _make(rows, d, v, B)
    # scratch of whole G would be 560 MB: there are three pieces
    assert _ffi.lib().ds_loss_bytes(rows, d, v, 1, 0) < 2 * rows * v
    leaves = hidden.clone().requires_grad_(True), weight.clone().requires_grad_(True)
    loss = losses.linear_cross_entropy(*leaves, target)
    dh, dw = torch.autograd.grad(loss, leaves)
    row_grad = torch.full((rows,), 1.0 / int((target != -100).sum()), device="cuda", dtype=torch.float64)
    _check_gradients(dh, dw, hidden, weight, target, row_grad, pieces=3)
    only_h = torch.autograd.grad(losses.linear_cross_entropy(leaves[0], weight, target), leaves[0])[0]
    only_w = torch.autograd.grad(losses.linear_cross_entropy(hidden, leaves[1], target), leaves[1])[0]
    assert torch.equal(only_h, dh) and torch.equal(only_w, dw)


@pytest.mark.parametrize("dtype", [B, H], ids=["bf16", "f16"])
def test_gradient_against_differences(cuda_device, dtype):
    """Along a direction of 16-bit steps; the loss is smooth, so the central difference is off by step^2 / 6 of a third derivative, which is
    at most the cube of the logits' change: 2^3 x 0.1 here, beside the gradients' own rounding to 16 bits."""
    from deepshift_b200 import losses
    hidden, weight, target = _make(60, 64, 200, dtype, seed=3)
    leaves = hidden.clone().requires_grad_(True), weight.clone().requires_grad_(True)
    grads = torch.autograd.grad(losses.linear_cross_entropy(*leaves, target, reduction="sum"), leaves)
    for i in range(2):
        g = torch.Generator(device="cuda").manual_seed(4 + i)
        step = torch.randn(leaves[i].shape, generator=g, device="cuda") * 0.02
        up = [t.detach().float() for t in leaves]
        ends = []
        for sign in (1, -1):
            args = [t.detach() for t in leaves]
            args[i] = (args[i].float() + sign * step).to(dtype)
            ends.append((args[i].double(), float(losses.linear_cross_entropy(*args, target, reduction="sum").double())))
        moved = ends[0][0] - ends[1][0]     # the steps as they were rounded
        want = float((grads[i].double() * moved).sum())
        size = float((grads[i].double() * moved).norm())
        assert abs((ends[0][1] - ends[1][1]) - want) <= 0.02 * size + 0.05, (ends[0][1] - ends[1][1], want)


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_no_row_counts(cuda_device, reduction):
    from deepshift_b200 import losses
    hidden, weight, target = _make(20, 64, 50, B)
    target.fill_(-100)
    leaves = hidden.requires_grad_(True), weight.requires_grad_(True)
    loss = losses.linear_cross_entropy(*leaves, target, reduction=reduction)
    if reduction == "mean":
        assert math.isnan(float(loss))
    else:
        assert float(loss.sum()) == 0
    dh, dw = torch.autograd.grad(loss.sum(), leaves)
    assert float(dh.abs().sum()) == 0 and float(dw.abs().sum()) == 0


def test_ignored_rows_may_hold_anything(cuda_device):
    from deepshift_b200 import losses
    for dtype in (B, H):
        hidden, weight, target = _make(150, 64, 300, dtype, ignore=7)
        target[target == 8] = 9
        ignored = target == 7
        assert int(ignored.sum()) > 3
        leaves = hidden.clone().requires_grad_(True), weight.clone().requires_grad_(True)
        loss = losses.linear_cross_entropy(*leaves, target, ignore_index=7)
        want = torch.autograd.grad(loss, leaves)
        big = hidden.clone()
        big[ignored] = torch.finfo(dtype).max
        leaves = big.requires_grad_(True), weight.clone().requires_grad_(True)
        loss2 = losses.linear_cross_entropy(*leaves, target, ignore_index=7)
        got = torch.autograd.grad(loss2, leaves)
        assert torch.equal(loss, loss2) and torch.equal(got[0], want[0])
        assert bool(torch.isfinite(got[1].float()).all()) and torch.equal(got[1], want[1])


def test_extreme_logits_and_targets(cuda_device):
    from deepshift_b200 import losses
    # logits of +-3 10^4: exponentials of all but the largest vanish
    hidden = torch.tensor([[200.0] * 8, [-200.0] * 8], dtype=B, device="cuda")
    weight = torch.tensor([[20.0] * 8, [-20.0] * 8, [0.0] * 8], dtype=B, device="cuda")
    each = losses.linear_cross_entropy(hidden, weight, torch.tensor([0, 0], device="cuda"), reduction="none")
    assert each.tolist() == [0.0, 64000.0]
    # a target that does not exist
    hidden, weight, _ = _make(4, 16, 10, B)
    leaves = hidden.requires_grad_(True), weight.requires_grad_(True)
    each = losses.linear_cross_entropy(*leaves, torch.tensor([1, 10, -1, -100], device="cuda"), reduction="none")
    assert torch.isnan(each).tolist() == [False, True, True, False]
    assert math.isnan(float(losses.linear_cross_entropy(*leaves, torch.tensor([1, 10, 2, -100], device="cuda"))))
    dh, dw = torch.autograd.grad(each.sum(), leaves)
    assert torch.isnan(dh).all(1).tolist() == [False, True, True, False] and bool(torch.isnan(dw).all())
    # a row of its own infinities is not a number, the others are not touched
    x = hidden.detach().clone()
    x[2, 3] = float("inf")
    each = losses.linear_cross_entropy(x, weight.detach(), torch.tensor([1, 2, 3, 4], device="cuda"), reduction="none")
    assert torch.isfinite(each).tolist() == [True, True, False, True]


def test_shapes_strides_offsets_and_types_of_target(cuda_device):
    from deepshift_b200 import losses
    hidden, weight, target = _make(60, 40, 90, B)
    want = losses.linear_cross_entropy(hidden, weight, target, reduction="none")
    folded = losses.linear_cross_entropy(hidden.view(4, 15, 40), weight, target.view(4, 15).int(), reduction="none")
    assert folded.shape == (4, 15) and torch.equal(folded.view(-1), want)
    off = torch.zeros(1 + hidden.numel(), dtype=B, device="cuda")[1:].view(60, 40)   # no 16-byte alignment
    off.copy_(hidden)
    leaves = off.detach().requires_grad_(True), weight.clone().requires_grad_(True)
    loss = losses.linear_cross_entropy(*leaves, target, reduction="none")
    assert torch.equal(loss, want)
    grads = torch.autograd.grad(loss.sum(), leaves)
    same = hidden.clone().requires_grad_(True), weight.clone().requires_grad_(True)
    ref = torch.autograd.grad(losses.linear_cross_entropy(*same, target, reduction="none").sum(), same)
    assert torch.equal(grads[0], ref[0]) and torch.equal(grads[1], ref[1])
    wide = torch.zeros(60, 80, dtype=B, device="cuda")
    wide[:, ::2] = hidden
    assert torch.equal(losses.linear_cross_entropy(wide[:, ::2], weight.t().contiguous().t(), target, reduction="none"), want)
    empty = losses.linear_cross_entropy(hidden[:0].clone().requires_grad_(True), same[1], target[:0], reduction="sum")
    assert float(empty) == 0 and float(torch.autograd.grad(empty, same[1])[0].abs().sum()) == 0


def test_other_stream_and_graph(cuda_device):
    from deepshift_b200 import losses
    hidden, weight, target = _make(150, 64, 300, B, seed=9)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        each = losses.linear_cross_entropy(hidden, weight, target, reduction="none")
    stream.synchronize()
    _check_each(each, hidden, weight, target)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        each = losses.linear_cross_entropy(hidden, weight, target, reduction="none")
    hidden.mul_(-1)
    graph.replay()
    torch.cuda.synchronize()
    _check_each(each, hidden, weight, target)


def test_refusals(cuda_device):
    from deepshift_b200 import losses
    hidden, weight, target = _make(10, 16, 20, B)
    with pytest.raises(ValueError):
        losses.linear_cross_entropy(hidden, weight, target, reduction="max")
    for args in ((hidden.cpu(), weight, target), (hidden.float(), weight.float(), target), (hidden, weight.half(), target),
                 (hidden, weight[:, :8], target), (hidden, weight[0], target), (hidden, weight, target[:9]), (hidden, weight, target.float()),
                 (hidden, weight, target.cpu()), (hidden, weight[:0], target)):
        with pytest.raises(RuntimeError):
            losses.linear_cross_entropy(*args)
