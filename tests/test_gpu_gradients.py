"""Global norm and clipping against the formula in 64 bits.

Bounds.  The norm: squares are summed by eights in fp32 (eight roundings of 2^-24 each, at most 2^-21 of a sum of
positive numbers), the sums in double, the root and the conversion to fp32 round once more: 2^-21 in all, with room.  A scaled
value: the norm's error, the factor's two roundings and the product's, 2^-20, then half a unit in the last place of its type."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
NORM, SCALED = 2.0 ** -21, 2.0 ** -20
UNIT = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
LEAST = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}


def _expected(tensors, max_norm):
    norm = math.sqrt(math.fsum(float(t.double().square().sum()) for t in tensors))
    return norm, min(1.0, max_norm / (norm + 1e-6))


def _check(tensors, out, norm, max_norm, before):
    want, factor = _expected(before, max_norm)
    assert abs(float(norm) - want) <= NORM * want
    for b, o in zip(before, out):
        ref = b.double() * factor
        assert torch.all((o.double() - ref).abs() <= (SCALED + UNIT[o.dtype]) * ref.abs() + LEAST[o.dtype]), o.shape


def _make(sizes, dtypes, seed, std=0.1):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [(torch.randn(n, generator=g, device="cuda") * std).to(dtypes[i % len(dtypes)]) for i, n in enumerate(sizes)]


F, B, H = torch.float32, torch.bfloat16, torch.float16


@pytest.mark.parametrize("sizes", [[1], [7], [8192], [8193, 1, 0, 31], [5] * 32, [65] * 33, [100, 3] * 300, [1 << 20, 9]])
@pytest.mark.parametrize("dtypes", [(F,), (B,), (H,), (F, B, H)])
@pytest.mark.parametrize("share", [0.25, 4.0])
def test_in_place_and_out_of_place(cuda_device, sizes, dtypes, share):
    from deepshift_b200 import gradients
    tensors = _make(sizes, dtypes, 1)
    before = [t.clone() for t in tensors]
    max_norm = share * _expected(before, 1.0)[0]
    out = [torch.full_like(t, 7) for t in tensors]
    norm = gradients.clip_norm(tensors, max_norm, out=out)
    assert all(torch.equal(a, b) for a, b in zip(tensors, before))
    _check(tensors, out, norm, max_norm, before)
    wide = [torch.full(t.shape, 7.0, device="cuda") for t in tensors]
    gradients.clip_norm(tensors, max_norm, out=wide)
    _check(tensors, wide, norm, max_norm, before)
    again = gradients.clip_norm(tensors, max_norm)
    assert torch.equal(again, norm) and torch.equal(gradients.global_norm(before), norm)
    assert all(torch.equal(a, b) for a, b in zip(tensors, out))
    if share > 1:
        assert all(torch.equal(a, b) for a, b in zip(tensors, before))


@pytest.mark.parametrize("value", [0.0, 1e-30, 1e-22, 1e25, 3e38])
def test_values_whose_squares_leave_fp32(cuda_device, value):
    from deepshift_b200 import gradients
    t = [torch.full((n,), value, device="cuda") for n in (3, 20000)]
    want = value * math.sqrt(20003)
    norm = float(gradients.global_norm(t))
    assert norm == math.inf if want > 3.5e38 else abs(norm - want) <= NORM * want
    small = [torch.tensor([1e25, 1e-25, 1.0], device="cuda"), torch.tensor([1e-25], device="cuda")]
    assert abs(float(gradients.global_norm(small)) - 1e25) <= NORM * 1e25


def test_non_finite(cuda_device):
    from deepshift_b200 import gradients
    a, b = torch.tensor([1.0, math.inf], device="cuda"), torch.ones(5, device="cuda")
    assert float(gradients.clip_norm([a, b], 1.0)) == math.inf
    assert float(a[0]) == 0.0 and math.isnan(float(a[1])) and float(b.abs().max()) == 0.0
    a, b = torch.tensor([1.0, math.nan], device="cuda"), torch.ones(5, device="cuda")
    assert math.isnan(float(gradients.clip_norm([a, b], 1.0)))
    assert bool(torch.isnan(a).all()) and bool(torch.isnan(b).all())


def test_layouts_offsets_and_parameters(cuda_device):
    from deepshift_b200 import gradients
    whole = _make([1003], (B,), 3)[0]
    tensors = [whole[3:500], whole[501:1003], torch.randn(6, 4, 5, device="cuda").permute(2, 0, 1),
               torch.randn(2, 3, 4, 4, device="cuda").contiguous(memory_format=torch.channels_last), torch.randn((), device="cuda")]
    kept = whole[500].clone()
    before = [t.clone() for t in tensors]
    norm = gradients.clip_norm(tensors, 0.5)
    _check(tensors, tensors, norm, 0.5, before)
    assert torch.equal(whole[500], kept)
    p = [torch.nn.Parameter(torch.zeros(n, device="cuda")) for n in (4, 5, 6)]
    p[0].grad, p[2].grad = torch.ones(4, device="cuda"), torch.ones(6, device="cuda")
    assert abs(float(gradients.clip_grad_norm_(p, 1.0)) - math.sqrt(10)) <= NORM * 4
    assert p[1].grad is None
    assert abs(float(gradients.global_norm([p[0].grad, p[2].grad])) - 1.0) < 1e-5
    assert float(gradients.clip_norm([], 1.0)) == 0.0


def test_other_stream_and_graph(cuda_device):
    from deepshift_b200 import gradients
    tensors = _make([4000, 33], (F,), 4)
    out = [torch.empty_like(t) for t in tensors]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        norm = gradients.clip_norm(tensors, 0.1, out=out)
    s.synchronize()
    _check(tensors, out, norm, 0.1, tensors)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = gradients.clip_norm(tensors, 0.1, out=out)
    tensors[0].mul_(3)
    graph.replay()
    torch.cuda.synchronize()
    _check(tensors, out, captured, 0.1, tensors)


def test_refusals(cuda_device):
    from deepshift_b200 import gradients
    a = torch.ones(8, device="cuda")
    for bad in (-1.0, math.nan):
        with pytest.raises(ValueError):
            gradients.clip_norm([a], bad)
    for tensors, out in (([torch.ones(3)], None), ([a.double()], None), ([a[::2]], None), ([a, a], None), ([a], []),
                         ([a], [torch.ones(7, device="cuda")]), ([a], [a.long()]), ([a, torch.ones(3)], None),
                         ([torch.ones(4, 2, device="cuda")], [torch.ones(2, 4, device="cuda").t()])):
        with pytest.raises(RuntimeError):
            gradients.clip_norm(tensors, 1.0, out=out)
    assert torch.equal(a, torch.ones(8, device="cuda"))
