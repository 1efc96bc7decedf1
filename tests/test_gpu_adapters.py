"""Adapters of many requests against the formula in 64 bits.

Bounds, for sums of K products of numbers split to at least 21 bits: every product is off by 2^-21 of itself at most, every
addition rounds by up to 2^-23 of the running sum (the tensor core's additions cut off).  An element is therefore off by at most
(4 * 2^-21 + (K + R + 8) * 2^-23) times the sum of its terms' magnitudes, and a tensor, whose roundings are mostly independent, by
2^-19 + (2 sqrt(K) + K / 8) * 2^-23 of its 2-norm; half a unit in the last place of the type comes on top."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
F, B, H = torch.float32, torch.bfloat16, torch.float16
UNIT = {F: 2.0 ** -24, B: 2.0 ** -8, H: 2.0 ** -11}
LEAST = {F: 2.0 ** -149, B: 2.0 ** -133, H: 2.0 ** -24}


def _check(got, ref, size, terms, what):
    d, unit = (got.double() - ref).abs(), UNIT[got.dtype]
    limit = (4 * 2.0 ** -21 + (terms + 8) * 2.0 ** -23) * size + unit * ref.abs() + LEAST[got.dtype]
    assert bool((d <= limit).all()), "%s: element off by %g of its bound" % (what, float((d / limit).max()))
    if ref.numel() and float(ref.norm()):
        rel = float(d.norm() / ref.norm())
        # values below the normal range of 16-bit floats round by an absolute amount
        floor = LEAST[got.dtype] * math.sqrt(ref.numel()) / float(ref.norm())
        assert rel <= 2.0 ** -19 + (2 * math.sqrt(terms) + terms / 8) * 2.0 ** -23 + unit + floor, "%s: off by %g" % (what, rel)


def _formula(x, base, down, up, scale, ids, grad=None):
    """The operator and its gradients in 64 bits, and for each the sum of its terms' magnitudes."""
    x, down, up, scale = x.double(), down.double(), up.double(), scale.double()
    n = up.shape[2]
    y = base.double().clone() if base is not None else x.new_zeros(len(x), n)
    out = {"y": [y, y.abs()]}
    if grad is not None:
        grad = grad.double()
        out.update({k: [torch.zeros_like(v), torch.zeros_like(v)] for k, v in (("x", x), ("down", down), ("up", up))})
    for a in range(len(down)):
        at = torch.nonzero(ids == a)[:, 0]
        for i, (xa, d, u, s, g) in enumerate(((x[at], down[a], up[a], scale[a], grad[at] if grad is not None else None),
                                              (x[at].abs(), down[a].abs(), up[a].abs(), scale[a].abs(),
                                               grad[at].abs() if grad is not None else None))):
            h = xa @ d.T
            out["y"][i][at] += s * (h @ u)
            if grad is not None:
                dh = s * (g @ u.T)
                out["x"][i][at] = dh @ d
                out["down"][i][a] = dh.T @ xa
                out["up"][i][a] = s * (h.T @ g)
    return out


def _make(rows, k, n, rank, count, xt, wt, seed=0, layout="random"):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    ids = torch.randint(-1, count, (rows,), generator=g, device="cuda", dtype=torch.int32)
    if layout == "sorted":
        ids = ids.sort().values
    elif layout == "one":
        ids = torch.full_like(ids, count - 1)
    elif layout == "none":
        ids = torch.full_like(ids, -1)
    return dict(x=r(rows, k).to(xt), base=r(rows, n).to(xt), down=(r(count, rank, k) / math.sqrt(k)).to(wt),
                up=(r(count, rank, n) / math.sqrt(rank)).to(wt), scale=torch.rand(count, generator=g, device="cuda") + 0.5,
                ids=ids.contiguous(), grad=r(rows, n).to(xt))


PAIRS = [(F, F), (F, B), (F, H), (B, B), (H, H), (B, F), (H, F)]
SHAPES = [  # rows, k, n, rank, count, layout
    (1, 64, 64, 8, 1, "one"), (1, 1, 1, 1, 1, "one"), (3, 40, 24, 4, 2, "random"), (16, 512, 512, 16, 4, "random"),
    (33, 100, 71, 5, 7, "random"), (64, 1024, 256, 16, 64, "random"), (17, 8, 1000, 64, 3, "sorted"), (130, 264, 136, 33, 9, "sorted"),
    (513, 72, 64, 24, 2, "random"), (600, 333, 130, 7, 5, "sorted"), (700, 128, 192, 72, 3, "one"), (50, 16, 16, 8, 300, "random"),
    (40, 24, 40, 8, 6, "none"), (2000, 96, 80, 32, 40, "random"), (5, 2048, 24, 130, 2, "random"),
]


@pytest.mark.parametrize("pair", PAIRS, ids=lambda p: "-".join(str(t)[6:] for t in p))
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_forward_and_backward(cuda_device, pair, shape):
    from deepshift_b200 import adapters
    rows, k, n, rank, count, layout = shape
    s = _make(rows, k, n, rank, count, *pair, layout=layout)
    plan = adapters.plan_rows(s["ids"], count)
    want = _formula(s["x"], s["base"], s["down"], s["up"], s["scale"], s["ids"], s["grad"])
    y = adapters.apply(s["x"], s["down"], s["up"], s["scale"], plan, base=s["base"])
    assert y.dtype == s["x"].dtype
    _check(y, *want["y"], k + rank, "y")
    none = s["ids"] == -1
    assert torch.equal(y[none], s["base"][none])
    leaves = [t.clone().requires_grad_(True) for t in (s["x"], s["down"], s["up"], s["base"])]
    y2 = adapters.apply(leaves[0], leaves[1], leaves[2], s["scale"], plan, base=leaves[3])
    assert torch.equal(y2, y)
    dx, ddown, dup, dbase = torch.autograd.grad(y2, leaves, s["grad"])
    assert torch.equal(dbase, s["grad"])
    most = int(torch.bincount(s["ids"].long() + 1, minlength=2)[1:].max())
    _check(dx, *want["x"], n + rank, "dx")
    _check(ddown, *want["down"], n + most, "ddown")
    _check(dup, *want["up"], k + most, "dup")
    again = torch.autograd.grad(adapters.apply(*leaves[:3], s["scale"], plan, base=leaves[3]), leaves[:3], s["grad"])
    assert all(torch.equal(a, b) for a, b in zip(again, (dx, ddown, dup)))


@pytest.mark.parametrize("pair", [(F, F), (B, B)], ids=["f32", "bf16"])
def test_strides_in_place_and_without_base(cuda_device, pair):
    from deepshift_b200 import adapters
    s = _make(50, 48, 40, 8, 3, *pair, seed=2)
    plan = adapters.plan_rows(s["ids"], 3)
    args = (s["down"], s["up"], s["scale"], plan)
    y = adapters.apply(s["x"], *args, base=s["base"])
    for pad in (8, 3):   # rows apart by a multiple of 16 bytes, and by none
        wide = torch.zeros(50, 48 + pad, dtype=pair[0], device="cuda")
        wide[:, pad:] = s["x"]
        out = torch.full((50, 40 + pad), 9, dtype=pair[0], device="cuda")
        base = torch.zeros(50, 41 + pad, dtype=pair[0], device="cuda")[:, 1:41]
        base.copy_(s["base"])
        got = adapters.apply(wide[:, pad:], *args, base=base, out=out[:, pad:])
        assert got.data_ptr() == out[:, pad:].data_ptr()
        _check(out[:, pad:], *_formula(s["x"], s["base"], *args[:3], s["ids"])["y"], 56, "strided")
        assert bool((out[:, :pad] == 9).all())
    inplace = s["base"].clone()
    adapters.apply(s["x"], *args, base=inplace, out=inplace)
    assert torch.equal(inplace, y)
    alone = adapters.apply(s["x"], *args)
    _check(alone, *_formula(s["x"], None, *args[:3], s["ids"])["y"], 56, "without base")
    assert float(alone[s["ids"] == -1].abs().sum()) == 0.0
    folded = adapters.apply(s["x"].view(5, 10, 48), *args, base=s["base"].view(5, 10, 40))
    assert folded.shape == (5, 10, 40) and torch.equal(folded.view(50, 40), y)


def test_gradient_against_differences(cuda_device):
    """fp32 throughout; the loss is linear in each argument alone, so a central difference has no error of its own: what is left is the
    roundings of the two losses, 2^-19 of the sum of magnitudes each, over twice the step."""
    from deepshift_b200 import adapters
    s = _make(20, 24, 16, 4, 3, F, F, seed=5)
    plan = adapters.plan_rows(s["ids"], 3)
    leaves = [s[e].clone().requires_grad_(True) for e in ("x", "down", "up")]
    y = adapters.apply(*leaves, s["scale"], plan, base=s["base"])
    grads = torch.autograd.grad(y, leaves, s["grad"])
    size = float((_formula(s["x"], s["base"], s["down"], s["up"], s["scale"], s["ids"])["y"][1] * s["grad"].abs().double()).sum())
    g = torch.Generator(device="cuda").manual_seed(6)
    for i, t in enumerate(leaves):
        step = torch.randn(t.shape, generator=g, device="cuda")
        loss = []
        for sign in (1.0, -1.0):
            args = [u.detach() for u in leaves]
            args[i] = args[i] + sign * step
            loss.append(float((adapters.apply(*args, s["scale"], plan, base=s["base"]).double() * s["grad"].double()).sum()))
        want = float((grads[i].double() * step.double()).sum())
        assert abs((loss[0] - loss[1]) / 2 - want) <= 4 * 2.0 ** -19 * size


def test_masked_rows_may_hold_anything(cuda_device):
    from deepshift_b200 import adapters
    for xt, wt in PAIRS:
        s = _make(40, 64, 48, 8, 4, xt, wt, seed=3)
        plan = adapters.plan_rows(s["ids"], 4)
        clean = [t.clone().requires_grad_(True) for t in (s["x"], s["down"], s["up"])]
        y = adapters.apply(*clean, s["scale"], plan, base=s["base"])
        want = torch.autograd.grad(y, clean, s["grad"])
        none = s["ids"] == -1
        assert int(none.sum()) > 1
        x = s["x"].clone()
        x[none] = float("nan")
        x[torch.nonzero(none)[0]] = float("inf")
        grad = s["grad"].clone()
        grad[none] = float("nan")
        dirty = [t.clone().requires_grad_(True) for t in (x, s["down"], s["up"])]
        y2 = adapters.apply(*dirty, s["scale"], plan, base=s["base"])
        got = torch.autograd.grad(y2, dirty, grad)
        assert torch.equal(y2, y)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        # an adapter that no row uses
        none_left = adapters.plan_rows(torch.where(s["ids"] == 2, -1, s["ids"]), 4)
        down = s["down"].clone()
        down[2] = float("nan")
        leaves = [t.clone().requires_grad_(True) for t in (s["x"], down, s["up"])]
        got = torch.autograd.grad(adapters.apply(*leaves, s["scale"], none_left, base=s["base"]), leaves, s["grad"])
        assert float(got[1][2].abs().sum()) == 0 and float(got[2][2].abs().sum()) == 0
        assert all(bool(torch.isfinite(t.float()).all()) for t in got)


@pytest.mark.parametrize("rows,count", [(0, 3), (1, 1), (31, 2), (33, 255), (1000, 256), (1000, 5000), (40000, 70), (513, 65535)])
def test_plan(cuda_device, rows, count):
    from deepshift_b200 import adapters
    g = torch.Generator().manual_seed(rows + count)
    ids = torch.randint(-1, count, (rows,), generator=g, dtype=torch.int32)
    for given in (ids.cuda(), ids.long().cuda(), ids, ids.tolist()):
        plan = adapters.plan_rows(given, count)
        assert plan.invalid() == 0
    key = torch.where(ids < 0, count, ids)
    words = plan.data.cpu()
    tile_rows = 16 if rows <= 512 else 128
    offsets = words[4:4 + count + 2]
    assert torch.equal(offsets, torch.searchsorted(key.sort().values, torch.arange(count + 2, dtype=torch.int32)).int())
    at = (4 + count + 2 + 3) // 4 * 4
    most = rows // tile_rows + min(rows, count + 1)
    order = words[at + 4 * most:at + 4 * most + rows]
    assert torch.equal(order.long(), key.sort(stable=True).indices)
    tiles = words[at:at + 4 * int(words[0])].view(-1, 4).tolist()
    want = []
    for a in torch.unique(key).tolist():
        lo, hi = int(offsets[a]), int(offsets[a + 1])
        want += [[a, p, min(tile_rows, hi - p), 0] for p in range(lo, hi, tile_rows)]
    assert tiles == want and len(tiles) <= most


def test_invalid_indices_count_as_none(cuda_device):
    from deepshift_b200 import adapters
    s = _make(20, 16, 16, 4, 3, F, F)
    ids = s["ids"].clone().long()
    ids[4], ids[7], ids[9] = 3, -2, 1 << 40
    plan = adapters.plan_rows(ids, 3)
    assert plan.invalid() == 3
    y = adapters.apply(s["x"], s["down"], s["up"], s["scale"], plan, base=s["base"])
    assert torch.equal(y[[4, 7, 9]], s["base"][[4, 7, 9]])
    with pytest.raises(RuntimeError):
        adapters.plan_rows([0, 3], 3)


def test_no_rows(cuda_device):
    from deepshift_b200 import adapters
    s = _make(0, 16, 24, 4, 3, F, F)
    leaves = [s[e].clone().requires_grad_(True) for e in ("x", "down", "up")]
    y = adapters.apply(*leaves, s["scale"], adapters.plan_rows(s["ids"], 3), base=s["base"])
    got = torch.autograd.grad(y, leaves, s["grad"])
    assert y.shape == (0, 24) and all(float(t.abs().sum()) == 0 for t in got)


def test_offsets_beyond_32_bits(cuda_device):
    """Rows that begin more than 2^31 elements into their tensor."""
    from deepshift_b200 import adapters
    stride = (1 << 31) // 40
    x = torch.zeros(41 * stride, dtype=B, device="cuda").view(41, stride)[:, :16]
    s = _make(41, 16, 16, 8, 2, B, B, seed=8)
    x.copy_(s["x"])
    plan = adapters.plan_rows(s["ids"], 2)
    got = adapters.apply(x, s["down"], s["up"], s["scale"], plan, base=s["base"])
    assert torch.equal(got, adapters.apply(s["x"], s["down"], s["up"], s["scale"], plan, base=s["base"]))


def test_other_stream_and_graph(cuda_device):
    from deepshift_b200 import adapters
    s = _make(30, 64, 64, 8, 4, F, B, seed=4)
    want = _formula(s["x"], s["base"], s["down"], s["up"], s["scale"], s["ids"])["y"]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        plan = adapters.plan_rows(s["ids"], 4)
        y = adapters.apply(s["x"], s["down"], s["up"], s["scale"], plan, base=s["base"])
    stream.synchronize()
    _check(y, *want, 72, "side stream")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        plan = adapters.plan_rows(s["ids"], 4)
        y = adapters.apply(s["x"], s["down"], s["up"], s["scale"], plan, base=s["base"])
    s["ids"].copy_(s["ids"].flip(0))   # the graph sorts the rows anew
    s["x"].mul_(2)
    graph.replay()
    torch.cuda.synchronize()
    _check(y, *_formula(s["x"], s["base"], s["down"], s["up"], s["scale"], s["ids"])["y"], 72, "replayed")


def test_beside_a_shift_layer(cuda_device):
    from deepshift_b200 import adapters, modules
    torch.manual_seed(0)
    shift = modules.LinearShift(64, 48, use_kernel=True, act_integer_bits=4, act_fraction_bits=12).cuda()
    layer = adapters.AdaptedLinear(shift, 3, 4, alpha=8, device="cuda")
    x = torch.randn(10, 64, device="cuda")
    plan = adapters.plan_rows(torch.tensor([0, 1, 2, -1, 0, 0, 1, 2, 2, -1], device="cuda"), 3)
    with torch.no_grad():
        assert torch.equal(layer(x, plan), shift(x))
        layer.up.normal_()
        want = _formula(x, shift(x), layer.down, layer.up, layer.scale, torch.tensor([0, 1, 2, -1, 0, 0, 1, 2, 2, -1], device="cuda"))
        _check(layer(x, plan), *want["y"], 68, "layer")
    leaf = x.clone().requires_grad_(True)
    layer(leaf, plan).sum().backward()
    own = shift._float_weight().sum(0)
    assert torch.allclose(leaf.grad[3], own, rtol=1e-6, atol=1e-6)   # a row without an adapter: the frozen layer's part alone
    assert layer.down.grad is not None and layer.up.grad is not None
    assert all(p.grad is None for p in shift.parameters())


def test_refusals(cuda_device):
    from deepshift_b200 import adapters
    s = _make(10, 16, 24, 4, 3, F, F)
    plan = adapters.plan_rows(s["ids"], 3)
    good = dict(x=s["x"], down=s["down"], up=s["up"], scale=s["scale"], plan=plan, base=s["base"], out=None)
    adapters.apply(**good)
    for bad in (dict(x=s["x"].cpu()), dict(x=s["x"].double()), dict(x=s["x"][:9]), dict(x=s["x"][:, :15]), dict(x=s["x"].half(), down=s["down"].bfloat16()),
                dict(down=s["down"].transpose(1, 2)), dict(down=s["down"][:2]), dict(up=s["up"].half()), dict(up=s["up"][:, :3]),
                dict(scale=s["scale"][:2]), dict(scale=s["scale"].double()), dict(base=s["base"].half()), dict(base=s["base"][:, :8]),
                dict(base=s["base"].t().contiguous().t()), dict(out=torch.empty(10, 23, device="cuda")),
                dict(plan=adapters.plan_rows(s["ids"], 4)), dict(plan=adapters.plan_rows(s["ids"][:4], 3)),
                dict(down=torch.zeros(3, 257, 16, device="cuda"), up=torch.zeros(3, 257, 24, device="cuda")),
                dict(x=s["x"].clone().requires_grad_(True), out=torch.empty(10, 24, device="cuda"))):
        with pytest.raises(RuntimeError):
            adapters.apply(**{**good, **bad})
    for ids, count in ((s["ids"].float(), 3), (s["ids"].view(2, 5), 3), (s["ids"], 0), (s["ids"], 70000)):
        with pytest.raises(RuntimeError):
            adapters.plan_rows(ids, count)
