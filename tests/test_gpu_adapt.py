"""Adapters, loss and clipping together, as a program uses them."""
import pytest

pytestmark = pytest.mark.gpu


def test_training_and_serving(cuda_device, capsys):
    from deepshift_b200 import adapt
    curve, right, ids = adapt.main(["--steps", "40", "--rows", "1024"])
    assert "probability" in capsys.readouterr().out
    # from the logarithm of the vocabulary (a random head adds half the variance of its logits, 1/2) to a task that is learnt
    assert 8.0 < curve[0] < 9.6 and curve[-1] < 2.0
    # the rows of tasks answer theirs; one without an adapter knows none of 4000 tokens
    assert float(right[ids >= 0].mean()) > 0.3 and float(right[ids < 0].mean()) < 0.02


def test_the_clipping_holds(cuda_device):
    import torch
    from deepshift_b200 import adapt, adapters, gradients
    torch.manual_seed(1)
    model = adapt.AdaptedModel(1000, 64, 96, 3, 5)
    for layer in (model.into, model.back):
        torch.nn.init.normal_(layer.up)
    tokens, ids = torch.randint(0, 1000, (100,), device="cuda"), torch.randint(0, 3, (100,), device="cuda")
    model.loss(tokens, model.answer(tokens, ids), adapters.plan_rows(ids, 3)).backward()
    trained = [p for p in model.parameters() if p.requires_grad]
    assert len(trained) == 4 and all(p.grad is not None for p in trained)
    want = torch.sqrt(sum(p.grad.double().square().sum() for p in trained))
    norm = gradients.clip_grad_norm_(trained, 0.5 * float(want))
    assert abs(float(norm) / float(want) - 1) < 1e-6
    assert abs(float(gradients.global_norm([p.grad for p in trained])) / float(want) - 0.5) < 1e-5


def test_rows_answer_alone_as_in_a_batch(cuda_device):
    """A request's answer does not depend on what else is in its batch, beyond the rounding of differently ordered sums."""
    import torch
    from deepshift_b200 import adapt
    torch.manual_seed(2)
    model = adapt.AdaptedModel(1000, 64, 96, 3, 5)
    for layer in (model.into, model.back):
        torch.nn.init.normal_(layer.up, std=0.1)
    tokens, ids = torch.randint(0, 1000, (40,), device="cuda"), torch.arange(40, device="cuda") % 4 - 1
    together = adapt.serve(model, tokens, ids, 3)
    alone = torch.cat([adapt.serve(model, tokens[i:i + 1], ids[i:i + 1], 3) for i in range(40)])
    # hidden states are rounded to bfloat16 (2^-9) before the head: a logit of a few units may move by some 2^-9 of itself
    assert torch.allclose(together, alone, rtol=0.05, atol=0)


@pytest.mark.parametrize("rows, rank", [(1, 1), (17, 8), (512, 64)])
def test_products_without_keeping_the_inner_ones(cuda_device, rows, rank):
    """Up to 512 rows and a rank of 64 need no place for h; the result is the one with it, bit for bit."""
    import torch
    from deepshift_b200 import _ffi, adapters
    torch.manual_seed(rows)
    x, down, up, base = (torch.randn(s, device="cuda") for s in ((rows, 100), (3, rank, 100), (3, rank, 72), (rows, 72)))
    plan = adapters.plan_rows(torch.arange(rows) % 4 - 1, 3)
    with torch.no_grad():
        without = adapters.apply(x, down, up, None, plan, base=base)
    kept = adapters.apply(x, down.requires_grad_(True), up, None, plan, base=base)
    assert kept.requires_grad and torch.equal(without, kept)
    # more of either have to bring it
    for m, r in ((513, 8), (16, 65)):
        more = (torch.randn(s, device="cuda") for s in ((m, 100), (3, r, 100), (3, r, 72)))
        x, down, up = more
        plan = adapters.plan_rows(torch.arange(m) % 4 - 1, 3)
        out = torch.empty(m, 72, device="cuda")
        with pytest.raises(RuntimeError, match="bad argument"):
            _ffi.run("ds_adapters_apply", x.get_device(), _ffi.pack_adapters(
                m, 100, 72, r, 3, 0, 0, plan.data.data_ptr(), down.data_ptr(), up.data_ptr(), 0, x.data_ptr(), 100, 0, 0, out.data_ptr(), 72,
                0, 0, 0, 0, 0, 0, 0, 0, 0, 0))
