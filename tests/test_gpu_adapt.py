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
