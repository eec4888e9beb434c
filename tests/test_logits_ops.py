"""Log probabilities and distillation off the GPU, where they are made of torch's operations; their refusals; what
looks through them."""

import math

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from _logits_oracle import distill, score
from _logits_strict import distill_by_formula, within
from fairring_b200.ops import distillation_loss, token_log_probs


def _logits(*shape, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * 3


@pytest.mark.parametrize("temperature", [1.0, 0.7])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16, torch.float64])
def test_log_probs(temperature, dtype):
    x = _logits(2, 5, 33).to(dtype).requires_grad_(True)
    x.data[0, 1, 3:9] = float("-inf")
    tokens = torch.tensor([[0, 32, -100, 4, -1], [1, 2, 3, 4, 5]])
    got = token_log_probs(x, tokens, temperature=temperature, entropy=True, top_k=4)
    g, h = torch.full((2, 5), 0.7), torch.full((2, 5), 0.3)
    want, want_h, want_grad, logp = score(x, tokens, temperature, g, h)
    torch.testing.assert_close(got.log_probs.double(), want, rtol=1e-6, atol=2e-6)  # a few roundings of values up to 16
    torch.testing.assert_close(got.entropy.double(), want_h, rtol=1e-6, atol=2e-6)
    (grad,) = torch.autograd.grad((got.log_probs * g).sum() + (got.entropy * h).sum(), x)
    torch.testing.assert_close(grad.double(), want_grad, rtol=torch.finfo(dtype).eps / 2 + 1e-6, atol=2e-6)
    order = x.detach().sort(dim=-1, descending=True, stable=True).indices[..., :4]
    counts = (tokens >= 0).unsqueeze(-1)
    assert torch.equal(got.top_tokens, order.where(counts, -1))
    torch.testing.assert_close(got.top_log_probs.double(), logp.gather(-1, order).where(counts, float("-inf")), rtol=1e-6, atol=2e-6)
    assert not got.top_log_probs.requires_grad


def test_rows_that_do_not_count_are_not_looked_at():
    x = _logits(3, 11)
    x[1], x[2, 4] = float("nan"), float("inf")
    leaf = x.requires_grad_(True)
    got = token_log_probs(leaf, torch.tensor([3, -1, -100]), entropy=True, top_k=2)
    (grad,) = torch.autograd.grad(got.log_probs.sum() + got.entropy.sum(), leaf)
    assert got.log_probs[1:].tolist() == [0, 0] and got.entropy[1:].tolist() == [0, 0] and not grad[1:].any()
    assert got.top_tokens[1:].tolist() == [[-1, -1]] * 2 and bool(grad.isfinite().all())
    loss = distillation_loss(leaf, torch.tensor([[3, 4], [-1, -1], [-1, -2]]), torch.zeros(3, 2))
    (grad,) = torch.autograd.grad(loss, leaf)
    assert bool(loss.isfinite()) and not grad[1:].any() and bool(grad.isfinite().all())


def test_tokens_past_the_vocabulary():
    leaf = _logits(2, 7).requires_grad_(True)
    got = token_log_probs(leaf, torch.tensor([6, 7]))
    assert math.isfinite(got.log_probs[0]) and math.isnan(got.log_probs[1])
    (grad,) = torch.autograd.grad(got.log_probs.sum(), leaf)
    assert bool(grad[0].isfinite().all()) and bool(grad[1].isnan().all())
    for rest in (False, True):
        loss = distillation_loss(leaf, torch.tensor([[6, 1], [2, 7]]), torch.full((2, 2), -1.0), rest=rest, reduction="none")
        assert math.isfinite(loss[0]) and math.isnan(loss[1])
        (grad,) = torch.autograd.grad(loss.sum(), leaf)
        assert bool(grad[0].isfinite().all()) and bool(grad[1].isnan().all())


@pytest.mark.parametrize("temperature", [1.0, 2.0])
@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float64])
def test_distillation(rest, temperature, dtype):
    x = _logits(6, 21).to(dtype)
    tokens = torch.tensor([[0, 20, 3], [1, 1, 2], [-1, -1, -1], [5, -100, 6], [9, 8, 7], [4, 4, 4]])
    given = torch.log(torch.tensor([0.3, 0.25, 0.2])).expand(6, 3).clone()
    given[4, 1] = float("-inf")
    leaf = x.clone().requires_grad_(True)
    loss = distillation_loss(leaf, tokens, given, temperature=temperature, rest=rest, reduction="none")
    want, want_grad, _ = distill(x, tokens, given, temperature, rest)
    torch.testing.assert_close(loss.double(), want, rtol=1e-5, atol=5e-6)
    (grad,) = torch.autograd.grad(loss.sum(), leaf)
    torch.testing.assert_close(grad.double(), want_grad, rtol=torch.finfo(dtype).eps / 2 + 1e-5, atol=5e-6)
    mean = distillation_loss(x, tokens, given, temperature=temperature, rest=rest)
    assert abs(float(mean) - float(want.sum()) / 5) < 1e-5
    total = distillation_loss(x, tokens, given, temperature=temperature, rest=rest, reduction="sum")
    assert abs(float(total) - float(want.sum())) < 5e-5
    assert float(distillation_loss(x, tokens.clamp_max(-1), given, rest=rest)) == 0.0


def test_every_token_listed():
    x = _logits(2, 4).requires_grad_(True)
    tokens, given = torch.arange(4).expand(2, 4), torch.full((2, 4), math.log(0.25))
    loss = distillation_loss(x, tokens, given, rest=True)
    want, want_grad, _ = distill(x, tokens, given, rest=True)
    torch.testing.assert_close(float(loss.detach()), float(want.mean()), rtol=1e-5, atol=1e-6)
    torch.testing.assert_close(torch.autograd.grad(loss, x)[0].double(), want_grad / 2, rtol=1e-5, atol=1e-6)


def test_a_teacher_that_agrees():
    x = _logits(3, 50)
    for rest in (False, True):
        top = token_log_probs(x, top_k=50 if not rest else 10, temperature=1.5)
        given = top.top_log_probs if rest else top.top_log_probs * 1.5
        assert abs(float(distillation_loss(x, top.top_tokens, given, temperature=1.5, rest=rest))) < 1e-5


def test_refusals():
    x, t = torch.zeros(2, 10), torch.zeros(2, dtype=torch.long)
    for bad in (dict(tokens=t[:1]), dict(tokens=t.float()), dict(tokens=t > 0), dict(tokens=None), dict(tokens=t, temperature=0.0),
                dict(tokens=t, temperature=-1.0), dict(tokens=t, temperature=float("nan")), dict(tokens=t, temperature=float("inf")),
                dict(tokens=t, top_k=11), dict(tokens=t, top_k=-1)):
        with pytest.raises(ValueError):
            token_log_probs(x, **bad)
    with pytest.raises(ValueError):
        token_log_probs(x.long(), t)
    with pytest.raises(ValueError):
        token_log_probs(x[:, :0], t)
    t, v = torch.zeros(2, 3, dtype=torch.long), torch.zeros(2, 3)
    for bad in ((x, t[:, :2], v), (x, t, v[:1]), (x, t.float(), v), (x, t, t), (x, t[:, :0], v[:, :0]), (x, t[0], v[0]),
                (x, t, v.clone().requires_grad_(True)), (x.long(), t, v), (x[:, :0], t, v)):
        with pytest.raises(ValueError):
            distillation_loss(*bad)
    for bad in (dict(temperature=0.0), dict(reduction="batchmean")):
        with pytest.raises(ValueError):
            distillation_loss(x, t, v, **bad)


def test_what_looks_through_them():
    """Tracing, compilation and fake GPU tensors find torch's operations, with the same values."""
    x, t = _logits(3, 20), torch.tensor([1, -1, 19])
    tokens, given = torch.tensor([[1, 2], [3, -1], [-1, -1]]), torch.full((3, 2), -1.2)
    both = lambda z: (*token_log_probs(z, t, entropy=True, top_k=3), distillation_loss(z, tokens, given, rest=True))  # noqa: E731
    want = both(x)
    torch._dynamo.reset()
    for got in (torch.compile(both, fullgraph=True, backend="eager")(x), torch.jit.trace(both, (x,), check_trace=False)(x),
                torch.fx.experimental.proxy_tensor.make_fx(both)(x)(x)):
        for a, b in zip(got, want):
            torch.testing.assert_close(a, b)
    with FakeTensorMode():
        z = torch.empty(4, 30, device="cuda", dtype=torch.bfloat16, requires_grad=True)
        out = token_log_probs(z, torch.empty(4, device="cuda", dtype=torch.long), entropy=True, top_k=5)
        assert out.top_tokens.shape == (4, 5) and out.log_probs.requires_grad
        loss = distillation_loss(z, out.top_tokens, out.top_log_probs)
        assert loss.shape == () and loss.dtype == torch.float32 and loss.device.type == "cuda"
    slope = torch.func.grad(lambda z: token_log_probs(z, t).log_probs.sum())(x)
    torch.testing.assert_close(slope, score(x, t, g=torch.ones(3))[2].float(), rtol=1e-5, atol=1e-6)


def test_the_entropys_gradient_past_the_vocabulary():
    """NaN as the log probability's, though the entropy itself is known; twice, where the gradient has a graph."""
    x, tokens = _logits(3, 7), torch.tensor([6, 7, -1])
    for graph in (False, True):
        leaf = x.clone().requires_grad_(True)
        got = token_log_probs(leaf, tokens, entropy=True)
        want, want_grad = score(x, tokens.clamp_max(6), h=torch.ones(3))[1:3]
        torch.testing.assert_close(got.entropy.double(), want, rtol=1e-6, atol=2e-6)
        (grad,) = torch.autograd.grad(got.entropy.sum(), leaf, create_graph=graph)
        assert bool(grad[1].isnan().all()) and not grad[2].any()
        torch.testing.assert_close(grad[0].double(), want_grad[0], rtol=1e-6, atol=2e-6)
        if graph:
            (second,) = torch.autograd.grad((grad[0] ** 2).sum(), leaf)
            assert bool(second[0].isfinite().all()) and bool(second[0].any())


def _without_others():
    """Rows of 12 logits whose every other token is masked, with every token listed, with a single other one, and
    with one that the teacher gives nothing; the distributions' parts of 0.9."""
    x = _logits(4, 12, seed=3)
    tokens = torch.arange(12).expand(4, 12).clone()
    tokens[0, 3:], tokens[2, 11], tokens[3, 5:] = -1, -1, -1
    x[0, 3:] = float("-inf")
    x[3, 8:] = float("-inf")
    given = (torch.linspace(-2, 0, 12).expand(4, 12).masked_fill(tokens < 0, float("-inf")).log_softmax(-1) - 0.105).where(tokens >= 0, -3.0)
    p, q = x.double().softmax(-1), torch.zeros(4, 12, dtype=torch.float64)
    q.scatter_add_(1, tokens.clamp_min(0), given.double().exp().where(tokens >= 0, 0.0))
    for r in (0, 1):  # rows 2 and 3 are the oracle's
        assert not distill(x[r:r + 1], tokens[r:r + 1], given[r:r + 1], rest=True)[0].isfinite()
    want = torch.cat([(p - q)[:2], distill(x[2:], tokens[2:], given[2:], rest=True)[1]])
    return x, tokens, given, want


def test_a_rest_without_probability():
    """The loss is infinite, and the gradient that of the row's sum alone, Q p - q with Q = 1, as from the kernel."""
    x, tokens, given, want = _without_others()
    for graph in (False, True):
        leaf = x.clone().requires_grad_(True)
        loss = distillation_loss(leaf, tokens, given, rest=True, reduction="none")
        assert loss.isinf().tolist() == [True, True, False, False]
        (grad,) = torch.autograd.grad(loss.sum(), leaf, create_graph=graph)
        torch.testing.assert_close(grad.double(), want, rtol=1e-5, atol=1e-6)
        if graph:
            assert bool(torch.autograd.grad((grad ** 2).sum(), leaf)[0].isfinite().all())


def test_the_strict_check_sees_what_is_no_number():
    """A NaN or an infinity where the oracle has a number, or the other way round, does not pass, whatever the room."""
    value, room = torch.tensor([1.0, -2.0, 3.0]), torch.tensor([0.1, 0.1, 0.1])
    within(value, value.double(), room)
    within(value, value.double() + 0.09, room)
    odd = torch.tensor([1.0, float("nan"), float("-inf")])
    within(odd, odd.double(), room)
    for other in (float("nan"), float("inf"), 1.11):
        for swapped in (False, True):
            wrong = value.clone()
            wrong[0] = other
            with pytest.raises(AssertionError):
                within(*((value, wrong.double()) if swapped else (wrong, value.double())), room)
    for no_room in (float("nan"), float("inf"), -1.0):
        with pytest.raises(AssertionError):
            within(value, value.double(), torch.tensor([0.1, no_room, 0.1]))


@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("temperature", [1.0, 2.5])
def test_the_formula_against_the_definition(rest, temperature):
    """The closed form of the loss's gradient in 64 bits against autograd's of the definition."""
    x = _logits(7, 23, seed=5)
    x[6, 15:] = float("-inf")
    tokens = torch.tensor([[0, 22, 3, 7], [1, 1, 2, 1], [-1, -1, -1, -1], [5, -100, 6, 8], [9, 8, 7, 22], [4, 4, 4, 4], [3, 2, 1, 0]])
    given = torch.log(torch.tensor([0.3, 0.25, 0.2, 0.1])).expand(7, 4).clone()
    given[4, 1], g = float("-inf"), torch.linspace(-1, 2, 7)
    want, want_grad, want_logp = distill(x, tokens, given, temperature, rest, g)
    loss, grad, logp, _ = distill_by_formula(x, tokens, given, temperature, rest, g)
    for a, b in ((loss, want), (grad, want_grad), (logp[:2], want_logp[:2])):
        torch.testing.assert_close(a, b, rtol=1e-12, atol=1e-12)
