"""The distillation loss and its gradient against 64 bits."""

import math

import pytest
import torch

from _logits_oracle import distill, half_step, relative, smallest_step

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]


@pytest.fixture(autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _case(rows, vocab, k, dtype, seed=0, padded=0.1):
    """Student and teacher that see much the same, some entries and one row padded."""
    gen = _gen(seed + vocab)
    x = torch.randn(rows, vocab, device="cuda", generator=gen) * 3
    teacher = (x + torch.randn(rows, vocab, device="cuda", generator=gen) * 0.5).log_softmax(-1)
    values, tokens = teacher.topk(min(k, vocab), -1)
    gone = torch.rand(tokens.shape, device="cuda", generator=gen) < padded
    gone[:, 0] = False
    if rows > 2:
        gone[2] = True
    return x.to(dtype), tokens.where(~gone, -1), values


def _check(x, tokens, given, temperature=1.0, rest=False):
    from fairring_b200.ops import distillation_loss

    rows = x.shape[:-1]
    g = torch.randn(rows, device="cuda", generator=_gen(1))
    leaf = x.detach().requires_grad_(True)
    loss = distillation_loss(leaf, tokens, given, temperature=temperature, rest=rest, reduction="none")
    (grad,) = torch.autograd.grad(loss, leaf, g)
    want, want_grad, logp = distill(x, tokens, given, temperature, rest, g)
    assert loss.dtype == torch.float32 and grad.dtype == x.dtype and grad.shape == x.shape
    # the two sums' errors move the loss by as much as they are off, relatively; the teacher's probabilities are 2^-21 of
    # themselves off plus the roundings of their exponents, and weigh differences of logarithms
    there = tokens >= 0
    apart = (logp.gather(-1, tokens.clamp_min(0)).clamp_min(-110).abs() + given.double().clamp_min(-110).abs() + 8).where(there, 0.0)
    room = 2.0 ** -16.5 + 2.0 ** -20 * apart.amax(-1) + 2.0 ** -23 * want.abs()
    fine = want.isfinite()
    assert torch.equal(fine, loss.isfinite())
    off = (loss.double() - want).abs()
    assert bool((off <= room)[fine].all()), (float(off[fine].max()), float(room.min()))
    p = logp.exp()
    q = torch.zeros_like(p).scatter_add_(-1, tokens.clamp_min(0), torch.where(there, 1.0, 0.0).double())
    scale = g.double().abs().unsqueeze(-1) / temperature
    # a probability's error; with the rest the weight of the others' is a difference of two numbers up to 1, over p_rest
    share = p
    if rest:
        others = p.masked_fill(q > 0, 0.0)
        share = p + others / others.sum(-1, keepdim=True).clamp_min(1e-300)
    room = half_step(x.dtype) * want_grad.abs() + scale * (2 * relative(logp) * share + 2.0 ** -19 * (q > 0)) + smallest_step(x.dtype)
    bad = (grad.double() - want_grad).abs() > room
    assert not bad.any(), (int(bad.sum()), float((grad.double() - want_grad).abs().max()))
    return loss, grad


# as for the log probabilities: the parts of a row, one batch and the next, sliced rows and whole ones
@pytest.mark.parametrize("rows", [1, 5, 299])
@pytest.mark.parametrize("vocab,k", [(2, 1), (7, 3), (8, 8), (1001, 256), (8192, 5), (8193, 64), (16385, 33), (50265, 100)])
@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
def test_every_row_length(rows, vocab, k, rest, dtype):
    loss, grad = _check(*_case(rows, vocab, k, dtype), rest=rest)
    if rows > 2:
        assert loss[2] == 0 and not grad[2].any()


# rows of a warp each, and rows that are taken by blocks that stay
@pytest.mark.parametrize("vocab,k", [(7, 3), (264, 256), (1001, 5), (4099, 100), (8192, 128), (8193, 64), (20011, 33)])
@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
def test_many_rows(vocab, k, rest, dtype):
    x, tokens, given = _case(1300, vocab, k, dtype)
    tokens[100:900] = -1  # most blocks have rows that do not count
    tokens[950:1000, 1:] = tokens[950:1000, :1]  # one token all over
    tokens[1299, :-1] = -1  # only the last entry
    _check(x, tokens, given - 0.2 if rest else given, 1.3, rest)


@pytest.mark.parametrize("rest", [False, True])
def test_several_rows_a_block(rest):
    x, tokens, given = _case(4001, 8200, 6, torch.float32)
    tokens[500:1500] = -1
    tokens[torch.rand(4001, device="cuda", generator=_gen(3)) < 0.3] = -100
    _check(x, tokens, given - 0.2 if rest else given, 1.0, rest)


@pytest.mark.parametrize("temperature", [0.5, 2.0])
@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
def test_temperature(temperature, rest, dtype):
    x, tokens, given = _case(9, 3001, 20, dtype)
    if rest:
        given = given * 1.2 - 0.1  # some distribution's log probabilities: they leave something
    _check(x, tokens, given, temperature, rest)


@pytest.mark.parametrize("rest", [False, True])
def test_tokens_named_twice_and_at_the_edges(rest):
    for dtype in DTYPES:
        for vocab in (1003, 30000):
            x, _, _ = _case(4, vocab, 5, dtype)
            tokens = torch.tensor([[0, vocab - 1, 0, 5, 0], [1, 2, 3, 4, 5], [7, 7, 7, 7, 7], [vocab - 1, 8, 16, 8, vocab - 2]],
                                  device="cuda")
            given = torch.log(torch.tensor([0.2, 0.1, 0.15, 0.3, 0.05], device="cuda")).expand(4, 5)
            _check(x, tokens, given, rest=rest)


@pytest.mark.parametrize("rest", [False, True])
def test_values_of_minus_infinity(rest):
    """Teacher's entries without mass, a row without any, and a student that excludes what is not listed."""
    low = float("-inf")
    for dtype in DTYPES:
        x, tokens, given = _case(6, 2050, 4, dtype, padded=0.0)
        tokens[2] = tokens[1]
        given = given.clone()
        given[0, 1:] = low
        given[1] = low
        if not rest:
            x[3, tokens[3, 0]] = low  # the loss is infinite
        tail = torch.ones(2050, dtype=torch.bool, device="cuda")
        tail[tokens[4]] = False
        x[4, tail] = low
        loss, grad = _check(x[:4], tokens[:4], given[:4], rest=rest)
        assert (loss[1] == 0) == (not rest) and (rest or not grad[1].any())
        from fairring_b200.ops import distillation_loss

        leaf = x[4:5].clone().requires_grad_(True)
        loss = distillation_loss(leaf, tokens[4:5], given[4:5], rest=rest)
        assert math.isinf(loss) == rest  # a class of no probability that the teacher gives some
        (grad,) = torch.autograd.grad(loss, leaf)
        assert bool(grad.isfinite().all())


def test_nothing_left_for_the_rest():
    """The teacher's entries are everything, or a rounding more: the rest has no part in the loss."""
    x, tokens, _ = _case(3, 500, 2, torch.float32, padded=0.0)
    tokens[2] = tokens[0]
    given = torch.log(torch.tensor([[0.5, 0.5], [0.75, 0.25], [0.5, 0.5000001]], device="cuda"))
    _check(x, tokens, given, rest=True)


def test_far_apart():
    """The rest is far below what is listed, or above: its probability comes from its own sum."""
    x, tokens, given = _case(4, 5000, 8, torch.float32, padded=0.0)
    tokens[2] = tokens[1]
    given = given - 0.2
    x.scatter_add_(1, tokens, torch.full_like(given, 40.0))
    _check(x, tokens, given, rest=True)
    x.scatter_add_(1, tokens, torch.full_like(given, -90.0))
    _check(x, tokens, given, rest=True)


@pytest.mark.parametrize("rest", [False, True])
def test_views(rest):
    for dtype in DTYPES:
        for vocab in (1000, 1003):
            x, tokens, given = _case(4 * 9, vocab + 5, 6, dtype)
            x, tokens, given = x.view(4, 9, -1), tokens.view(4, 9, -1).clamp_max(vocab - 1), given.view(4, 9, -1)
            for part in (lambda t: t[:, :-1], lambda t: t[1::2, ::2], lambda t: t.transpose(0, 1)):
                _check(part(x)[..., :vocab], part(tokens), part(given), rest=rest)
            _check(x[..., 3: vocab + 3], tokens, given, rest=rest)
            _check(x[..., :vocab].flip(2), tokens, given, rest=rest)
    x, tokens, given = _case(1, 777, 6, torch.float32)
    _check(x[0], tokens[0], given[0], rest=rest)


@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
def test_reductions(rest, dtype):
    from fairring_b200.ops import distillation_loss

    x, tokens, given = _case(50, 1003, 12, dtype)
    tokens[10:20] = -100
    each = distillation_loss(x, tokens, given, rest=rest, reduction="none").double()
    counts = int((tokens >= 0).any(-1).sum())
    assert counts == 39
    for reduction, scale in (("mean", 1 / counts), ("sum", 1.0)):
        leaf = x.clone().requires_grad_(True)
        loss = distillation_loss(leaf, tokens, given, rest=rest, reduction=reduction)
        assert abs(float(loss) - float(each.sum()) * scale) <= 50 * 2.0 ** -24 * float(each.sum()) * scale
        (grad,) = torch.autograd.grad(loss * 64, leaf)
        one = x.clone().requires_grad_(True)
        (want,) = torch.autograd.grad(distillation_loss(one, tokens, given, rest=rest, reduction="none"), one,
                                      torch.full((50,), 64 * scale, device="cuda"))
        # the two scale factors may differ by their roundings: a step of the result
        torch.testing.assert_close(grad.double(), want.double(), rtol=2 * half_step(dtype) + 2.0 ** -22, atol=smallest_step(dtype) * 2)
    tokens[:] = -1
    leaf = x.clone().requires_grad_(True)
    loss = distillation_loss(leaf, tokens, given, rest=rest)
    assert float(loss) == 0.0
    assert not torch.autograd.grad(loss, leaf)[0].any()


def test_gradient_against_differences():
    from fairring_b200.ops import distillation_loss

    x, tokens, given = _case(3, 40, 4, torch.float32)
    step = 2.0 ** -6
    for rest in (False, True):
        value = lambda z: distillation_loss(z, tokens, given - 0.1, rest=rest, reduction="none").double()  # noqa: E731
        leaf = x.clone().requires_grad_(True)
        (grad,) = torch.autograd.grad(value(leaf).sum(), leaf)
        for col in (0, int(tokens[0, 0]), int(tokens[1, 0]), 39):
            d = torch.zeros_like(x)
            d[:, col] = step
            slope = (value(x + d) - value(x - d)) / (2 * step)
            # the third derivative is at most 2; values up to 16, 2^-17 of them over the step
            assert bool((grad[:, col].double() - slope).abs().max() <= step ** 2 + 16 * 2.0 ** -17 / step)


@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_second_derivative(rest, reduction):
    from fairring_b200.ops import distillation_loss
    from fairring_b200.ops.distillation import _plain_distillation

    x, tokens, given = _case(5, 33, 6, torch.float32)
    given = given - 0.1
    tokens[3, 1] = tokens[3, 0]
    got = []
    for native in (True, False):
        leaf = (x if native else x.double()).clone().requires_grad_(True)
        if native:
            loss = distillation_loss(leaf, tokens, given, rest=rest, temperature=1.5, reduction=reduction)
        else:
            loss, counts = _plain_distillation(leaf, tokens, given, 1.5, rest)
            loss = loss.sum() / counts.sum() if reduction == "mean" else loss
        (g,) = torch.autograd.grad((loss ** 2).sum(), leaf, create_graph=True)
        got.append([g.double(), torch.autograd.grad((g ** 2).sum(), leaf)[0].double()])
    for a, b in zip(*got):
        torch.testing.assert_close(a, b, rtol=1e-4, atol=1e-6)


@pytest.mark.parametrize("rows", [40, 1350])
def test_bits_repeat_and_modes(rows):
    from fairring_b200 import launch_count
    from fairring_b200.ops import distillation_loss

    x, tokens, given = _case(rows, 50265, 64, torch.bfloat16)
    tokens[:, 3] = tokens[:, 0]
    for rest in (False, True):
        got = []
        for _ in range(4):
            leaf = x.clone().requires_grad_(True)
            loss = distillation_loss(leaf, tokens, given, rest=rest)
            got.append((loss.detach(), torch.autograd.grad(loss, leaf)[0]))
        assert all(torch.equal(a, got[0][0]) and torch.equal(b, got[0][1]) for a, b in got[1:])
        before = launch_count()
        with torch.inference_mode():
            assert torch.equal(distillation_loss(x, tokens, given, rest=rest), got[0][0])
        assert launch_count() == before + 2
        low = given.bfloat16()
        assert torch.equal(distillation_loss(x, tokens.int(), low, rest=rest), distillation_loss(x, tokens, low.float(), rest=rest))


def test_empty_and_refused():
    from fairring_b200.ops import distillation_loss

    none = torch.empty(0, 100, device="cuda", requires_grad=True)
    loss = distillation_loss(none, torch.empty(0, 3, dtype=torch.long, device="cuda"), torch.empty(0, 3, device="cuda"))
    assert float(loss.detach()) == 0.0 and torch.autograd.grad(loss, none)[0].shape == (0, 100)
    x, t, v = torch.zeros(2, 10, device="cuda"), torch.zeros(2, 3, dtype=torch.long, device="cuda"), torch.zeros(2, 3, device="cuda")
    for bad in ((x, t.cpu(), v), (x, t, v.cpu()), (x, t[:, :2], v), (x, t, v[:1]), (x, t.float(), v), (x, t, t), (x, t[:, :0], v[:, :0]),
                (x, t, v.clone().requires_grad_(True)), (x.long(), t, v)):
        with pytest.raises(ValueError):
            distillation_loss(*bad)
    for bad in (dict(temperature=-1.0), dict(temperature=float("inf")), dict(reduction="batchmean")):
        with pytest.raises(ValueError):
            distillation_loss(x, t, v, **bad)
    t[1, 2] = 10  # past the vocabulary
    for rest in (False, True):
        leaf = x.clone().requires_grad_(True)
        loss = distillation_loss(leaf, t, v - 2, rest=rest, reduction="none")
        assert math.isnan(loss[1]) and math.isfinite(loss[0])
        (g,) = torch.autograd.grad(loss.sum(), leaf)
        assert bool(g[1].isnan().all()) and bool(g[0].isfinite().all())


def test_a_captured_training_step():
    """Forward and backward of two losses in graphs, replayed in turn.  No eager graph of the same leaf may live meanwhile:
    torch then ties the capture to the stream of that graph's gradient, whatever the operation."""
    from fairring_b200.ops import distillation_loss

    x, tokens, given = _case(64, 12345, 16, torch.bfloat16)
    leaf = x.clone().requires_grad_(True)

    def call(rest):
        loss = distillation_loss(leaf, tokens, given, rest=rest)
        return loss.detach(), torch.autograd.grad(loss, leaf)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call(False), call(True)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for rest in (False, True):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(call(rest))
    with torch.no_grad():
        leaf.copy_(_case(64, 12345, 16, torch.bfloat16, seed=5)[0])
    for graph in (graphs[1], graphs[0], graphs[1]):
        graph.replay()
    for rest, out in zip((False, True), outs):
        assert all(torch.equal(a, b) for a, b in zip(out, call(rest)))


def test_a_teacher_and_its_student():
    """The teacher's largest entries, written down position by position, teach a student of the same family."""
    from fairring_b200.models import DecoderConfig, DecoderLM
    from fairring_b200.ops import distillation_loss, token_log_probs

    torch.manual_seed(0)
    cfg = DecoderConfig.tiny()
    teacher, student = DecoderLM(cfg).cuda().eval(), DecoderLM(cfg).cuda()
    tokens = torch.randint(0, cfg.vocab, (3, cfg.seq_len), device="cuda")
    follow = tokens[:, 1:].clone()
    follow[2, 40:] = -100  # a shorter sequence
    with torch.no_grad(), torch.autocast("cuda", dtype=torch.bfloat16):
        top = token_log_probs(teacher(tokens)[:, :-1], follow, temperature=2.0, top_k=50)
    for rest in (False, True):
        given = top.top_log_probs if rest else top.top_log_probs * 2.0  # back to differences of logits
        with torch.autocast("cuda", dtype=torch.bfloat16):
            logits = student(tokens)[:, :-1]
            loss = distillation_loss(logits, top.top_tokens, given, temperature=2.0, rest=rest)
        student.zero_grad()
        loss.backward()
        want, _, _ = distill(logits, top.top_tokens, given.clamp_min(-1e30), 2.0, rest)
        n = int((follow >= 0).sum())
        assert abs(float(loss) - float(want.sum()) / n) <= 2.0 ** -16
        _check(logits.detach(), top.top_tokens, given, 2.0, rest)
        assert all(p.grad is not None and bool(p.grad.isfinite().all()) for p in student.parameters())


@pytest.mark.parametrize("rest", [False, True])
def test_second_derivative_past_rows_that_do_not_count(rest):
    """A padded row's logits may be anything, its first and second derivatives are 0."""
    from fairring_b200.ops import distillation_loss

    x, tokens, given = _case(4, 33, 6, torch.float32)
    x[2] = float("nan")  # _case pads that row
    leaf = x.requires_grad_(True)
    loss = distillation_loss(leaf, tokens, given - 0.1, rest=rest)
    (g,) = torch.autograd.grad(loss ** 2, leaf, create_graph=True)
    (h,) = torch.autograd.grad((g ** 2).sum(), leaf)
    for d in (g, h):
        assert bool((d[2] == 0).all()) and bool((d[0] != 0).any()) and bool(d.isfinite().all())


@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("rows,vocab", [(60, 20011), (1300, 20011), (1300, 1003)])
def test_two_streams_at_once(rows, vocab, rest):
    from fairring_b200.ops import distillation_loss

    inputs = [_case(rows, vocab, 20, torch.bfloat16, seed=i) for i in range(2)]

    def call(i):
        leaf = inputs[i][0].detach().requires_grad_(True)
        loss = distillation_loss(leaf, *inputs[i][1:], rest=rest)
        return loss.detach(), torch.autograd.grad(loss, leaf)[0]

    want = [call(i) for i in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = [[], []]
    for _ in range(8):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(call(i))
    torch.cuda.synchronize()
    for i in range(2):
        for out in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(out, want[i]))


def test_the_mean_of_very_many_rows():
    from fairring_b200.ops import distillation_loss

    x, tokens, given = _case(300_007, 24, 4, torch.bfloat16)
    each = distillation_loss(x, tokens, given, reduction="none").double()
    want = each.sum() / int((tokens >= 0).any(-1).sum())
    # summed in 64 bits and rounded once
    assert abs(float(distillation_loss(x, tokens, given)) - float(want)) <= 2.0 ** -23 * float(want)
