"""Log probabilities, entropy and largest entries against 64 bits, where rows, ties, masks and strides can go wrong."""

import math

import pytest
import torch

from _logits_oracle import half_step, relative, score, smallest_step

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]


@pytest.fixture(autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _logits(rows, vocab, dtype, seed=0, scale=3.0):
    gen = _gen(seed + vocab)
    x = torch.randn(rows, vocab, device="cuda", generator=gen) * scale
    x[:, vocab // 2] += 6
    return x.to(dtype)


def _check(logits, tokens, temperature=1.0, entropy=True):
    """Values and gradients; every row's upstream is its own."""
    from fairring_b200.ops import token_log_probs

    gen = _gen(1)
    g = torch.randn(tokens.shape, device="cuda", generator=gen)
    h = torch.randn(tokens.shape, device="cuda", generator=gen)
    leaf = logits.detach().requires_grad_(True)
    got = token_log_probs(leaf, tokens, temperature=temperature, entropy=entropy)
    (grad,) = torch.autograd.grad([got.log_probs, got.entropy] if entropy else got.log_probs, leaf, [g, h] if entropy else g)
    want, want_h, want_grad, logp = score(logits, tokens, temperature, g, h if entropy else None)
    assert got.log_probs.dtype == torch.float32 and grad.dtype == logits.dtype and grad.shape == logits.shape
    # the difference to the maximum, the temperature, the product and the sum: 2^-24 each; the sum's own error
    finite = want.isfinite()
    assert torch.equal(finite, got.log_probs.isfinite())
    off = (got.log_probs.double() - want).abs()
    assert bool((off <= 2.0 ** -17.3 + 4 * 2.0 ** -24 * want.abs())[finite].all()), float(off[finite].max())
    if entropy:
        # both terms are at most log V + 1; each probability's error times its part of the entropy
        err = (logp.exp() * (1 + logp.clamp_min(-110).abs()) * relative(logp)).sum(-1) * 2 + 2.0 ** -17.3
        assert bool(((got.entropy.double() - want_h).abs() <= err).all()), float((got.entropy.double() - want_h).abs().max())
    p = logp.exp()
    size = p * (g.double().abs().unsqueeze(-1) + (h.double().abs() * (1 + want_h)).unsqueeze(-1) * (1 + logp.clamp_min(-110).abs())) / temperature
    room = half_step(logits.dtype) * want_grad.abs() + 2 * relative(logp) * size + smallest_step(logits.dtype)
    # A probability below 2^-126 is zero, and its entry then off by as much times the factor: with one over T it may be a normal number.
    room = room + 2.0 ** -126 * (g.double().abs() + 128 * h.double().abs()).unsqueeze(-1) / temperature
    room = room + 2.0 ** -22 * g.double().abs().unsqueeze(-1) / temperature * torch.zeros_like(p).scatter_(
        -1, tokens.clamp_min(0).unsqueeze(-1), 1.0)
    beyond = (want_grad.abs() > torch.finfo(logits.dtype).max) & (grad == want_grad.sign() * float("inf"))  # as it rounds
    bad = ((grad.double() - want_grad).abs() > room) & ~beyond
    assert not bad.any(), (int(bad.sum()), float((grad.double() - want_grad).abs().max()))
    return got, grad


# one thread's worth, remainders on both sides of the 16-byte vectors, one batch of a block (256 x 4 vectors) and the
# next; 19 rows are cut into slices from 512 vectors a slice on, 400 rows are not; 1300 rows are taken by blocks that stay
@pytest.mark.parametrize("rows", [1, 19, 400, 1300])
@pytest.mark.parametrize("vocab", [1, 7, 8, 9, 1000, 1001, 4096, 4097, 8191, 8192, 8193, 16385, 32776, 50265])
@pytest.mark.parametrize("dtype", DTYPES)
def test_every_row_length(rows, vocab, dtype):
    logits = _logits(rows, vocab, dtype)
    tokens = torch.randint(0, vocab, (rows,), device="cuda", generator=_gen(vocab))
    if rows > 5:
        tokens[3], tokens[4], tokens[5] = -100, 0, vocab - 1
    _, grad = _check(logits, tokens)
    if rows > 5:
        assert not grad[3].any()


@pytest.mark.parametrize("temperature", [0.3, 0.7, 2.0])
@pytest.mark.parametrize("entropy", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
def test_temperature(temperature, entropy, dtype):
    logits = _logits(37, 5003, dtype)
    _check(logits, torch.randint(0, 5003, (37,), device="cuda", generator=_gen(2)), temperature, entropy)


# few rows, a row per warp, blocks that stay
@pytest.mark.parametrize("rows,vocab", [(5, 20011), (700, 1003), (700, 9001)])
@pytest.mark.parametrize("entropy", [False, True])
def test_where_the_fast_exponent_does_not_reach(rows, vocab, entropy):
    """Logits far from zero, temperatures near zero and far above one, and all of them in one batch."""
    for dtype in DTYPES:
        tokens = torch.randint(0, vocab, (rows,), device="cuda", generator=_gen(9))
        logits = _logits(rows, vocab, dtype)
        tokens[::3] = logits[::3].float().argmax(-1)
        for temperature in (1e-6, 1e-3, 1e6):
            _check(logits, tokens, temperature, entropy)
    logits = _logits(rows, vocab, torch.float32)
    for shift in (3e6, -3e6, 1e30, -1e30):
        part = logits.clone()
        part[::2] += shift
        _check(part, tokens, 1.0, entropy)


@pytest.mark.parametrize("rows,vocab", [(3, 1001), (3, 50265), (300, 20000), (1301, 1001), (1301, 20000)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_masked_logits(rows, vocab, dtype):
    """Minus infinity and the type's lowest value, up to rows of nothing else."""
    from fairring_b200.ops import token_log_probs

    lowest = torch.finfo(dtype).min
    for fill in (float("-inf"), lowest):
        logits = _logits(rows, vocab, dtype)
        gone = torch.rand(rows, vocab, device="cuda", generator=_gen(3)) < 0.9
        gone[1] = True
        gone[1, vocab - 1] = False  # a single logit left
        gone[2, : vocab - 2] = True  # whole slices without one
        gone[2, vocab - 2:] = False
        gone[:, 5] = False
        logits.masked_fill_(gone, fill)
        tokens = torch.full((rows,), 5, device="cuda")
        tokens[1] = vocab - 1
        _check(logits, tokens)
    logits[0] = lowest
    logits[1] = float("-inf")
    tokens[0] = 0
    leaf = logits.requires_grad_(True)
    got = token_log_probs(leaf, tokens, entropy=True, top_k=2)
    assert abs(float(got.log_probs[0]) + math.log(vocab)) < 1e-5 and abs(float(got.entropy[0]) - math.log(vocab)) < 1e-4
    assert got.top_tokens[0].tolist() == [0, 1] and got.top_tokens[1].tolist() == [0, 1]
    for value in (got.log_probs[1], got.entropy[1], got.top_log_probs[1, 0]):
        assert math.isnan(value)  # as log_softmax
    (grad,) = torch.autograd.grad(got.log_probs.sum(), leaf)
    assert bool(grad[1].isnan().all()) and bool(grad[0].isfinite().all()) and bool(grad[2:].isfinite().all())


@pytest.mark.parametrize("rows", [6, 320, 1400])
@pytest.mark.parametrize("dtype", DTYPES)
def test_values_that_are_no_numbers(rows, dtype):
    """NaN and infinity make their own row NaN and no other; a row that does not count may hold anything."""
    from fairring_b200.ops import token_log_probs

    for vocab in (129, 17001):
        logits = _logits(rows, vocab, dtype)
        logits[0, 77] = float("nan")
        logits[1, 99] = float("inf")
        logits[2] = float("nan")
        logits[3] = float("nan")
        logits[4, 0] = float("inf")
        tokens = torch.full((rows,), 7, device="cuda")
        tokens[3], tokens[4] = -1, -100
        leaf = logits.requires_grad_(True)
        got = token_log_probs(leaf, tokens, entropy=True, top_k=3)
        (grad,) = torch.autograd.grad(got.log_probs.sum() + got.entropy.sum(), leaf)
        for r in (0, 1, 2):
            assert math.isnan(got.log_probs[r]) and math.isnan(got.entropy[r]) and bool(grad[r].isnan().any())
        assert got.top_tokens[0, 0] == 77 and got.top_tokens[1, 0] == 99 and got.top_tokens[2].tolist() == [0, 1, 2]
        for r in (3, 4):
            assert got.log_probs[r] == 0 and got.entropy[r] == 0 and not grad[r].any()
            assert got.top_tokens[r].tolist() == [-1] * 3 and bool((got.top_log_probs[r] == float("-inf")).all())
        assert bool(grad[5:].isfinite().all()) and bool(got.log_probs[5:].isfinite().all())


def _check_top(logits, k, temperature=1.0):
    from fairring_b200.ops import token_log_probs

    got = token_log_probs(logits, top_k=k, temperature=temperature)
    assert got.log_probs is None and got.entropy is None
    order = logits.float().sort(dim=-1, descending=True, stable=True).indices[..., :k]
    assert got.top_tokens.dtype == torch.long and torch.equal(got.top_tokens, order)
    want = (logits.double() / temperature).log_softmax(-1).gather(-1, order)
    fine = want.isfinite()
    assert torch.equal(fine, got.top_log_probs.isfinite())
    off = (got.top_log_probs.double() - want).abs()
    assert bool((off <= 2.0 ** -17.3 + 4 * 2.0 ** -24 * want.abs())[fine].all())


@pytest.mark.parametrize("rows", [1, 7, 60, 330, 1250])
@pytest.mark.parametrize("vocab,k", [(1, 1), (5, 5), (130, 128), (1000, 7), (1024, 128), (8193, 1), (32003, 20), (51200, 64),
                                     (50265, 128)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_top(rows, vocab, k, dtype):
    _check_top(_logits(rows, vocab, dtype), k, 0.7)


@pytest.mark.parametrize("rows", [2, 310, 1201])
@pytest.mark.parametrize("vocab", [300, 9001, 51200])
@pytest.mark.parametrize("kind", ["equal", "few values", "rising", "falling", "in one place", "few left", "zeros", "scattered left"])
@pytest.mark.parametrize("dtype", DTYPES)
def test_top_of_rows_that_are_hard_to_rank(rows, vocab, kind, dtype):
    x = torch.zeros(rows, vocab, device="cuda")
    at = torch.arange(vocab, device="cuda").float()
    if kind == "few values":
        x += torch.randint(0, 3, (rows, vocab), device="cuda", generator=_gen(4))
    elif kind == "rising":
        x += at / vocab * 20
    elif kind == "falling":
        x -= at / vocab * 20
    elif kind == "in one place":
        x += torch.randn(rows, vocab, device="cuda", generator=_gen(5))
        x[:, 100:250] += 10
    elif kind in ("few left", "scattered left"):  # fewer than k that are not masked, and ties among the masked
        x.fill_(float("-inf"))
        x[:, -3:] = at[:3]
        if kind == "scattered left":
            x[:, :: vocab // 40] = 1.0
    elif kind == "zeros":  # both zeros are equal
        x[:, ::2] = -0.0
    for k in (1, 6, 100):
        _check_top(x.to(dtype), k)


def test_views():
    """Batches without their last position, vocabularies without their padding, another order of the dimensions, rows
    off a 16-byte boundary; and what has to be copied."""
    for dtype in DTYPES:
        for vocab in (1000, 1003, 12289):
            wide = _logits(4 * 9, vocab + 5, dtype).view(4, 9, vocab + 5)
            tokens = torch.randint(0, vocab, (4, 9), device="cuda", generator=_gen(6))
            tokens[1, 3] = -100
            for x in (wide[..., :vocab], wide[..., 3: vocab + 3], wide.transpose(0, 1)[..., :vocab].contiguous().transpose(0, 1),
                      wide[..., :vocab].flip(2), wide[::2, 1::3, :vocab], wide[:1, :, :vocab].expand(4, 9, vocab),
                      wide.view(2, 2, 9, vocab + 5)[:, :, 1:8, :vocab]):
                t = tokens.view(2, 2, 9)[:, :, 1:8] if x.dim() == 4 else tokens[::2, 1::3] if x.shape[0] == 2 else tokens
                assert t.shape == x.shape[:-1]
                _check(x, t)
    _check(_logits(1, 1003, torch.float32)[0], torch.tensor(5, device="cuda"))  # one row without a leading dimension


# a row per warp; several rows per block of those that stay; one
@pytest.mark.parametrize("rows,vocab", [(20000, 264), (4001, 8200), (1500, 17000)])
@pytest.mark.parametrize("share", [0.0, 0.02, 0.5, 0.99, 1.0])
def test_rows_that_do_not_count_among_many(rows, vocab, share):
    """Whole runs of rows of a block without one that counts, and the last rows of all."""
    from fairring_b200.ops import token_log_probs

    gen = _gen(8)
    logits = _logits(rows, vocab, torch.float32)
    tokens = torch.randint(0, vocab, (rows,), device="cuda", generator=gen)
    tokens[torch.rand(rows, device="cuda", generator=gen) < share] = -100
    tokens[: rows // 4] = -1
    logits[tokens < 0] = float("nan")
    _check(logits.nan_to_num(), tokens)
    got = token_log_probs(logits, tokens, entropy=True, top_k=3)
    assert bool(got.entropy.isfinite().all()) and bool((got.top_tokens[tokens < 0] == -1).all())
    assert torch.equal(got.top_tokens[tokens >= 0], logits[tokens >= 0].sort(dim=1, descending=True, stable=True).indices[:, :3])


def test_kinds_of_gradients():
    """Only one output used, one value for all rows, another type of upstream, a part of a graph that is a leaf's child."""
    from fairring_b200.ops import token_log_probs

    x = _logits(6, 1009, torch.float32)
    tokens = torch.tensor([0, 1, -100, 1008, 7, 5], device="cuda")
    # (function, largest upstream value: log probabilities here are above -30)
    for f, up in ((lambda o: o.log_probs.mean(), 1 / 6), (lambda o: o.entropy.mean(), 1 / 6),
                  (lambda o: (o.entropy * o.log_probs).sum(), 30.0), (lambda o: o.log_probs[1] * 3, 3.0),
                  (lambda o: (o.log_probs.double() + o.entropy).sum(), 1.0)):
        got, want = [], []
        for native in (True, False):
            leaf = x.clone().requires_grad_(True)
            if native:
                o = token_log_probs(leaf * 1.5, tokens, entropy=True, top_k=4)
                assert not o.top_log_probs.requires_grad and not o.top_tokens.requires_grad
                got = torch.autograd.grad(f(o), leaf)[0]
            else:
                from fairring_b200.ops.token_log_probs import _plain_token_log_probs

                leaf = leaf.detach().double().requires_grad_(True)
                want = torch.autograd.grad(f(_plain_token_log_probs(leaf * 1.5, tokens, 1.0, True, 0)), leaf)[0]
        # An entry up * 1.5 * p (log p + H) vanishes where log p = -H: there its error is that of its two terms.  p is
        # 2^-20 of itself off (see the oracle: u up to 20 here), p |log p| <= 0.37 and p H <= ln 1009 < 7.
        torch.testing.assert_close(got.double(), want, rtol=2.0 ** -16, atol=up * 1.5 * 2.0 ** -20 * 7.4)
    o = token_log_probs(x.requires_grad_(True), entropy=True)  # no token asked for
    assert o.log_probs is None
    torch.testing.assert_close(torch.autograd.grad(o.entropy.sum(), x)[0].double(),
                               score(x, torch.zeros(6, dtype=torch.long, device="cuda"), h=torch.ones(6, device="cuda"))[2],
                               rtol=2.0 ** -15, atol=1e-7)


def test_gradient_against_differences():
    from fairring_b200.ops import token_log_probs

    x = _logits(3, 40, torch.float32, scale=1.0)
    tokens = torch.tensor([3, 39, 0], device="cuda")
    value = lambda z: (lambda o: o.log_probs.double() * 0.7 + o.entropy.double() * 0.3)(token_log_probs(z, tokens, entropy=True))  # noqa: E731
    leaf = x.clone().requires_grad_(True)
    (grad,) = torch.autograd.grad(value(leaf).sum(), leaf)
    step = 2.0 ** -6
    for col in (0, 3, 20, 39):
        d = torch.zeros_like(x)
        d[:, col] = step
        slope = (value(x + d) - value(x - d)) / (2 * step)
        # central differences: the third derivative is at most 2; 2^-17 of values up to 8 over the step
        assert bool((grad[:, col].double() - slope).abs().max() <= step ** 2 + 8 * 2.0 ** -17 / step)


def test_second_derivative():
    from fairring_b200.ops import token_log_probs

    x = _logits(5, 17, torch.float32)
    tokens = torch.tensor([1, -100, 0, 16, 2], device="cuda")
    got = []
    for native in (True, False):
        leaf = x.clone().double().requires_grad_(True) if not native else x.clone().requires_grad_(True)
        if native:
            o = token_log_probs(leaf, tokens, entropy=True, temperature=1.5)
            value = (o.log_probs ** 2).sum() + o.entropy.sum()
        else:
            logp = (leaf / 1.5).log_softmax(-1)
            counts = tokens >= 0
            of = torch.where(counts, logp.gather(1, tokens.clamp_min(0)[:, None])[:, 0], 0.0)
            value = (of ** 2).sum() + torch.where(counts, -(logp.exp() * logp).sum(1), 0.0).sum()
        (g,) = torch.autograd.grad(value, leaf, create_graph=True)
        got.append([g.double(), torch.autograd.grad((g ** 2).sum(), leaf)[0].double()])
    for a, b in zip(*got):
        torch.testing.assert_close(a, b, rtol=1e-4, atol=1e-5)


@pytest.mark.parametrize("rows", [40, 1350])
def test_bits_repeat_and_modes(rows):
    from fairring_b200 import launch_count
    from fairring_b200.ops import token_log_probs

    x = _logits(rows, 50265, torch.bfloat16)
    tokens = torch.randint(0, 50265, (rows,), device="cuda", generator=_gen(7))
    first = token_log_probs(x, tokens, entropy=True, top_k=50)
    for _ in range(5):
        for a, b in zip(first, token_log_probs(x, tokens, entropy=True, top_k=50)):
            assert torch.equal(a, b)
    before = launch_count()
    with torch.inference_mode():
        again = token_log_probs(x, tokens, entropy=True, top_k=50)
    assert launch_count() == before + 1
    assert all(torch.equal(a, b) for a, b in zip(first, again))
    alone = token_log_probs(x, tokens).log_probs  # not the same kernel: its sums are in another order
    with torch.autocast("cuda", dtype=torch.bfloat16):
        assert torch.equal(token_log_probs(x, tokens).log_probs, alone)
    assert torch.equal(token_log_probs(x, tokens.int()).log_probs, alone)


def test_empty_and_refused():
    from fairring_b200.ops import token_log_probs

    none = torch.empty(0, 100, device="cuda", requires_grad=True)
    out = token_log_probs(none, torch.empty(0, dtype=torch.long, device="cuda"), entropy=True, top_k=3)
    assert out.log_probs.shape == (0,) and out.top_tokens.shape == (0, 3)
    (g,) = torch.autograd.grad(out.log_probs.sum(), none)
    assert g.shape == (0, 100)
    x = torch.zeros(2, 10, device="cuda")
    t = torch.zeros(2, dtype=torch.long, device="cuda")
    for bad in (dict(tokens=t.cpu()), dict(tokens=t[:1]), dict(tokens=t.float()), dict(tokens=None), dict(tokens=t, temperature=0.0),
                dict(tokens=t, temperature=float("nan")), dict(tokens=t, top_k=11), dict(tokens=t, top_k=-1)):
        with pytest.raises(ValueError):
            token_log_probs(x, **bad)
    t[1] = 10  # past the vocabulary
    leaf = x.clone().requires_grad_(True)
    out = token_log_probs(leaf, t, entropy=True)
    assert math.isnan(out.log_probs[1]) and abs(float(out.log_probs[0]) + math.log(10)) < 1e-6
    (g,) = torch.autograd.grad(out.log_probs.sum(), leaf)
    assert bool(g[1].isnan().all()) and bool(g[0].isfinite().all())


@pytest.mark.parametrize("rows", [1, 64, 1200])
def test_streams_and_graphs(rows):
    """Two captured calls with their own inputs, replayed in turn and on another stream."""
    from fairring_b200.ops import token_log_probs

    inputs = [(_logits(rows, 20011, torch.bfloat16, seed=i), torch.randint(0, 20011, (rows,), device="cuda", generator=_gen(i)))
              for i in range(2)]
    leaves = [x.clone().requires_grad_(True) for x, _ in inputs]

    def call(i):
        o = token_log_probs(leaves[i], inputs[i][1], entropy=True, top_k=9)
        return [*(v.detach() for v in o), *torch.autograd.grad(o.log_probs.sum() + o.entropy.sum(), leaves[i])]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for i in range(2):
            call(i)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for i in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[i]):
            outs.append(call(i))
    fresh = [_logits(rows, 20011, torch.bfloat16, seed=10 + i) for i in range(2)]
    with torch.no_grad():
        for leaf, x in zip(leaves, fresh):
            leaf.copy_(x)
    side.wait_stream(torch.cuda.current_stream())
    graphs[0].replay()
    with torch.cuda.stream(side):
        graphs[1].replay()
    torch.cuda.current_stream().wait_stream(side)
    for i in range(2):
        for a, b in zip(outs[i], call(i)):
            assert torch.equal(a, b)


def test_second_derivative_past_rows_that_do_not_count():
    """A padded row's logits may be anything, its first and second derivatives are 0."""
    from fairring_b200.ops import token_log_probs

    x = _logits(3, 17, torch.float32)
    x[1] = float("nan")
    leaf = x.requires_grad_(True)
    o = token_log_probs(leaf, torch.tensor([1, -100, 5], device="cuda"), entropy=True)
    (g,) = torch.autograd.grad((o.log_probs ** 2).sum() + o.entropy.sum(), leaf, create_graph=True)
    (h,) = torch.autograd.grad((g ** 2).sum(), leaf)
    for d in (g, h):
        assert bool((d[1] == 0).all()) and bool((d[::2] != 0).any()) and bool(d.isfinite().all())


@pytest.mark.parametrize("rows,vocab,top_k", [(60, 20011, 0), (1300, 20011, 0), (1300, 1003, 0), (700, 20011, 9)])
def test_two_streams_at_once(rows, vocab, top_k):
    from fairring_b200.ops import token_log_probs

    inputs = [(_logits(rows, vocab, torch.bfloat16, seed=i), torch.randint(0, vocab, (rows,), device="cuda", generator=_gen(i)))
              for i in range(2)]

    def call(i):
        leaf = inputs[i][0].detach().requires_grad_(True)
        o = token_log_probs(leaf, inputs[i][1], entropy=True, top_k=top_k)
        return [v.detach() for v in o if v is not None] + list(torch.autograd.grad(o.log_probs.sum() + o.entropy.sum(), leaf))

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


def test_a_vocabulary_past_the_kernels():
    """More columns than an int may step over: refused by the kernels' entry without a look at the logits."""
    from fairring_b200 import _C

    x = torch.zeros(1, device="cuda").expand(1, _C.MOST_VOCAB + 1)
    with pytest.raises(ValueError):
        _C.token_log_probs(x, torch.zeros(1, dtype=torch.long, device="cuda"), 1.0, False, 0)


@pytest.mark.parametrize("vocab", [1, 31, 255, 264, 1025, 2051, 4099, 8200])
@pytest.mark.parametrize("k", [1, 24, 25, 64])
@pytest.mark.parametrize("kind", ["spread", "equal", "few values", "rising", "few left", "not a number"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_top_of_many_short_rows(vocab, k, kind, dtype):
    """One warp a row: vectors that some lanes lack, groups of 1, 2, 4 and 8 vectors, lists that overflow."""
    from fairring_b200.ops import token_log_probs

    rows, k = 5000, min(k, vocab)
    x = _logits(rows, vocab, dtype)
    if kind == "equal":
        x.zero_()
    elif kind == "few values":
        x = x.sign()
    elif kind == "rising":
        x = torch.arange(vocab, device="cuda").expand(rows, vocab).to(dtype).contiguous()
    elif kind == "few left":
        x[:, 3:] = float("-inf")
    elif kind == "not a number":
        x[::3, vocab // 3] = float("nan")
        x[1::3, vocab // 2] = float("inf")
    tokens = torch.randint(0, vocab, (rows,), device="cuda", generator=_gen(3))
    tokens[::7] = -100
    got = token_log_probs(x, tokens, temperature=0.8, top_k=k, entropy=True)
    counts = tokens >= 0
    order = x.sort(dim=1, descending=True, stable=True).indices[:, :k]
    assert torch.equal(got.top_tokens, torch.where(counts[:, None], order, -1))
    logp = (x.double() / 0.8).log_softmax(-1)
    want = torch.where(counts[:, None], logp.gather(1, order), float("-inf"))
    # as _check() has it for the log probabilities
    torch.testing.assert_close(got.top_log_probs.double(), want, rtol=4 * 2.0 ** -24, atol=2.0 ** -17.3, equal_nan=True)
    of = torch.where(counts, logp.gather(1, tokens.clamp_min(0)[:, None])[:, 0], 0.0)
    torch.testing.assert_close(got.log_probs.double(), of, rtol=4 * 2.0 ** -24, atol=2.0 ** -17.3, equal_nan=True)
