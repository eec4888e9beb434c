"""The operators on logits over the whole range of values, temperatures and vocabularies, every value and gradient shown
to be close."""

import pytest
import torch

from _logits_strict import check_distill, check_score
from test_gpu_distillation import _case

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]


@pytest.fixture(autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _at(rows, vocab, top, seed=0):
    """fp32 rows of deviation 2, one logit 12 above their mean, and that one at `top`."""
    x = torch.randn(rows, vocab, device="cuda", generator=_gen(seed + vocab)) * 2
    x[:, vocab // 2] = 12.0
    return x - 12.0 + top.view(-1, 1)


def _teacher(x, k, seed=0):
    """Some of a row's largest logits and some that are not, unequal parts of 0.9."""
    rows, vocab = x.shape
    tokens = torch.cat([x[:, : vocab // 2 + 1].topk(k - k // 2, -1).indices,
                        vocab // 2 + 1 + torch.rand(rows, vocab - vocab // 2 - 1, device="cuda", generator=_gen(seed)).topk(k // 2, -1).indices], -1)
    given = torch.randn(rows, k, device="cuda", generator=_gen(seed + 1)).log_softmax(-1) - 0.105
    return tokens, given


# The forms that sweep a row: slices of a cluster, a block, blocks that stay, a warp; with largest entries a block and a warp.
FORMS = [(61, 20011), (300, 9001), (732, 17001), (732, 1003)]


# A thread's maximum starts where the fast exponent ends, at -2^20 / c.  Rows whose largest logit is less than 126 below
# have some exponentials left there, and have lost others.
@pytest.mark.parametrize("rows,vocab", FORMS)
@pytest.mark.parametrize("scale", [1.0, 1e-3])
@pytest.mark.parametrize("entropy,top_k", [(True, 0), (False, 0), (True, 5)])
def test_log_probs_at_the_end_of_the_fast_exponent(rows, vocab, scale, entropy, top_k):
    x = _at(rows, vocab, -726850.0 - torch.arange(rows, device="cuda") % 61) * scale
    tokens = torch.randint(0, vocab, (rows,), device="cuda", generator=_gen(2))
    tokens[::2] = vocab // 2
    check_score(x, tokens, scale, entropy, top_k)


@pytest.mark.parametrize("rows,vocab", FORMS)
@pytest.mark.parametrize("scale", [1.0, 1e-3])
@pytest.mark.parametrize("rest", [False, True])
def test_distillation_at_the_end_of_the_fast_exponent(rows, vocab, scale, rest):
    x = _at(rows, vocab, -726850.0 - torch.arange(rows, device="cuda") % 61) * scale
    tokens, given = _teacher(x, 8)
    if rest:  # with every other row's listed logits where they are commonly
        near = (torch.arange(rows, device="cuda") % 2 == 0).view(-1, 1)
        x.scatter_(1, tokens, torch.where(near, x.gather(1, tokens) + 726880.0 * scale, x.gather(1, tokens)))
    check_distill(x, tokens, given if rest else given * scale, scale, rest)


def _equal_but_one(rows, vocab, dtype, top, step):
    """Every logit `step` below `top`, but for one in what each thread of a block sees first: then the exponentials are no powers
    of two, and each addition of one to a sum rounds the same way."""
    x = torch.full((rows, vocab), top - step, device="cuda", dtype=dtype)
    each = 16 // x.element_size()
    x[:, : 256 * each: each] = top
    return x


# What a sum of V logits may be off: 16 additions of a batch's and one for each of V / 4096 batches (32 values of 16 bits or 16 of 32
# a thread of 256, by one block), 23 that merge and rescale; 2^-24 each.
def _sums(vocab):
    return (16 + vocab / 4096 + 23) * 2.0 ** -24


# eight slices a row, two, blocks that stay
@pytest.mark.parametrize("rows", [1, 160, 600])
@pytest.mark.parametrize("kind", ["equal", "spread"])
@pytest.mark.parametrize("dtype", DTYPES)
def test_a_million_columns(rows, kind, dtype):
    vocab = (1 << 20) + (5 if kind == "spread" else 0)
    x = (_equal_but_one(rows, vocab, dtype, 0.0, 5.625) if kind == "equal" else
         (torch.randn(rows, vocab, device="cuda", generator=_gen(1)) * 3).to(dtype))
    tokens = torch.randint(0, vocab, (rows,), device="cuda", generator=_gen(2))
    some = torch.tensor([0, rows // 2, rows - 1], device="cuda")
    check_score(x, tokens, rows=some, sums=_sums(vocab))
    check_score(x, tokens, entropy=False, rows=some, sums=_sums(vocab))


# by a block, and by a warp, whose lanes would round 2^15 times
@pytest.mark.parametrize("rows", [1, 600])
def test_a_million_columns_that_are_looked_at_again(rows):
    x = _equal_but_one(rows, 1 << 20, torch.float32, -3e6, 2.5)
    tokens = torch.randint(0, 1 << 20, (rows,), device="cuda", generator=_gen(2))
    check_score(x, tokens, rows=torch.tensor([0, rows - 1], device="cuda"), sums=40 * 2.0 ** -24)


# ---- what the other tests of these operators look at too, with checks that a NaN cannot pass ----------------------------
def _logits(rows, vocab, dtype, seed=0):
    x = torch.randn(rows, vocab, device="cuda", generator=_gen(seed + vocab)) * 3
    x[:, vocab // 2] += 6
    return x.to(dtype)


def _tokens(rows, vocab):
    tokens = torch.randint(0, vocab, (rows,), device="cuda", generator=_gen(vocab))
    if rows > 5:
        tokens[3], tokens[4], tokens[5] = -100, 0, vocab - 1
    return tokens


@pytest.mark.parametrize("rows", [1, 19, 400, 1300])
@pytest.mark.parametrize("vocab", [1, 7, 9, 1001, 4096, 8193, 16385, 32776])
@pytest.mark.parametrize("dtype", DTYPES)
def test_log_probs_of_every_form(rows, vocab, dtype):
    x, tokens = _logits(rows, vocab, dtype), _tokens(rows, vocab)
    check_score(x, tokens, 0.7, top_k=min(vocab, 5))
    check_score(x, tokens, entropy=False)


@pytest.mark.parametrize("rows", [1, 19, 400, 1300])
@pytest.mark.parametrize("vocab,k", [(2, 1), (7, 3), (1001, 256), (8193, 64), (16385, 33), (32776, 5)])
@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
def test_distillation_of_every_form(rows, vocab, k, rest, dtype):
    x, tokens, given = _case(rows, vocab, k, dtype)
    check_distill(x, tokens, given - 0.2 if rest else given, 1.3, rest)


@pytest.mark.parametrize("rows,vocab", FORMS)
@pytest.mark.parametrize("temperature", [1e-6, 1e-3, 1e6])
@pytest.mark.parametrize("dtype", DTYPES)
def test_log_probs_at_extreme_temperatures(rows, vocab, temperature, dtype):
    x, tokens = _logits(rows, vocab, dtype), _tokens(rows, vocab)
    tokens[6::3] = x[6::3].float().argmax(-1)
    check_score(x, tokens, temperature, top_k=5)


@pytest.mark.parametrize("rows,vocab", FORMS)
@pytest.mark.parametrize("temperature", [1e-6, 1e-3, 1e6])
@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
def test_distillation_at_extreme_temperatures(rows, vocab, temperature, rest, dtype):
    """The teacher is as sharp as the student, or with the rest is what it is."""
    x, tokens, given = _case(rows, vocab, 20, dtype)
    check_distill(x, tokens, given * 1.2 - 0.1 if rest else given, temperature, rest)


@pytest.mark.parametrize("rows,vocab", FORMS)
@pytest.mark.parametrize("shift", [3e6, -3e6, 1e30, -1e30])
@pytest.mark.parametrize("rest", [False, True])
def test_distillation_far_from_zero(rows, vocab, shift, rest):
    """Every row, every other row, and of every other row what is not listed or only that."""
    base, tokens, given = _case(rows, vocab, 9, torch.float32, padded=0.0)
    given = given * 1.2 - 0.1 if rest else given
    listed = torch.zeros(rows, vocab, dtype=torch.bool, device="cuda").scatter_(1, tokens.clamp_min(0), True)
    odd = (torch.arange(rows, device="cuda") % 2 == 1).view(-1, 1)
    for where in (torch.ones_like(odd), odd, odd & ~listed, odd & listed):
        check_distill(torch.where(where, base + shift, base), tokens, given, 1.0, rest)


@pytest.mark.parametrize("rows,vocab", FORMS)
@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
def test_distillation_of_masked_logits(rows, vocab, rest, dtype):
    """Minus infinity and the type's lowest value, up to all that is not listed and whole rows."""
    lowest = torch.finfo(dtype).min
    for fill in (float("-inf"), lowest):
        x, tokens, given = _case(rows, vocab, 9, dtype)
        given = given * 1.2 - 0.1 if rest else given
        listed = torch.zeros(rows, vocab, dtype=torch.bool, device="cuda").scatter_(1, tokens.clamp_min(0), True)
        gone = torch.rand(rows, vocab, device="cuda", generator=_gen(3)) < 0.9
        gone[1] = True
        gone[1, vocab - 1] = False  # a single one left that is not listed
        gone[3, : vocab - 30] = True  # whole slices without one
        gone &= ~listed
        gone[:, 5] &= fill == lowest  # with the rest, of minus infinity the loss would be infinite
        if fill == lowest:
            gone[4], x[5] = ~listed[4], lowest
        check_distill(x.masked_fill(gone, fill), tokens, given, 1.0, rest)


@pytest.mark.parametrize("rows,vocab", FORMS)
@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
def test_distillation_of_values_that_are_no_numbers(rows, vocab, rest, dtype):
    """NaN and infinity, listed or not, make their own row NaN and no other; a row that does not count may hold anything."""
    from fairring_b200.ops import distillation_loss

    x, tokens, given = _case(rows, vocab, 9, dtype, padded=0.0)
    given = given * 1.2 - 0.1 if rest else given
    tokens[4:6], bad = -1, x.clone()
    listed = torch.zeros(rows, vocab, dtype=torch.bool, device="cuda").scatter_(1, tokens.clamp_min(0), True)
    bad[0, int((~listed[0]).nonzero()[7])] = float("nan")
    bad[1, int((~listed[1]).nonzero()[-1])] = float("inf")
    bad[6, tokens[6, 2]], bad[3, tokens[3, 4]] = float("nan"), float("inf")
    bad[4], bad[5, 0] = float("nan"), float("inf")
    got = []
    for z in (x, bad):
        leaf = z.clone().requires_grad_(True)
        loss = distillation_loss(leaf, tokens, given, rest=rest, reduction="none")
        got.append((loss.detach(), torch.autograd.grad(loss, leaf, torch.ones(rows, device="cuda"))[0]))
    broken = [0, 1, 3, 6]
    fine = torch.ones(rows, dtype=torch.bool, device="cuda")
    fine[broken] = False
    for a, b in zip(*got):
        assert bool(b[broken].isnan().all()) and bool(a.isfinite().all())
        assert torch.equal(a[fine], b[fine]) and not b[4:6].any()


# slices with more shared memory than a launch has by itself; a block a row where blocks that stay would hold too many marks;
# the widest
@pytest.mark.parametrize("rows,vocab", [(5, 1 << 20), (160, 520_001), (600, 220_001), (600, 1 << 20)])
@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_distillation_over_wide_vocabularies(rows, vocab, rest, dtype):
    x = torch.randn(rows, vocab, device="cuda", generator=_gen(vocab)).mul_(3).to(dtype)
    tokens = torch.randint(0, vocab, (rows, 64), device="cuda", generator=_gen(1))
    tokens[:, 3], tokens[:, 4], tokens[1, 9], tokens[0, 7] = 0, vocab - 1, tokens[1, 8], -1
    given = torch.randn(rows, 64, device="cuda", generator=_gen(2)).log_softmax(-1) - 0.105
    x.scatter_add_(1, tokens.clamp_min(0), torch.full((rows, 64), 6.0, device="cuda", dtype=dtype))
    check_distill(x, tokens, given, 1.0, rest, rows=torch.tensor([0, 1, rows // 2, rows - 1], device="cuda"), sums=_sums(vocab))


# blocks that stay, a block a row where there are largest entries or marks too many, a warp a row
@pytest.mark.parametrize("rows,vocab", [(2100, 1 << 20), (2_200_003, 1001)])
def test_rows_past_two_to_the_31_elements(rows, vocab):
    x = torch.empty(rows, vocab, device="cuda", dtype=torch.bfloat16).normal_(0, 3, generator=_gen(1))
    some = torch.tensor([0, 1, rows // 2, rows - 2, rows - 1], device="cuda")
    check_score(x, torch.randint(0, vocab, (rows,), device="cuda", generator=_gen(2)), top_k=9, rows=some, sums=_sums(vocab))
    check_score(x, torch.randint(0, vocab, (rows,), device="cuda", generator=_gen(2)), entropy=False, rows=some, sums=_sums(vocab))
    tokens = torch.randint(0, vocab, (rows, 6), device="cuda", generator=_gen(3))
    given = torch.randn(rows, 6, device="cuda", generator=_gen(4)).log_softmax(-1) - 0.2
    for rest in (False, True):
        check_distill(x, tokens, given, 1.0, rest, rows=some, sums=_sums(vocab))
