"""The operators on logits over the whole range of values, temperatures and vocabularies, every value and gradient shown
to be close."""

import pytest
import torch

from _logits_strict import check_distill, check_score

pytestmark = pytest.mark.gpu


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
