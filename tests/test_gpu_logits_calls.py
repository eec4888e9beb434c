"""How the operators on logits are called: what a program around them may have done before, between and after."""

import ctypes

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _student_and_teacher(rows, vocab, k, dtype=torch.bfloat16):
    x = torch.randn(rows, vocab, device="cuda", generator=_gen(vocab)) * 3
    values, tokens = (x + torch.randn(rows, vocab, device="cuda", generator=_gen(1))).log_softmax(-1).topk(k, -1)
    return x.to(dtype), tokens, values


# by a warp a piece, and by a block a piece
@pytest.mark.parametrize("vocab", [1003, 16384])
@pytest.mark.parametrize("k", [5, 40])
def test_the_backward_of_rows_that_were_given_up(vocab, k):
    """Such a row has NaN statistics, and where its tokens would be, whatever the memory held: its gradient is NaN, and
    nothing else is touched."""
    from fairring_b200.ops import distillation_loss

    rows = 7
    x, tokens, given = _student_and_teacher(rows, vocab, k)
    lost = [1, 4, 6]
    found = []

    def give_up(t):
        if t.dim() != 1:
            return t
        t = t.clone()  # 4 floats, 4 of each row, and of each row k pairs of a token's number and a probability
        assert t.numel() == 4 + 4 * rows + 2 * k * rows
        stats, pairs = t[4:4 + 4 * rows].view(rows, 4), t[4 + 4 * rows:].view(rows, k, 2).view(torch.int32)
        assert torch.equal(pairs[..., 0].long(), tokens)
        stats[lost] = float("nan")
        held = torch.tensor([2 ** 31 - 1, vocab, -2 ** 31, -1, 0x7FC00000, vocab + 8, 3], dtype=torch.int32, device="cuda")
        for i, r in enumerate(lost):
            pairs[r, :, 0] = held[(torch.arange(k, device="cuda") + i) % len(held)]
        found.append(True)
        return t

    got = []
    for unpack in (lambda t: t, give_up):
        leaf = x.clone().requires_grad_(True)
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack):
            loss = distillation_loss(leaf, tokens, given, reduction="none")
        got.append(torch.autograd.grad(loss, leaf, torch.ones(rows, device="cuda"))[0])
    assert found
    for r in range(rows):
        assert bool(got[1][r].isnan().all()) if r in lost else torch.equal(got[0][r], got[1][r])


# the forms of the forward: slices of a cluster, a block with more shared memory than a launch has by itself, blocks that stay, a
# warp a row
@pytest.mark.parametrize("rows,vocab", [(3, 20011), (160, 300001), (700, 20011), (700, 1003)])
def test_an_error_that_the_host_has_pending(rows, vocab):
    """It is neither reported by these calls nor cleared."""
    from fairring_b200.ops import distillation_loss, token_log_probs

    x, tokens, given = _student_and_teacher(rows, vocab, 5)
    first = tokens[:, 0].contiguous()
    runtime = ctypes.CDLL("libcudart.so.12")  # the one that torch and the package use

    def calls():
        yield from token_log_probs(x, first, entropy=True)[:2]
        yield from token_log_probs(x, first, top_k=4)[2:]
        for rest in (False, True):
            yield distillation_loss(x, tokens, given, rest=rest)

    want = list(calls())
    torch.cuda.synchronize()
    refused = runtime.cudaSetDevice(4096)  # no such device: an error of the host call alone
    assert refused != 0
    try:
        got = list(calls())
    finally:
        pending = runtime.cudaGetLastError()
    assert pending == refused
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_the_entropys_gradient_past_the_vocabulary(dtype):
    """NaN by the kernel, by the backward that has a graph and by torch's operations, whichever output is used."""
    from fairring_b200.ops.token_log_probs import _plain_token_log_probs, token_log_probs

    x = _student_and_teacher(4, 1003, 1, dtype)[0]
    tokens = torch.tensor([5, 1003, -100, 2 ** 40], device="cuda")
    for used in (lambda o: o.entropy.sum(), lambda o: o.log_probs.sum(), lambda o: o.entropy.sum() + o.log_probs.sum()):
        grads = []
        for call, graph in ((token_log_probs, False), (token_log_probs, True),
                            (lambda z, t, entropy: _plain_token_log_probs(z, t, 1.0, entropy, 0), False)):
            leaf = x.clone().requires_grad_(True)
            out = call(leaf, tokens, entropy=True)
            assert bool(out.entropy.isfinite().all())
            grads.append(torch.autograd.grad(used(out), leaf, create_graph=graph)[0].detach())
        for grad in grads:
            assert bool(grad[1].isnan().all()) and bool(grad[3].isnan().all()) and not grad[2].any()
            # A probability is 2^-20 of itself off, and p |log p| + p H is below 7.4: both sides 2^-17.1, and a rounding to the type.
            torch.testing.assert_close(grad[0], grads[0][0], rtol=torch.finfo(dtype).eps + 2.0 ** -19, atol=2.0 ** -16)


@pytest.mark.parametrize("temperature", [1.0, 2.0])
def test_a_rest_without_probability(temperature):
    """The same by the kernel, by the backward that has a graph and by torch's operations; second derivatives too."""
    from fairring_b200.ops import distillation_loss
    from fairring_b200.ops.distillation import _plain_distillation
    from test_logits_ops import _without_others

    x, tokens, given, want = (t.cuda() for t in _without_others())
    grads, seconds = [], []
    for native, graph in ((True, False), (True, True), (False, True)):
        leaf = (x * temperature).requires_grad_(True)
        loss = (distillation_loss(leaf, tokens, given, temperature=temperature, rest=True, reduction="none") if native
                else _plain_distillation(leaf, tokens, given, temperature, True)[0])
        assert loss.isinf().tolist() == [True, True, False, False]
        (grad,) = torch.autograd.grad(loss.sum(), leaf, create_graph=graph)
        # a probability's 2^-17, and a few roundings of numbers up to 1
        torch.testing.assert_close(grad.double(), want / temperature, rtol=2.0 ** -16, atol=2.0 ** -20)
        if graph:
            seconds.append(torch.autograd.grad((grad ** 2).sum(), leaf)[0])
    assert bool(seconds[0].isfinite().all())
    torch.testing.assert_close(*seconds, rtol=1e-4, atol=1e-6)


@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_second_derivative_past_a_teacher_without_mass(rest, reduction):
    """Listed tokens of minus infinity: without the rest the row does not count, and its derivatives are 0."""
    from fairring_b200.ops import distillation_loss
    from fairring_b200.ops.distillation import _plain_distillation

    x, tokens, given = _student_and_teacher(4, 33, 6, torch.float32)
    given = given - 0.1
    given[1], given[2, 1:] = float("-inf"), float("-inf")
    got = []
    for native in (True, False):
        leaf = x.clone().requires_grad_(True)
        if native:
            loss = distillation_loss(leaf, tokens, given, rest=rest, reduction=reduction)
        else:
            loss, counts = _plain_distillation(leaf, tokens, given, 1.0, rest)
            loss = loss.sum() / counts.sum() if reduction == "mean" else loss
        (g,) = torch.autograd.grad((loss ** 2).sum(), leaf, create_graph=True)
        got.append([g, torch.autograd.grad((g ** 2).sum(), leaf)[0]])
    for a, b in zip(*got):
        assert bool(a.isfinite().all()) and bool(a[1].any()) == rest
        torch.testing.assert_close(a, b, rtol=1e-4, atol=1e-6)


def _other_layout(t):
    """The same values, the last dimension no longer the one without gaps."""
    return t if t.dim() < 2 else t.transpose(-1, -2).contiguous().transpose(-1, -2)


@pytest.mark.parametrize("hooks", ["pinned", "pageable", "another layout"])
@pytest.mark.parametrize("rest", [False, True])
def test_saved_tensors_that_come_back_in_another_layout(hooks, rest):
    from fairring_b200.ops import distillation_loss, token_log_probs

    x, tokens, given = (t.view(4, 9, -1) for t in _student_and_teacher(36, 1003, 5))
    first = tokens[..., 0].clone()
    first[1, 3] = -100

    def grads():
        leaf = x.clone().requires_grad_(True)
        with hook:
            out = token_log_probs(leaf, first, entropy=True)
            loss = distillation_loss(leaf, tokens, given, rest=rest)
        up = torch.randn(2, 4, 9, device="cuda", generator=_gen(3))
        return [*torch.autograd.grad([out.log_probs, out.entropy], leaf, list(up)), *torch.autograd.grad(loss, leaf)]

    hook = torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t)
    want = grads()
    hook = (torch.autograd.graph.saved_tensors_hooks(lambda t: t, _other_layout) if hooks == "another layout"
            else torch.autograd.graph.save_on_cpu(pin_memory=hooks == "pinned"))
    for a, b in zip(grads(), want):
        assert torch.equal(a, b)


def _device_time(call, repeat=5):
    """The least of some runs' microseconds, by events."""
    call()
    times = []
    for _ in range(repeat):
        start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        start.record()
        call()
        end.record()
        end.synchronize()
        times.append(start.elapsed_time(end) * 1000)
    return min(times)


# by a block, by one warp of those that stay, by a warp a row
@pytest.mark.parametrize("rows,vocab", [(40, 51200), (700, 51200), (1400, 8000)])
@pytest.mark.parametrize("fill", [float("-inf"), torch.finfo(torch.bfloat16).min])
def test_a_rest_that_is_masked_takes_no_longer_with_more_listed(rows, vocab, fill):
    """Students that may say nothing but what their teacher lists are looked at again, row by row.  That was done with a look
    through the listed tokens for every logit: 28 times as long with 256 of them as with four."""
    from fairring_b200.ops import distillation_loss

    x, tokens, given = _student_and_teacher(rows, vocab, 256)
    x = torch.full_like(x, fill).scatter_(1, tokens, x.gather(1, tokens))
    few = torch.where(torch.arange(256, device="cuda") < 4, tokens, -1)
    masked = torch.full_like(x, fill).scatter_(1, tokens[:, :4], x.gather(1, tokens[:, :4]))
    times = [_device_time(lambda: distillation_loss(z, t.contiguous(), given[:, : t.shape[1]].contiguous(), rest=True, reduction="none"))
             for z, t in ((masked, few[:, :4]), (x, tokens))]
    assert times[1] <= 8 * times[0], times
