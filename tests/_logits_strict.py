"""Checks of the operators on logits that a NaN cannot pass: the error has to be shown small, not large."""

import torch

from _logits_oracle import half_step, relative, score, smallest_step


def within(got, want, room):
    """Every value within its room of the one wanted; NaN and infinities where those are, and nowhere else."""
    got, room = got.detach().double(), torch.as_tensor(room, device=got.device).expand(got.shape)
    assert got.shape == want.shape and bool((room >= 0).all()) and bool(room.isfinite().all())
    ok = torch.where(want.isnan(), got.isnan(), (got == want) | ((got - want).abs() <= room))
    assert bool(ok.all()), (int((~ok).sum()), got[~ok][:4].tolist(), want[~ok][:4].tolist(), room[~ok][:4].tolist())


def _rounded(grad, dtype):
    """Infinite where the type has no such number: what lies past its largest number by half a step."""
    past = grad.abs() > torch.finfo(dtype).max * (1 + half_step(dtype) / 2)
    return torch.where(past, grad.sign() * float("inf"), grad)


def check_score(logits, tokens, temperature=1.0, entropy=True, top_k=0, rows=None, sums=2.0 ** -17.3):
    """`rows`: those of a [rows, vocab] matrix whose values are looked at.  `sums`: the relative error of a row's sum.  The other
    bounds are those of the oracle's relative()."""
    from fairring_b200.ops import token_log_probs

    gen = torch.Generator(device=logits.device).manual_seed(1)
    g = torch.randn(tokens.shape, device=logits.device, generator=gen)
    h = torch.randn(tokens.shape, device=logits.device, generator=gen)
    leaf = logits.detach().requires_grad_(True)
    got = token_log_probs(leaf, tokens, temperature=temperature, entropy=entropy, top_k=top_k)
    (grad,) = torch.autograd.grad([got.log_probs, got.entropy] if entropy else got.log_probs, leaf, [g, h] if entropy else g)
    if rows is not None:
        got = type(got)(*(v if v is None else v.detach()[rows] for v in got))
        logits, tokens, g, h, grad = (t[rows] for t in (logits, tokens, g, h, grad))
    want, want_h, want_grad, logp = score(logits, tokens, temperature, g, h if entropy else None)
    counts = tokens >= 0
    # the difference to the maximum, the temperature, the product and the sum: 2^-24 each
    within(got.log_probs, want, sums + 4 * 2.0 ** -24 * want.abs().where(want.isfinite(), 0.0))
    p, far = logp.exp(), logp.clamp_min(-110).abs()
    off = relative(logp) + sums
    if entropy:
        within(got.entropy, want_h, torch.where(counts, (p * (1 + far) * off).sum(-1) * 2 + sums, 0.0))
    if top_k:
        order = logits.float().sort(dim=-1, descending=True, stable=True).indices[..., :top_k]
        assert torch.equal(got.top_tokens, order.where(counts.unsqueeze(-1), -1))
        top = logp.gather(-1, order)
        room = sums + 4 * 2.0 ** -24 * top.abs().where(top.isfinite(), 0.0)
        within(got.top_log_probs, top.where(counts.unsqueeze(-1), float("-inf")), room)
    size = p * (g.double().abs().unsqueeze(-1) + (h.double().abs() * (1 + want_h)).unsqueeze(-1) * (1 + far)) / temperature
    # the type's half step; the probability; its flush to zero below 2^-126, with the factors that it meets; the 1 of the token
    room = half_step(logits.dtype) * want_grad.abs() + 2 * off * size + smallest_step(logits.dtype)
    room = room + 2.0 ** -126 * (g.double().abs() + 128 * h.double().abs()).unsqueeze(-1) / temperature
    room = room + 2.0 ** -22 * g.double().abs().unsqueeze(-1) / temperature * torch.zeros_like(p).scatter_(
        -1, tokens.clamp_min(0).unsqueeze(-1), 1.0)
    within(grad, _rounded(want_grad, logits.dtype), torch.where(counts.unsqueeze(-1), room, 0.0))
    return got, grad


def distill_by_formula(logits, tokens, given, temperature=1.0, rest=False, g=None):
    """(loss of every row, gradient of sum(g * loss), log-softmax, logarithm of the others' share), in 64 bits.  Beside logits of
    1e16 and more a logarithm is lost even there, so every sum is of differences to its own largest value."""
    low = float("-inf")
    x, given = logits.detach().double(), given.detach().double()
    there = tokens >= 0
    at = tokens.clamp_min(0)
    counts = (there if rest else there & (given != low)).any(-1)

    def log_sum(z):
        top = z.amax(-1, keepdim=True)
        return top, ((z - top) / temperature).exp().sum(-1, keepdim=True).log()

    top, log_s = log_sum(x)
    logp = (x - top) / temperature - log_s
    p = logp.exp()
    if rest:
        log_q = given.masked_fill(~there, low)
    else:
        log_q = (given / temperature).masked_fill(~(there & counts.unsqueeze(-1)), low).log_softmax(-1)
        log_q = log_q.masked_fill(~there, low)
    q = torch.where(there & counts.unsqueeze(-1), log_q.exp(), 0.0)
    loss = torch.where(q > 0, q * (log_q - logp.gather(-1, at)), 0.0).sum(-1)
    q_of = torch.zeros_like(p).scatter_add_(-1, at, q)
    mass, log_rest = q.sum(-1, keepdim=True), None
    grad = p * mass - q_of
    if rest:
        left = 1 - mass
        left = left.where(left >= 2.0 ** -20, 0.0)  # less is the rounding of the teacher's values
        listed = torch.zeros_like(p).scatter_add_(-1, at, there.double()) > 0
        others = x.masked_fill(listed, low)
        top_o, log_o = log_sum(others)
        none = top_o == low
        log_rest = torch.where(none, low, (top_o - top) / temperature + log_o - log_s)
        share = torch.where(none | listed, 0.0, ((others - top_o) / temperature - log_o).exp())
        loss = loss + torch.where(left > 0, left * (left.log() - log_rest), 0.0).squeeze(-1)
        grad = torch.where(listed, p * (mass + left) - q_of, share * ((mass + left) * log_rest.exp() - left))
        log_rest = log_rest.squeeze(-1)
    up = 1.0 if g is None else g.double().unsqueeze(-1)
    grad = torch.where(counts.unsqueeze(-1), grad * up / temperature, 0.0)
    return torch.where(counts, loss, 0.0), grad, logp, log_rest


def check_distill(logits, tokens, given, temperature=1.0, rest=False, rows=None, sums=2.0 ** -17.4):
    """`rows`: those of a [rows, vocab] matrix whose values are looked at."""
    from fairring_b200.ops import distillation_loss

    gen = torch.Generator(device=logits.device).manual_seed(1)
    g = torch.randn(logits.shape[:-1], device=logits.device, generator=gen)
    leaf = logits.detach().requires_grad_(True)
    loss = distillation_loss(leaf, tokens, given, temperature=temperature, rest=rest, reduction="none")
    (grad,) = torch.autograd.grad(loss, leaf, g)
    assert loss.dtype == torch.float32 and grad.dtype == logits.dtype and grad.shape == logits.shape
    if rows is not None:
        logits, tokens, given, g, loss, grad = (t[rows] for t in (logits, tokens, given, g, loss.detach(), grad))
    want, want_grad, logp, others = distill_by_formula(logits, tokens, given, temperature, rest, g)
    low = float("-inf")
    there = (tokens >= 0) & ~(given == low)
    counts = ((tokens >= 0) if rest else there).any(-1)
    log_q = given.double() if rest else (given.double() / temperature).masked_fill(~there, low).log_softmax(-1)
    log_q = torch.where(there & counts.unsqueeze(-1), log_q, -1e30)
    log_p = logp.gather(-1, tokens.clamp_min(0))
    apart = log_q.abs() + log_p.abs().where(log_p.isfinite(), 0.0) + 1
    # A teacher's probability: an exponential (2^-22), its argument's roundings (2^-23 of it) and a sum of up to 13
    # additions (2^-20.3), once more in what it weighs; the logarithms' own roundings; the row's sum, and the rest's.
    q_off = 2.0 ** -19.5 + 2.0 ** -22 * log_q.abs().clamp_max(110)
    room = (log_q.exp() * apart * (q_off + 2.0 ** -22)).sum(-1) + 2 * sums + 2.0 ** -24
    if rest:  # what is left is the sum's rounding off, 2^-23, and weighs the logarithm of the others' share
        room = room + (2.0 ** -21 + log_q.exp().sum(-1) * 2.0 ** -21) * (1 + others.abs().where(others.isfinite(), 0.0))
    room = room + 2.0 ** -22 * want.abs().where(want.isfinite(), 0.0)
    past = want.abs() > torch.finfo(torch.float32).max
    within(loss, torch.where(past, want.sign() * float("inf"), want), torch.where(counts, room, 0.0))
    p = logp.exp()
    share, named = p, torch.zeros_like(p).scatter_add_(-1, tokens.clamp_min(0), (tokens >= 0).double()) > 0
    if rest:  # the weight of the others' is a difference of two numbers up to 1, over their probability
        x = logits.double().masked_fill(named, low)
        share = p + ((x - x.amax(-1, keepdim=True).clamp_min(torch.finfo(torch.float32).min)) / temperature).softmax(-1).nan_to_num(0.0)
    scale = g.double().abs().unsqueeze(-1) / temperature
    room = half_step(logits.dtype) * want_grad.abs() + smallest_step(logits.dtype)
    room = room + scale * (2 * (relative(logp) + sums) * share + 2.0 ** -18.5 * named + 2.0 ** -126)
    within(grad, _rounded(want_grad, logits.dtype), torch.where(counts.unsqueeze(-1), room, 0.0))
    return loss, grad
