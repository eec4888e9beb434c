"""Log probabilities and distillation in 64 bits, from the definitions, with torch's autograd for the gradients."""

import math

import torch


def score(logits, tokens, temperature=1.0, g=None, h=None):
    """(log probabilities, entropy, gradient of sum(g * log_probs) + sum(h * entropy), log-softmax)."""
    leaf = logits.detach().double().requires_grad_(True)
    logp = (leaf / temperature).log_softmax(-1)
    counts = tokens >= 0
    of = logp.gather(-1, tokens.clamp_min(0).unsqueeze(-1)).squeeze(-1)
    of = torch.where(counts, of, 0.0)
    entropy = -(logp.exp() * logp.masked_fill(logp == float("-inf"), 0.0)).sum(-1)
    entropy = torch.where(counts, entropy, 0.0)
    total = (of * (0.0 if g is None else g.double())).sum() + (entropy * (0.0 if h is None else h.double())).sum()
    (grad,) = torch.autograd.grad(total, leaf)
    return of.detach(), entropy.detach(), grad, logp.detach()


def distill(logits, tokens, given, temperature=1.0, rest=False, g=None):
    """(loss of every row, gradient of sum(g * loss), log-softmax), a row at a time."""
    flat = logits.detach().double().reshape(-1, logits.shape[-1])
    where = tokens.reshape(flat.shape[0], -1).cpu().tolist()
    values = given.detach().double().reshape(flat.shape[0], -1).tolist()
    losses, grads, all_logp = [], [], []
    up = torch.ones_like(flat[:, 0]) if g is None else g.double().reshape(-1)
    for r in range(flat.shape[0]):
        x = flat[r].clone().requires_grad_(True)
        logp = (x / temperature).log_softmax(-1)
        all_logp.append(logp.detach())
        there = [k for k, t in enumerate(where[r]) if t >= 0]
        if not rest and all(values[r][k] == float("-inf") for k in there):
            there = []
        if not there:
            losses.append(torch.zeros_like(flat[r, 0]))
            grads.append(torch.zeros_like(flat[r]))
            continue
        at = torch.tensor([where[r][k] for k in there], device=flat.device)
        logq = torch.tensor([values[r][k] for k in there], dtype=torch.float64, device=flat.device)
        if not rest:
            logq = (logq / temperature).log_softmax(-1)
        some = logq > float("-inf")
        loss = (logq[some].exp() * (logq[some] - logp[at[some]])).sum()
        left = 1 - float(logq.exp().sum())
        if rest and left >= 2.0 ** -20:  # less is the rounding of the teacher's values
            others = torch.ones_like(x, dtype=torch.bool)
            others[at] = False
            loss = loss + left * (math.log(left) - logp[others].logsumexp(0))
        losses.append(loss.detach())
        grads.append(torch.autograd.grad(loss, x)[0] * up[r])
    shape = logits.shape
    return torch.stack(losses).view(shape[:-1]), torch.stack(grads).view(shape), torch.stack(all_logp).view(shape)


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def smallest_step(dtype):
    """Half the distance of the type's smallest numbers; results of the kernels' exponentials below fp32's normal
    numbers are zero."""
    return {torch.float16: 2.0 ** -25}.get(dtype, 2.0 ** -126)


# A probability's relative error: exp2's own is 2^-22, its argument's three roundings (difference, constant,
# product) are 2^-24 of it each, and it is at most 150 for what is not zero: 2^-14.7 at the far end, where the
# probability is 2^-150.  For log2(p) = u it is 2^-22 + 3 * 2^-24 |u|.  The sum of a row takes at most 4 * 4 additions in a
# thread's batch, one per batch (32 of them for 131072 logits of 16 bits) and 5 + 8 + 8 merges, 2^-24 each and two more for
# the rescaling: 2^-17.4 if all go one way.
def relative(logp):
    return 2.0 ** -17.4 + 2.0 ** -22 + 3 * 2.0 ** -24 / 0.6931 * logp.clamp_min(-110.0).abs()
