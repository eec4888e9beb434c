"""The operators on a language-model head's logits, as cases that can be timed.

``score``    ``token_log_probs``: log probabilities of given tokens, entropy and top alternatives, with
             ``train`` also the gradient of the logits
``distill``  ``distillation_loss``: divergence from a teacher's top log probabilities, with ``train`` also
             the gradient of the logits

Where ``own`` is false, :func:`run` computes them from elementary torch operations in fp32; where it is
true, through the package.  A case: ``batch`` x ``seq`` rows of ``vocab`` logits; with ``shift`` the
logits are those of ``seq + 1`` positions without the last, as a language model is scored against the
tokens that follow, so that the rows of a sequence are contiguous and the batch is not.
"""

import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
DEVICE = "cuda"
MOST_BYTES = 8192 * 51200 * 2  # of the logits of a drawn case, as in the largest listed ones


# ---- the cases --------------------------------------------------------------------------------
def _score(name, batch, seq, vocab, dtype, *, top_k=0, entropy=False, temperature=1.0, tokens=True, ignored=0.0,
           masked=0.0, shift=False, train=False):
    return {"name": name, "kind": "score", "batch": batch, "seq": seq, "vocab": vocab, "dtype": dtype, "top_k": top_k,
            "entropy": entropy, "temperature": temperature, "tokens": tokens, "ignored": ignored, "masked": masked,
            "shift": shift, "train": train}


def _distill(name, batch, seq, vocab, dtype, k, *, rest=False, temperature=1.0, ignored=0.0, reduction="mean",
             shift=False, train=True):
    return {"name": name, "kind": "distill", "batch": batch, "seq": seq, "vocab": vocab, "dtype": dtype, "k": k,
            "rest": rest, "temperature": temperature, "ignored": ignored, "reduction": reduction, "shift": shift,
            "train": train}


def listed():
    return [
        # One token of one sequence has been drawn from the decoder's vocabulary: its log probability, the
        # entropy and five alternatives go with the answer.  All latency.
        _score("score_1x51200", 1, 1, 51200, "bf16", top_k=5, entropy=True),
        # The same for a batch of sequences over an odd vocabulary, sampled at 0.7 from a grammar that
        # allows a tenth of the tokens.
        _score("score_48x50265", 1, 48, 50265, "fp16", top_k=20, entropy=True, temperature=0.7, masked=0.9),
        # Texts scored in full precision (perplexity, ranking): log probabilities only.
        _score("score_2x1023x50265", 2, 1023, 50265, "fp32", ignored=0.1, shift=True),
        # A teacher's top 64 of every position of eight sequences, to be learnt from later.
        _score("teacher_8192x51200", 8, 1024, 51200, "bf16", top_k=64, tokens=False),
        # Policy-gradient training: the log probabilities of what was sampled, an entropy bonus, a
        # quarter of the positions are prompt.
        _score("policy_4x1024x51200", 4, 1024, 51200, "bf16", entropy=True, ignored=0.25, shift=True, train=True),
        # The same in full precision at sizes that divide into nothing, without the bonus.
        _score("policy_701x32003", 1, 701, 32003, "fp32", temperature=0.9, ignored=0.3, train=True),
        # Distilling into the small test model: all launches and host.
        _distill("distill_4x63x1024", 4, 63, 1024, "fp32", 8, shift=True),
        # The decoder learns from a teacher's top 64 at temperature 2.
        _distill("distill_8192x51200", 8, 1024, 51200, "bf16", 64, temperature=2.0),
        # The same with the teacher's remaining probability as one more class; padded sequences.
        _distill("distill_rest_2x1024x51200", 2, 1024, 51200, "bf16", 32, rest=True, ignored=0.1, shift=True),
        # Masked positions of the encoder under an odd vocabulary, in half precision, weighted one by one.
        _distill("distill_1229x50265", 1, 1229, 50265, "fp16", 100, temperature=1.5, reduction="none", ignored=0.05),
        # Validation: the loss of every position without a gradient, full precision, a wide vocabulary.
        _distill("distill_eval_515x128003", 1, 515, 128003, "fp32", 16, rest=True, reduction="none", train=False),
    ]


def draw(rng):
    def spread(low, high):
        return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))

    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    vocab = spread(512, 131072)
    most = MOST_BYTES // (vocab * (4 if dtype == "fp32" else 2))
    rows = min(spread(1, 8192), most - 8)
    batch = min(rows, rng.choice([1, 1, 2, 3, 8]))
    seq = max(1, rows // batch)
    shift = seq > 1 and rng.random() < 0.4
    temperature = rng.choice([1.0, 1.0, 0.7, 2.0])
    ignored = rng.choice([0.0, 0.1, 0.5]) if rows >= 8 else 0.0
    if rng.random() < 0.5:
        train = rng.random() < 0.5
        entropy = rng.random() < 0.5
        top_k = 0 if train else rng.choice([0, 1, 5, 20, spread(1, 128)])
        tokens = train or top_k == 0 or rng.random() < 0.7
        case = _score("", batch, seq, vocab, dtype, top_k=top_k, entropy=entropy, temperature=temperature, tokens=tokens,
                      ignored=ignored if tokens else 0.0, masked=rng.choice([0.0, 0.0, 0.8]), shift=shift, train=train)
    else:
        case = _distill("", batch, seq, vocab, dtype, spread(4, 128), rest=rng.random() < 0.5, temperature=temperature,
                        ignored=ignored, reduction=rng.choice(["mean", "none"]), shift=shift, train=rng.random() < 0.7)
    del case["name"]
    return case


# ---- inputs -----------------------------------------------------------------------------------
def prepare(case, seed):
    """Logits as a trained head gives them: frequent and rare tokens, and at every position one or a few
    that stand out; masked ones are minus infinity."""
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    b, s, v = case["batch"], case["seq"], case["vocab"]
    rows = b * s if b == 1 or not case["shift"] else b * (s + 1)
    rows += 1 if b == 1 and case["shift"] else 0
    x = torch.randn(rows, v, device=DEVICE, generator=gen)
    x += torch.randn(v, device=DEVICE, generator=gen) * 2
    likely = torch.randint(0, v, (rows, 3), device=DEVICE, generator=gen)
    x.scatter_add_(1, likely, torch.rand(rows, 3, device=DEVICE, generator=gen) * 8)
    x = x.to(DTYPES[case["dtype"]]).view(b, -1, v)
    logits = x[:, :s]
    likely = likely.view(b, -1, 3)[:, :s]
    counts = torch.rand(b, s, device=DEVICE, generator=gen) >= case["ignored"]
    state = {"case": case, "logits": logits}
    if case["kind"] == "score":
        tokens = likely[..., 0]
        if case["masked"]:
            mask = torch.rand(b, s, v, device=DEVICE, generator=gen) < case["masked"]
            mask.scatter_(2, tokens.unsqueeze(2), False)
            logits.masked_fill_(mask, float("-inf"))
        state["tokens"] = tokens.where(counts, -100).contiguous() if case["tokens"] else None
    else:
        # The teacher sees almost what the student sees; its log probabilities are over the whole vocabulary.
        k, t = min(case["k"], v), case["temperature"] if case["rest"] else 1.0
        values, tokens = logits.topk(k, dim=-1)
        values = values.float() + torch.randn(b, s, k, device=DEVICE, generator=gen) * 0.3
        values, order = values.sort(dim=-1, descending=True)
        kept = 0.98 if k < v else 1.0
        state["teacher_log_probs"] = (values / t).log_softmax(-1) + math.log(kept)
        state["teacher_tokens"] = tokens.gather(-1, order).where(counts.unsqueeze(2), -1)
    if case["train"]:  # half precision is trained with a scaled loss
        scale = 8192.0 if case["dtype"] == "fp16" else 1.0
        if case["kind"] == "distill" and case["reduction"] == "mean":
            state["upstream"] = [torch.full((), scale, device=DEVICE)]
        else:
            state["upstream"] = [torch.randn(b, s, device=DEVICE, generator=gen) * (scale / (b * s)),
                                 torch.full((b, s), 1e-3 * scale / (b * s), device=DEVICE)]
    return state


# ---- plain forms ------------------------------------------------------------------------------
def _largest(x, k):
    """The k largest of each row in falling order, the lowest index first among equals: (values, indices)."""
    bits = (x.float() + 0.0).view(torch.int32)
    key = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).to(torch.int64) << 32
    key |= 0xFFFFFFFF - torch.arange(x.shape[-1], device=x.device)
    at = 0xFFFFFFFF - (key.topk(k, dim=-1).values & 0xFFFFFFFF)
    return x.float().gather(-1, at), at


def _plain_score(state):
    case, x = state["case"], state["logits"]
    tokens, scale = state["tokens"], 1.0 / case["temperature"]
    z = x.float() * scale
    d = z - z.amax(-1, keepdim=True)
    e = d.exp()
    total = e.sum(-1, keepdim=True)
    low = total.log()
    out = {}
    counts = tokens >= 0 if tokens is not None else torch.ones(x.shape[:-1], dtype=torch.bool, device=x.device)
    if tokens is not None:
        at = tokens.clamp_min(0).unsqueeze(-1)
        out["log_probs"] = torch.where(counts, (d.gather(-1, at) - low).squeeze(-1), 0.0)
    if case["entropy"]:
        h = low - torch.where(e > 0, e * d, 0.0).sum(-1, keepdim=True) / total
        out["entropy"] = torch.where(counts, h.squeeze(-1), 0.0)
    if case["top_k"]:
        values, at = _largest(x, case["top_k"])
        log_probs = values * scale - z.amax(-1, keepdim=True) - low
        out["top_log_probs"] = torch.where(counts.unsqueeze(-1), log_probs, float("-inf"))
        out["top_tokens"] = torch.where(counts.unsqueeze(-1), at, -1)
    if case["train"]:
        g = state["upstream"][0].unsqueeze(-1) * scale
        p = e / total
        grad = -p * g
        if case["entropy"]:
            gh = state["upstream"][1].unsqueeze(-1) * scale
            grad = grad - gh * torch.where(p > 0, p * (d - low + h), 0.0)
        grad.scatter_add_(-1, tokens.clamp_min(0).unsqueeze(-1), g)
        out["grad"] = torch.where(counts.unsqueeze(-1), grad, 0.0).to(x.dtype)
    return out


def _plain_distill(state):
    case, x, tokens, given = state["case"], state["logits"], state["teacher_tokens"], state["teacher_log_probs"]
    scale = 1.0 / case["temperature"]
    there = tokens >= 0
    counts = there.any(-1)
    at = tokens.clamp_min(0)
    z = x.float() * scale
    d = z - z.amax(-1, keepdim=True)
    e = d.exp()
    total = e.sum(-1, keepdim=True)
    if case["rest"]:
        q = torch.where(there, given.exp(), 0.0)
        log_q = given
    else:
        t = torch.where(there, given * scale, float("-inf"))
        t = t - t.amax(-1, keepdim=True).clamp_min(-1e30)
        below = t.exp().sum(-1, keepdim=True)
        log_q = t - below.log()
        q = torch.where(there, log_q.exp(), 0.0)
    terms = torch.where(q > 0, q * (log_q - (d.gather(-1, at) - total.log())), 0.0)
    rows = terms.sum(-1)
    if case["rest"]:
        q_rest = (1 - q.sum(-1, keepdim=True)).clamp_min(0)
        outside = torch.ones_like(z).scatter_(-1, at, 0.0)
        e_rest = e * outside
        p_rest = e_rest.sum(-1, keepdim=True) / total
        rows = rows + torch.where(q_rest > 0, q_rest * (q_rest.log() - p_rest.log()), 0.0).squeeze(-1)
    rows = torch.where(counts, rows, 0.0)
    number = counts.sum().clamp_min(1)
    out = {"loss": rows.sum() / number if case["reduction"] == "mean" else rows}
    if case["train"]:
        grad = e / total
        if case["rest"]:
            grad = grad * (q.sum(-1, keepdim=True) + q_rest)
            grad = grad - e_rest / e_rest.sum(-1, keepdim=True) * q_rest
        grad.scatter_add_(-1, at, -q)
        up = state["upstream"][0]
        up = up.unsqueeze(-1) if case["reduction"] == "none" else up / number
        out["grad"] = torch.where(counts.unsqueeze(-1), grad * (up * scale), 0.0).to(x.dtype)
    return out


# ---- a pass -----------------------------------------------------------------------------------
def _own_score(state):
    from fairring_b200.ops import token_log_probs

    case = state["case"]
    logits = state["logits"].detach().requires_grad_(case["train"])
    got = token_log_probs(logits, state["tokens"], temperature=case["temperature"], entropy=case["entropy"],
                          top_k=case["top_k"])
    out = {name: value.detach() for name, value in got._asdict().items() if value is not None}
    if case["train"]:
        outputs = [got.log_probs, got.entropy] if case["entropy"] else [got.log_probs]
        out["grad"] = torch.autograd.grad(outputs, logits, state["upstream"][: len(outputs)])[0]
    return out


def _own_distill(state):
    from fairring_b200.ops import distillation_loss

    case = state["case"]
    logits = state["logits"].detach().requires_grad_(case["train"])
    loss = distillation_loss(logits, state["teacher_tokens"], state["teacher_log_probs"],
                             temperature=case["temperature"], rest=case["rest"], reduction=case["reduction"])
    out = {"loss": loss.detach()}
    if case["train"]:
        out["grad"] = torch.autograd.grad(loss, logits, state["upstream"][0])[0]
    return out


def run(state):
    if own:
        return _own_score(state) if state["case"]["kind"] == "score" else _own_distill(state)
    return _plain_score(state) if state["case"]["kind"] == "score" else _plain_distill(state)


def work(case):
    """Rows that do not count need not be read; their gradient is written all the same."""
    rows, v = case["batch"] * case["seq"], case["vocab"]
    size = 4 if case["dtype"] == "fp32" else 2
    read = rows * (1 - case["ignored"])
    moved, done = read * v * size, read * v * 4.0  # difference, product, exponential, sum
    if case["kind"] == "score":
        moved += rows * (8 + 4) if case["tokens"] else 0
        moved += rows * 4 if case["entropy"] else 0
        moved += rows * 12 * case["top_k"]
        done += read * v * 2 if case["entropy"] else 0
    else:
        moved += rows * 12 * case["k"] + (rows * 4 if case["reduction"] == "none" else 4)
    if case["train"]:
        moved += rows * v * size
        done += read * v * 3.0
    return {"bytes": moved, "flops": done}


# ---- the definition in 64 bits ------------------------------------------------------------------
def exact(case, seed):
    """From the definitions with torch's own log-softmax and autograd in double precision, some rows at a time."""
    state = prepare(case, seed)
    v = case["vocab"]
    shape = state["logits"].shape[:-1]
    x = state["logits"].reshape(-1, v)
    n = x.shape[0]
    flat = {k: state[k].reshape(n, -1) for k in ("tokens", "teacher_tokens", "teacher_log_probs")
            if state.get(k) is not None}
    ups = [u.double().expand(shape).reshape(n) for u in state.get("upstream", [])]
    number = max(1, int((flat["teacher_tokens"][:, 0] >= 0).sum())) if case["kind"] == "distill" else 1
    step = max(1, (1 << 25) // v)
    parts = []
    for i in range(0, n, step):
        leaf = x[i:i + step].double().requires_grad_(case["train"])
        mine = {k: t[i:i + step] for k, t in flat.items()}
        up = [u[i:i + step] for u in ups]
        parts.append(_exact_score(case, leaf, mine, up) if case["kind"] == "score"
                     else _exact_distill(case, leaf, mine, up, number))
    out = {k: torch.cat([p[k] for p in parts]) for k in parts[0]}
    if case["kind"] == "distill" and case["reduction"] == "mean":
        out["loss"] = out["loss"].sum() / number
    out = {k: t.reshape(*shape, *t.shape[1:]) if t.dim() else t for k, t in out.items()}
    if case["kind"] == "score" and case["top_k"]:
        out["top_tokens"] = None
    return out


def _exact_score(case, leaf, mine, up):
    logp = (leaf / case["temperature"]).log_softmax(-1)
    out, total = {}, 0.0
    counts = mine["tokens"][:, 0] >= 0 if "tokens" in mine else torch.ones(len(leaf), dtype=torch.bool, device=DEVICE)
    if "tokens" in mine:
        out["log_probs"] = logp.gather(1, mine["tokens"].clamp_min(0))[:, 0].masked_fill(~counts, 0.0)
        total = total + (out["log_probs"] * up[0]).sum() if case["train"] else 0.0
    if case["entropy"]:
        out["entropy"] = -(logp.exp() * logp.masked_fill(logp == float("-inf"), 0.0)).sum(1).masked_fill(~counts, 0.0)
        total = total + (out["entropy"] * up[1]).sum() if case["train"] else 0.0
    if case["top_k"]:
        out["top_log_probs"] = logp.topk(case["top_k"], 1).values.masked_fill(~counts[:, None], float("-inf"))
    if case["train"]:
        out["grad"] = torch.autograd.grad(total, leaf)[0]
    return {k: t.detach() for k, t in out.items()}


def _exact_distill(case, leaf, mine, up, number):
    logp = (leaf / case["temperature"]).log_softmax(-1)
    tokens, given = mine["teacher_tokens"], mine["teacher_log_probs"].double()
    counts = tokens[:, 0] >= 0
    at = tokens.clamp_min(0)
    q = given if case["rest"] else (given / case["temperature"]).log_softmax(-1)
    loss = (q.exp() * (q - logp.gather(1, at))).sum(1)
    if case["rest"]:
        left = 1 - q.exp().sum(1)
        others = torch.zeros_like(logp).scatter(1, at, float("-inf"))
        short = (left.clamp_min(1e-300).log() - (logp + others).logsumexp(1)) * left
        loss = loss + torch.where(left > 0, short, 0.0)
    loss = loss.masked_fill(~counts, 0.0)
    out = {"loss": loss}
    if case["train"]:
        total = (loss * up[0]).sum() / (number if case["reduction"] == "mean" else 1)
        out["grad"] = torch.autograd.grad(total, leaf)[0]
    return {k: t.detach() for k, t in out.items()}
