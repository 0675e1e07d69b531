"""Losses over a large vocabulary, straight from the last hidden states and from a
teacher's most likely tokens.

* ``cross`` - softmax cross entropy of hidden states times the output projection, without
  the logits [rows, vocab] ever being kept, and its gradient in both factors.
* ``distill`` - the divergence of a student's logits from a teacher of which the few most
  likely tokens of each row are known (their ids and log probabilities, as scoring the
  teacher's own logits gives them), and its gradient in the logits.
* ``linear`` - the same divergence straight from the student's hidden states and output
  projection, and its gradient in both.

With p = softmax(logits / T) and q_k the teacher's probability of its k-th token id_k, a
row's divergence is sum_k q_k (log q_k - log p[id_k]) and, where the rest counts, the term
q_rest (log q_rest - log p_rest) of everything else taken as one event, q_rest = 1 -
sum_k q_k.  A teacher's token of id -1 is none (rows of fewer, down to no tokens).
"""

import math
from types import SimpleNamespace

import torch

own = False

DEVICE = "cuda"
VOCAB = 151936
# hidden size of the two configurations of bench.py
HIDDEN = {"1.7b": 2048, "8b": 4096}
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
LARGEST = 4096 * VOCAB * 2048  # rows x vocabulary x hidden of the largest listed case


def listed():
    return [
        # training: the next-token loss of two 2048-token packs
        _case("cross_pack", "cross", 4096, VOCAB, HIDDEN["1.7b"]),
        # the same of one pack of a larger model, each row with a weight of its own
        _case("cross_8b", "cross", 1900, VOCAB, HIDDEN["8b"], reduction="none"),
        # an adapter is trained below a frozen output projection: short ragged answers
        _case("cross_frozen", "cross", 777, VOCAB, HIDDEN["1.7b"], grads="hidden"),
        # scoring the tokens of an answer, no gradient
        _case("cross_score", "cross", 300, VOCAB, HIDDEN["1.7b"], grads="none", reduction="none"),
        # a decoding step's rows are scored
        _case("cross_few", "cross", 8, VOCAB, HIDDEN["1.7b"], grads="none", reduction="none"),
        # a small float32 model with a vocabulary of odd size
        _case("cross_f32", "cross", 333, 10007, 512, dtype="f32"),
        # a student's logits against a teacher's 20 most likely tokens: two packs
        _case("distill_pack", "distill", 4096, VOCAB, top=20),
        # a few positions, many alternatives, loss only: where a student stands
        _case("distill_few", "distill", 8, VOCAB, top=64, grads="none", reduction="none"),
        # a small float32 vocabulary, a soft teacher, the teacher's tokens alone
        _case("distill_f32", "distill", 700, 10007, top=5, dtype="f32", temperature=2.0, rest=False),
        # distilling into a model without keeping its logits
        _case("linear_pack", "linear", 2048, VOCAB, HIDDEN["1.7b"], top=20),
        # the same of a larger model, more alternatives, a softer student
        _case("linear_8b", "linear", 1000, VOCAB, HIDDEN["8b"], top=64, temperature=1.5, rest=False),
        # a small float32 model, a handful of rows
        _case("linear_f32", "linear", 50, 10007, 512, top=8, dtype="f32", reduction="none"),
    ]


def _case(name, kind, rows, vocab, hidden=0, top=1, dtype="bf16", grads="both", temperature=1.0,
          rest=True, reduction="mean"):
    return {"name": name, "kind": kind, "rows": rows, "vocab": vocab, "hidden": hidden, "top": top,
            "dtype": dtype, "grads": grads, "temperature": temperature, "rest": rest,
            "reduction": reduction}


def draw(rng):
    """One more case of the listed ones' ranges."""
    log_int = lambda lo, hi: int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    kind = rng.choice(["cross", "cross", "distill", "linear"])
    dtype = rng.choice(["bf16", "bf16", "bf16", "f32"])
    vocab = rng.choice([VOCAB, log_int(300, 150000)])
    hidden, most = 0, (4096 if dtype == "bf16" else 1000) * VOCAB // vocab
    if kind != "distill":
        hidden = rng.choice([2048, 4096, 64 * rng.randint(2, 64), 8 * rng.randint(8, 200)])
        # float32 products run at a sixteenth of the rate
        most = (LARGEST if dtype == "bf16" else LARGEST // 50) // (vocab * hidden)
        most = min(most, 4096 * VOCAB // vocab)
    rows = log_int(1, max(1, min(most, 8192)))
    grads = rng.choice(["both", "both", "none"] if kind == "distill"
                       else ["both", "both", "both", "hidden", "weight", "none"])
    case = _case("", kind, rows, vocab, hidden, 1 if kind == "cross" else log_int(1, min(128, vocab // 2)),
                 dtype, grads, rng.choice([1.0, 1.0, 0.7, 2.0]), rng.random() < 0.7,
                 rng.choice(["mean", "mean", "sum", "none"]))
    case.pop("name")
    return case


# ----------------------------------------------------------------------------
# Inputs (from the seed alone)
# ----------------------------------------------------------------------------

def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    rnd = lambda *shape: torch.rand(shape, generator=gen, device=DEVICE)
    normal = lambda *shape: torch.randn(shape, generator=gen, device=DEVICE)
    R, V, H, top = case["rows"], case["vocab"], case["hidden"], case["top"]
    dtype = DTYPES[case["dtype"]]
    s = SimpleNamespace(case=case)
    # a row's tokens, all different, spread over the vocabulary
    first = torch.randint(0, V, (R, 1), generator=gen, device=DEVICE)
    step = torch.randint(1, max(2, (V - 1) // top), (R, 1), generator=gen, device=DEVICE)
    ids = (first + step * torch.arange(top, device=DEVICE)) % V
    # the teacher's log probabilities, in order; most of the mass, but not all of it
    q = (2.0 * normal(R, top)).softmax(-1).sort(-1, descending=True)[0] * (0.6 + 0.39 * rnd(R, 1))
    # how far a student's logits of these tokens stand out
    lift = 4.0 + 9.0 * rnd(R, 1) + q.log().clamp(min=-6.0) + 0.5 * normal(R, top)
    if case["kind"] == "distill":
        x = (2.5 * normal(R, V)).scatter_add_(1, ids, lift)
        s.logits = x.to(dtype).requires_grad_(case["grads"] != "none")
        s.leaves = [s.logits] if case["grads"] != "none" else []
    else:
        # logits of size 2.5 from normed hidden states, and the tokens' directions in them
        s.weight = (2.5 * H ** -0.5 * normal(V, H)).to(dtype)
        h = normal(R, H)
        for k in range(top):
            h += (lift[:, k:k + 1] / 6.25) * s.weight[ids[:, k]].float()
        s.hidden = h.to(dtype)
        s.hidden.requires_grad_(case["grads"] in ("both", "hidden"))
        s.weight.requires_grad_(case["grads"] in ("both", "weight"))
        s.leaves = [x for x in (s.hidden, s.weight) if x.requires_grad]
    # some rows count for nothing, some have fewer tokens than the others
    out = rnd(R, 1) < 0.05
    if case["kind"] == "cross":
        s.targets = torch.where(out, -100, ids)[:, 0].contiguous()
    else:
        few = torch.where(rnd(R, 1) < 0.2, torch.randint(1, top + 1, (R, 1), generator=gen, device=DEVICE), top)
        gone = out | (torch.arange(top, device=DEVICE) >= few)
        s.ids = torch.where(gone, -1, ids)
        s.log_q = q.log().masked_fill(gone, -math.inf)
    s.d_loss = normal(R) if case["reduction"] == "none" else None
    return s


# ----------------------------------------------------------------------------
# One pass
# ----------------------------------------------------------------------------

def run(s):
    c = s.case
    if not own:
        return _plain(s)
    from alodlm_amd import loss
    if c["kind"] == "cross":
        out = loss.linear_cross_entropy(s.hidden, s.weight, s.targets, temperature=c["temperature"],
                                        reduction=c["reduction"])
    elif c["kind"] == "distill":
        out = loss.distillation_loss(s.logits, s.ids, s.log_q, temperature=c["temperature"],
                                     rest=c["rest"], reduction=c["reduction"])
    else:
        out = loss.linear_distillation_loss(s.hidden, s.weight, s.ids, s.log_q, temperature=c["temperature"],
                                            rest=c["rest"], reduction=c["reduction"])
    grads = torch.autograd.grad(out, s.leaves, s.d_loss) if s.leaves else ()
    return [out.detach(), *grads]


# ----------------------------------------------------------------------------
# The plain forms
# ----------------------------------------------------------------------------

def _plain(s):
    c, inv_t = s.case, 1.0 / s.case["temperature"]
    with torch.no_grad():
        if c["kind"] == "distill":
            x = s.logits.float() * inv_t
        else:
            h, w = s.hidden.float(), s.weight.float()
            x = (h @ w.T).mul_(inv_t)
        cross = c["kind"] == "cross"
        ids = s.targets[:, None] if cross else s.ids
        given = ids >= 0
        at = ids.clamp(min=0)
        q = given.float() if cross else torch.where(given, s.log_q.exp(), 0.0)
        log_q = torch.where(q > 0, q.log() if cross else s.log_q, 0.0)
        counted = given.any(-1)
        largest = x.amax(-1, keepdim=True)
        z = x.gather(1, at) - largest
        x.sub_(largest).exp_()
        total = x.sum(-1, keepdim=True)
        loss = (q * (log_q - z + total.log())).sum(-1)
        mass = q.sum(-1)
        grad = None
        if s.leaves:
            grad = x * (1.0 / total)
        if not cross and c["rest"]:
            q_rest = (1.0 - torch.where(given, s.log_q.double().exp(), 0.0).sum(-1)).clamp(min=0).float()
            q_rest = q_rest * counted
            # an added column takes what the rows' missing tokens mark
            among = torch.zeros(x.shape[0], x.shape[1] + 1, dtype=torch.bool, device=x.device)
            among.scatter_(1, torch.where(given, ids, x.shape[1]), True)
            x.masked_fill_(among[:, :-1], 0.0)
            others = x.sum(-1, keepdim=True)
            part = q_rest * (q_rest.log() - (others / total).log()[:, 0])
            loss = loss + torch.where(q_rest > 0, part, 0.0)
            mass = mass + q_rest
            if s.leaves:
                grad.mul_(mass[:, None]).sub_(x.mul_(q_rest[:, None] / others))
        elif s.leaves:
            grad.mul_(mass[:, None])
        count = counted.sum().clamp(min=1)
        if c["reduction"] == "none":
            out = loss
        else:
            out = loss.double().sum() / (count if c["reduction"] == "mean" else 1)
            out = out.float()
        if not s.leaves:
            return [out]
        grad.scatter_add_(1, at, -q)
        if c["reduction"] == "none":
            grad.mul_((s.d_loss * inv_t)[:, None])
        else:
            grad.mul_(inv_t / count if c["reduction"] == "mean" else inv_t)
        if c["kind"] == "distill":
            return [out, grad.to(s.logits.dtype)]
        grads = []
        if s.hidden.requires_grad:
            grads.append((grad @ w).to(s.hidden.dtype))
        if s.weight.requires_grad:
            grads.append((grad.T @ h).to(s.weight.dtype))
        return [out, *grads]


# ----------------------------------------------------------------------------
# What a pass cannot do without
# ----------------------------------------------------------------------------

def work(case):
    es = 2 if case["dtype"] == "bf16" else 4
    R, V, H = case["rows"], case["vocab"], case["hidden"]
    known = R * (8 if case["kind"] == "cross" else 12 * case["top"]) + 4 * R
    if case["kind"] == "distill":
        grad = case["grads"] != "none"
        return {"bytes": R * V * es * (2 if grad else 1) + known, "flops": R * V * (9 if grad else 5)}
    sides = {"both": (1, 1), "hidden": (1, 0), "weight": (0, 1), "none": (0, 0)}[case["grads"]]
    # the logits are one product, the gradient of each factor another
    return {"bytes": es * H * (R * (1 + sides[0]) + V * (1 + sides[1])) + known,
            "flops": 2 * R * V * H * (1 + sum(sides))}


# ----------------------------------------------------------------------------
# The definitions in 64 bits
# ----------------------------------------------------------------------------

def exact(case, seed):
    """From the definition, the gradients by differentiating it, some rows at a time."""
    s = prepare(case, seed)
    cross = case["kind"] == "cross"
    ids = s.targets[:, None] if cross else s.ids
    rows = (ids >= 0).any(-1)
    each = (s.d_loss.double() if case["reduction"] == "none"
            else rows.double() / (max(int(rows.sum()), 1) if case["reduction"] == "mean" else 1))
    leaves = [x.detach().double().requires_grad_() for x in s.leaves]
    losses, sums = [], [torch.zeros_like(x, requires_grad=False) for x in leaves]
    held = {id(a): b for a, b in zip(s.leaves, leaves)}
    of = lambda x: held[id(x)] if id(x) in held else x.detach().double()
    factors = [of(s.logits)] if case["kind"] == "distill" else [of(s.hidden), of(s.weight)]
    for r in range(0, case["rows"], 512):
        logits = factors[0][r:r + 512]
        if len(factors) == 2:
            logits = logits @ factors[1].T
        lp = torch.log_softmax(logits / case["temperature"], -1)
        loss = _exact_rows(lp, ids[r:r + 512], None if cross else s.log_q[r:r + 512].double(), case["rest"])
        losses.append(loss.detach())
        if leaves:
            for total, g in zip(sums, torch.autograd.grad((loss * each[r:r + 512]).sum(), leaves)):
                total += g
    loss = torch.cat(losses)
    if case["reduction"] != "none":
        loss = (loss * each).sum()
    return [loss, *sums]


def _exact_rows(lp, ids, log_q, rest):
    given = ids >= 0
    own_lp = lp.gather(1, ids.clamp(min=0))
    if log_q is None:
        return torch.where(given, -own_lp, 0.0)[:, 0]
    q = torch.where(given, log_q.exp(), 0.0)
    loss = torch.where(given, q * (torch.where(given, log_q, 0.0) - own_lp), 0.0).sum(-1)
    if not rest:
        return loss
    wide = torch.cat((lp, torch.full_like(lp[:, :1], -math.inf)), 1)
    others = wide.scatter(1, torch.where(given, ids, lp.shape[1]), -math.inf).logsumexp(-1)
    q_rest = (1.0 - q.sum(-1)).clamp(min=0)
    has = given.any(-1) & (q_rest > 0)
    safe = torch.where(has, q_rest, 1.0)
    return loss + torch.where(has, safe * (safe.log() - others), 0.0)
