"""The losses of a language model's training, as measurable cases.

A case is a dict of plain values.  ``kind`` selects the operator:

  tokens      log-probabilities of labels from logits, and their gradient
  head        the same from hidden states and the LM head's weight, without logits
  preference  a preference loss over pairs of sequences, and its gradient
  policy      a clipped policy loss with a KL term, and its gradient

Where ``own`` is true ``run`` calls the framework's operators, else the same
formulas as elementary tensor operations.
"""

from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
IGNORE = -100


def listed():
    return [
        # a serving step: the log-probabilities of the tokens that a batch of 8 users just drew
        dict(name="tokens_step", kind="tokens", B=8, S=1, V=151936, dtype="bf16", prompt=0.0, T=1.0, grad=False),
        # answers scored under a frozen reference model
        dict(name="tokens_score", kind="tokens", B=2, S=1001, V=151936, dtype="bf16", prompt=0.25, T=1.0, grad=False),
        # a fine-tuning step: the loss over a batch of logits, and their gradient
        dict(name="tokens_train", kind="tokens", B=4, S=2048, V=151936, dtype="bf16", prompt=0.25, T=1.0, grad=True),
        # an fp32 training step, a vocabulary of no round size, a temperature
        dict(name="tokens_odd_f32", kind="tokens", B=2, S=513, V=50257, dtype="f32", prompt=0.0, T=0.7, grad=True),
        # one short answer scored straight from the hidden states
        dict(name="head_few", kind="head", B=1, S=33, V=151936, H=1024, prompt=0.0, T=1.0, grad=False),
        # the model's share of a small preference step: four sequences, prompts left out
        dict(name="head_train", kind="head", B=4, S=1023, V=151936, H=1024, prompt=0.25, T=1.0, grad=True),
        # a long batch at a wider model
        dict(name="head_large", kind="head", B=4, S=2048, V=151936, H=2048, prompt=0.0, T=1.0, grad=True),
        # sizes that fill no tile
        dict(name="head_odd", kind="head", B=3, S=301, V=50257, H=520, prompt=0.1, T=0.9, grad=True),
        # the loss of a small preference batch
        dict(name="preference_small", kind="preference", B=4, S=256, beta=0.1, smoothing=0.0, form="sigmoid"),
        # many long pairs, accumulated over a cluster's step
        dict(name="preference_large", kind="preference", B=256, S=4096, beta=0.1, smoothing=0.1, form="sigmoid"),
        # the loss of one prompt's group of answers
        dict(name="policy_small", kind="policy", B=8, S=512, low=0.2, high=0.2, kl=0.0, form="sequence"),
        # a whole rollout batch of long answers
        dict(name="policy_large", kind="policy", B=512, S=8192, low=0.2, high=0.28, kl=0.04, form="token"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["tokens", "head", "preference", "policy"])
    if kind == "tokens":
        V = _log_int(rng, 1000, 160000)
        N = _log_int(rng, 1, min(16384, int(1.2e9) // V))
        B = rng.choice([1, 1, 2, 4])
        return dict(kind=kind, B=B, S=max(1, N // B), V=V, dtype=rng.choice(["bf16", "bf16", "f32"]),
                    prompt=rng.choice([0.0, 0.25, 0.5]), T=rng.choice([1.0, 0.8, 1.5]), grad=rng.random() < 0.7)
    if kind == "head":
        V = _log_int(rng, 1000, 152000)
        H = 8 * _log_int(rng, 8, 512)
        N = _log_int(rng, 1, min(8192, int(2.5e12) // (V * H)))
        B = rng.choice([1, 1, 2, 4])
        return dict(kind=kind, B=B, S=max(1, N // B), V=V, H=H, prompt=rng.choice([0.0, 0.25, 0.5]),
                    T=rng.choice([1.0, 0.8, 1.5]), grad=rng.random() < 0.7)
    S = _log_int(rng, 16, 16384)
    if kind == "preference":
        return dict(kind=kind, B=_log_int(rng, 1, min(1024, (1 << 21) // S)), S=S, beta=rng.choice([0.05, 0.1, 0.5]),
                    smoothing=rng.choice([0.0, 0.1]), form=rng.choice(["sigmoid", "sigmoid", "hinge", "ipo"]))
    return dict(kind=kind, B=_log_int(rng, 1, min(1024, (1 << 22) // S)), S=S, low=0.2, high=rng.choice([0.2, 0.28]),
                kl=rng.choice([0.0, 0.04]), form=rng.choice(["token", "sequence"]))


def _labels(case, g):
    """Token ids of which the frequent ones recur, the first share of each sequence ignored."""
    B, S, V = case["B"], case["S"], case["V"]
    u = torch.rand(B, S, generator=g, device=DEV, dtype=torch.float64)
    ids = (torch.exp(u * math.log(V)).long() - 1).clamp_(0, V - 1)
    full = ids.clone()
    ids[:, :int(case["prompt"] * S)] = IGNORE
    return ids, full


def _kept(case, g):
    """The tokens of answers of differing length."""
    B, S = case["B"], case["S"]
    lens = torch.randint(max(1, S // 4), S + 1, (B, 1), generator=g, device=DEV)
    return torch.arange(S, device=DEV) < lens


def _log_probs(B, S, g):
    return -2 * torch.randn(B, S, generator=g, device=DEV).abs()


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    s = dict(case=case)
    if case["kind"] in ("tokens", "head"):
        B, S, V = case["B"], case["S"], case["V"]
        labels, full = _labels(case, g)
        s["labels"] = labels
        s["dy"] = torch.randn(B, S, generator=g, device=DEV) / (B * S)
        if case["kind"] == "tokens":
            dt = DTYPES[case["dtype"]]
            x = torch.randn(B, S, V, generator=g, device=DEV, dtype=dt).mul_(2)
            # a trained model gives the label far more than its share
            x.scatter_add_(2, full[..., None], torch.full((B, S, 1), 10.0, device=DEV, dtype=dt))
            s["logits"] = x.requires_grad_(case["grad"])
        else:
            H = case["H"]
            w = torch.randn(V, H, generator=g, device=DEV).mul_(0.02).bfloat16()
            h = torch.randn(B, S, H, generator=g, device=DEV).mul_(2 / (0.02 * math.sqrt(H)))
            h += w[full].float() * (10 / (0.02 ** 2 * H))
            s["weight"] = w.requires_grad_(case["grad"])
            s["hidden"] = h.bfloat16().requires_grad_(case["grad"])
    elif case["kind"] == "preference":
        B, S = case["B"], case["S"]
        for side in ("chosen", "rejected"):
            lp = _log_probs(B, S, g)
            s["ref_" + side] = lp
            s[side] = (lp + 0.1 * torch.randn(B, S, generator=g, device=DEV)).requires_grad_()
            s[side + "_mask"] = _kept(case, g)
    else:
        B, S = case["B"], case["S"]
        lp = _log_probs(B, S, g)
        s["old"] = lp + 0.15 * torch.randn(B, S, generator=g, device=DEV)
        s["ref"] = lp + 0.2 * torch.randn(B, S, generator=g, device=DEV) if case["kl"] else None
        s["lp"] = lp.requires_grad_()
        s["adv"] = torch.randn(B, generator=g, device=DEV)
        s["mask"] = _kept(case, g)
    return s


# ---------------------------------------------------------------- the framework's operators

def _own(s):
    import nano_qwen_amd as nq
    c = s["case"]
    if c["kind"] == "tokens":
        lp = nq.token_logprobs(s["logits"], s["labels"], temperature=c["T"])
        return [lp, *torch.autograd.grad(lp, s["logits"], s["dy"])] if c["grad"] else [lp]
    if c["kind"] == "head":
        lp = nq.linear_logprobs(s["hidden"], s["weight"], s["labels"], temperature=c["T"])
        return [lp, *torch.autograd.grad(lp, (s["hidden"], s["weight"]), s["dy"])] if c["grad"] else [lp]
    if c["kind"] == "preference":
        loss, rc, rr = nq.preference_loss(s["chosen"], s["rejected"], s["ref_chosen"], s["ref_rejected"],
                                          chosen_mask=s["chosen_mask"], rejected_mask=s["rejected_mask"],
                                          beta=c["beta"], kind=c["form"],
                                          label_smoothing=c["smoothing"] if c["form"] == "sigmoid" else 0.0)
        return [loss, rc, rr, *torch.autograd.grad(loss, (s["chosen"], s["rejected"]))]
    loss, kl, clipped = nq.policy_loss(s["lp"], s["old"], s["adv"], ref_logprobs=s["ref"], mask=s["mask"],
                                       clip_low=c["low"], clip_high=c["high"], kl_coef=c["kl"], reduction=c["form"])
    return [loss, kl, clipped, *torch.autograd.grad(loss, s["lp"])]


# ---------------------------------------------------------------- the plain forms

def _log_softmax_parts(z, labels):
    """(log-probability of each label, the softmax), of fp32 logits that this may overwrite."""
    m = z.amax(-1, keepdim=True)
    p = z.sub(m).exp_()
    total = p.sum(-1, keepdim=True)
    at = labels.clamp(min=0)[..., None]
    lp = z.gather(-1, at) - m - total.log()
    kept = labels != IGNORE
    return torch.where(kept, lp[..., 0], 0.0), p.div_(total)


def _logits_gradient(p, labels, dy, T):
    """dy (1[v = label] - p) / T, zero in ignored rows; in the memory of p."""
    dy = torch.where(labels != IGNORE, dy, 0.0)[..., None] / T
    p.mul_(-dy)
    return p.scatter_add_(-1, labels.clamp(min=0)[..., None], dy)


def _plain(s):
    c = s["case"]
    if c["kind"] == "tokens":
        lp, p = _log_softmax_parts(s["logits"].detach().float() / c["T"], s["labels"])
        if not c["grad"]:
            return [lp]
        return [lp, _logits_gradient(p, s["labels"], s["dy"], c["T"]).to(s["logits"].dtype)]
    if c["kind"] == "head":
        h, w = s["hidden"].detach().float(), s["weight"].detach().float()
        lp, p = _log_softmax_parts(h @ w.t() / c["T"], s["labels"])
        if not c["grad"]:
            return [lp]
        dz = _logits_gradient(p, s["labels"], s["dy"], c["T"])
        V, H = w.shape
        return [lp, (dz @ w).bfloat16(), (dz.view(-1, V).t() @ h.view(-1, H)).bfloat16()]
    if c["kind"] == "preference":
        # sums of many tokens whose difference is small: in 64 bits
        mc, mr = s["chosen_mask"], s["rejected_mask"]
        dc = torch.where(mc, s["chosen"].detach().double() - s["ref_chosen"], 0.0).sum(-1)
        dr = torch.where(mr, s["rejected"].detach().double() - s["ref_rejected"], 0.0).sum(-1)
        beta, e, B = c["beta"], c["smoothing"], c["B"]
        h = beta * (dc - dr)
        if c["form"] == "sigmoid":
            soft = torch.log1p(torch.exp(-h.abs())) + (-h).clamp(min=0)  # -log sigmoid(h)
            loss = (1 - e) * soft + e * (soft + h)
            slope = beta * (e - 1 / (1 + torch.exp(h)))
        elif c["form"] == "hinge":
            loss, slope = (1 - h).clamp(min=0), torch.where(h < 1, -beta, 0.0)
        else:
            d = dc - dr - 1 / (2 * beta)
            loss, slope = d * d, 2 * d
        slope = (slope / B).float()[:, None]
        return [loss.mean().float(), (beta * dc).float(), (beta * dr).float(), torch.where(mc, slope, 0.0),
                torch.where(mr, -slope, 0.0)]
    mask, lp, adv = s["mask"], s["lp"].detach(), s["adv"][:, None]
    # the log-ratio decides which side of a border a token is on: in 64 bits
    d = lp.double() - s["old"]
    r = torch.exp(d).float()
    over = (adv > 0) & (d > math.log1p(c["high"]))
    under = (adv < 0) & (d < math.log1p(-c["low"]))
    term = -torch.where(over, (1 + c["high"]) * adv, torch.where(under, (1 - c["low"]) * adv, r * adv))
    grad = torch.where(over | under, 0.0, -r * adv)
    if s["ref"] is not None:
        q = s["ref"].double() - lp  # e^q - q - 1 of a small q: in 64 bits
        kl = torch.exp(q) - q - 1
        term = term + c["kl"] * kl
        grad = grad + c["kl"] * (1 - torch.exp(q)).float()
    else:
        kl = torch.zeros_like(d)
    n = mask.sum()
    share = 1 / n if c["form"] == "token" else (1 / mask.sum(-1, keepdim=True).clamp(min=1)) / c["B"]
    kept = torch.where(mask, term.double() * share, 0.0)
    return [kept.sum().float(), (torch.where(mask, kl, 0.0).sum() / n).float(),
            ((over | under) & mask).sum().div(n), torch.where(mask, grad * share, 0.0)]


def run(state):
    if own:
        return _own(state)
    with torch.no_grad():
        return _plain(state)


def work(case):
    B, S = case["B"], case["S"]
    N = B * S
    if case["kind"] in ("tokens", "head"):
        kept = B * (S - int(case["prompt"] * S))
        V = case["V"]
        if case["kind"] == "tokens":
            e = 2 if case["dtype"] == "bf16" else 4
            return dict(bytes=kept * V * e + (N * V * e + 4 * N if case["grad"] else 0) + 12 * N,
                        flops=kept * V * (8 if case["grad"] else 4))
        H = case["H"]
        io = 2 * (kept * H + V * H) + 12 * N
        return dict(bytes=io + (2 * (N * H + V * H) + 4 * N if case["grad"] else 0),
                    flops=kept * V * H * (6 if case["grad"] else 2))
    if case["kind"] == "preference":
        return dict(bytes=N * (4 * 4 + 2 + 2 * 4) + 8 * B, flops=6 * N)
    return dict(bytes=N * (4 * (3 if case["kl"] else 2) + 1 + 4) + 4 * B, flops=(30 if case["kl"] else 15) * N)


# ---------------------------------------------------------------- the definitions in 64 bits

def _exact_tokens(case, s):
    x, labels = s["logits"].detach(), s["labels"]
    lps, grads = [], []
    for b in range(case["B"]):
        z = torch.log_softmax(x[b].double() / case["T"], -1)
        idx = labels[b].clamp(min=0)[:, None]
        keep = (labels[b] != IGNORE).double()
        lps.append(z.gather(1, idx)[:, 0] * keep)
        if case["grad"]:
            c = s["dy"][b].double() * keep / case["T"]
            grads.append(z.exp_().neg_().scatter_add_(1, idx, torch.ones_like(idx, dtype=torch.float64)).mul_(c[:, None]))
    return [torch.stack(lps), torch.stack(grads)] if case["grad"] else [torch.stack(lps)]


def _exact_head(case, s):
    H = case["H"]
    h, w = s["hidden"].detach().double().view(-1, H), s["weight"].detach().double()
    labels, dy = s["labels"].view(-1), s["dy"].view(-1).double()
    lp = torch.zeros(len(labels), dtype=torch.float64, device=DEV)
    dh, dw = torch.zeros_like(h), torch.zeros_like(w)
    at = torch.nonzero(labels != IGNORE)[:, 0]
    for rows in at.split(2048):
        z = torch.log_softmax(h[rows] @ w.t() / case["T"], -1)
        idx = labels[rows][:, None]
        lp[rows] = z.gather(1, idx)[:, 0]
        if case["grad"]:
            dz = z.exp_().neg_().scatter_add_(1, idx, torch.ones_like(idx, dtype=torch.float64))
            dz.mul_(dy[rows][:, None] / case["T"])
            dh[rows] = dz @ w
            dw.addmm_(dz.t(), h[rows])
    shape = s["labels"].shape
    return [lp.view(shape), dh.view(*shape, H), dw] if case["grad"] else [lp.view(shape)]


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "tokens":
        return _exact_tokens(case, s)
    if case["kind"] == "head":
        return _exact_head(case, s)
    with torch.enable_grad():
        if case["kind"] == "preference":
            c, r = (s[k].detach().double().requires_grad_() for k in ("chosen", "rejected"))
            mc, mr = s["chosen_mask"].double(), s["rejected_mask"].double()
            wc = ((c - s["ref_chosen"].double()) * mc).sum(1)
            wr = ((r - s["ref_rejected"].double()) * mr).sum(1)
            h = case["beta"] * (wc - wr)
            if case["form"] == "sigmoid":
                ls = torch.nn.functional.logsigmoid
                each = -(1 - case["smoothing"]) * ls(h) - case["smoothing"] * ls(-h)
            elif case["form"] == "hinge":
                each = torch.relu(1 - h)
            else:
                each = (wc - wr - 0.5 / case["beta"]) ** 2
            loss = each.mean()
            return [loss.detach(), case["beta"] * wc.detach(), case["beta"] * wr.detach(), *torch.autograd.grad(loss, (c, r))]
        lp = s["lp"].detach().double().requires_grad_()
        m = s["mask"].double()
        ratio, adv = torch.exp(lp - s["old"].double()), s["adv"].double()[:, None]
        bounded = ratio.clamp(1 - case["low"], 1 + case["high"])
        each = -torch.minimum(ratio * adv, bounded * adv)
        cut = (bounded * adv < ratio * adv).double()
        kl = torch.zeros_like(lp)
        if s["ref"] is not None:
            q = s["ref"].double() - lp
            kl = torch.expm1(q) - q
        each = each + case["kl"] * kl
        if case["form"] == "token":
            loss = (each * m).sum() / m.sum()
        else:
            loss = ((each * m).sum(1) / m.sum(1).clamp(min=1)).mean()
        (grad,) = torch.autograd.grad(loss, lp)
        return [loss.detach(), ((kl * m).sum() / m.sum()).detach(), (cut * m).sum() / m.sum(), grad]
