"""Log-probabilities of labels, the preference loss and the policy loss on the kernels,
against the same formulas in 64 bits.

Tolerances are sums of roundings: u = 2^-24 for each fp32 operation on a value, half a
step of the output's type for the result.
"""

import math

import pytest
import torch

import nano_qwen_amd as nq
from tests.helpers import randn, say

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, F32 = torch.bfloat16, torch.float32
U = 2.0 ** -24


def half_step(dt):
    return torch.finfo(dt).eps / 2


def within(got, want, tol, what):
    got = got.detach().double().cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{what}: NaN in other places"
    assert torch.equal(torch.isinf(got), torch.isinf(want)), f"{what}: infinities in other places"
    ok = torch.isfinite(want)
    err = (got - want).abs()
    tol = tol.expand_as(err) if isinstance(tol, torch.Tensor) else torch.full_like(err, tol)
    bad = (err > tol) & ok
    assert not bad.any(), (what, int(bad.sum()), float(err[ok].max()), float((err / tol)[bad].max()))


# ---------------------------------------------------------------- token_logprobs

def token_reference(x, labels, dy, T, ignore=-100):
    """(logprobs, dlogits, their tolerances before the output's own rounding), in 64 bits."""
    V = x.shape[-1]
    z = x.double() / T
    logp = torch.log_softmax(z, -1)  # subtracts the maximum first: exact also at the types' ends
    p = torch.exp(logp)
    at = labels.clamp(0, V - 1)[..., None].long()
    keep = labels != ignore
    bad = keep & ((labels < 0) | (labels >= V))
    lp = logp.gather(-1, at)[..., 0]
    lp = torch.where(bad, torch.nan, torch.where(keep, lp, 0.0))
    g = torch.where(keep, dy.double(), 0.0) / T
    g = torch.where(bad, torch.nan, g)[..., None]
    dz = torch.where(keep[..., None], -p * g, 0.0)
    dz = dz.scatter_add(-1, at, g)
    # exponents (x - m) c carry |z - m| u each, a thread adds V / 256 terms one after the
    # other, waves and workgroups join in some 16 steps of 4 operations
    fin = torch.where(torch.isfinite(z), z, torch.nan)
    span = torch.nan_to_num(torch.nan_to_num(fin, -math.inf).amax(-1) - torch.nan_to_num(fin, math.inf).amin(-1), 0, 0, 0)
    steps = (span * 2 + V / 256 + 80) * U
    tol_lp = steps + 4 * U * lp.abs().nan_to_num(0, 0, 0)
    tol_dz = g.abs().nan_to_num(0) * (p.nan_to_num(0) * steps[..., None] + 4 * U) + 1e-37
    return lp, dz, tol_lp, tol_dz


def run_token(x, labels, dy, T=1.0, **kw):
    xd = x.to(DEV).requires_grad_()
    lp = nq.token_logprobs(xd, labels.to(DEV), temperature=T, **kw)
    (dx,) = torch.autograd.grad(lp, xd, dy.to(DEV))
    return lp, dx


def check_token(x, labels, dy, T=1.0, what="", **kw):
    lp, dx = run_token(x, labels, dy, T, **kw)
    assert lp.dtype == F32 and lp.shape == labels.shape and dx.dtype == x.dtype and dx.shape == x.shape
    want, dwant, tol, dtol = token_reference(x, labels, dy, T, kw.get("ignore_index", -100))
    within(lp, want, tol, f"{what} logprobs")
    within(dx, dwant, dtol + half_step(x.dtype) * dwant.abs().nan_to_num(0), f"{what} dlogits")
    with torch.no_grad():
        assert torch.equal(nq.token_logprobs(x.to(DEV), labels.to(DEV), temperature=T, **kw).nan_to_num(9), lp.nan_to_num(9))


# rows of less than a vector, of whole vectors and not, of one and of many slices; one row to
# more than the split is for
@pytest.mark.parametrize("rows,V", [(1, 1), (1, 8), (3, 7), (2, 9), (5, 1000), (4, 8192), (3, 8200), (2, 50257), (1, 151936),
                                    (2100, 133), (260, 16391), (6, 2055), (6, 2056), (2049, 4100), (2048, 8199), (2048, 8200)])
@pytest.mark.parametrize("dt", [BF, F32])
def test_token_logprobs(rows, V, dt):
    say(f"token_logprobs {rows}x{V} {dt}")
    x = randn(rows, V, seed=7, dtype=dt, scale=3)
    labels = torch.randint(0, V, (rows,), generator=torch.Generator().manual_seed(8))
    labels[rows // 2] = V - 1
    if rows > 3:
        labels[::3] = -100
    check_token(x, labels, randn(rows, seed=9), T=0.7 if V % 2 else 1.0, what=f"{rows}x{V}")


@pytest.mark.parametrize("dt", [BF, F32])
@pytest.mark.parametrize("rows", [3, 3000])
def test_token_logprobs_of_special_rows(rows, dt):
    """Masked vocabularies, rows of -inf, infinities, NaN, labels outside, ignored rows of NaN."""
    say(f"token_logprobs special rows {rows} {dt}")
    V = 4099
    x = randn(12, V, seed=17, dtype=dt)
    inf = float("inf")
    x[0, 5:] = -inf                      # five tokens left, the label among them
    x[1, :4098] = -inf                   # only the last element, in the tail
    x[2] = -inf
    x[3, 77] = inf
    x[4, 4098] = inf
    x[5, 4098] = float("nan")
    x[6, 0] = float("nan")
    x[7, :4000] = -inf                   # the first threads and slices see nothing but -inf
    x[8] = torch.finfo(dt).min           # the type's lowest value everywhere
    x[9, ::2] = torch.finfo(dt).min      # and as a mask
    x[9, 1] = torch.finfo(dt).max / 2
    labels = torch.tensor([2, 4098, 3, 77, 0, 1, 0, 4050, 9, 1, 4099, -1])
    x, labels = x.repeat(rows // 3 + 1, 1)[:max(rows, 12)], labels.repeat(rows // 3 + 1)[:max(rows, 12)]
    check_token(x, labels, 1 + randn(len(x), seed=18).abs(), what="special")
    # ignored rows are not read and get zeros, whatever they hold
    lp, dx = run_token(x, torch.full_like(labels, -100), torch.full((len(x),), float("nan")))
    assert not lp.any() and not dx.any()
    # a label of -inf among finite ones: -inf, and a finite gradient
    y = randn(rows, V, seed=19, dtype=dt)
    y[:, 3] = -inf
    check_token(y, torch.full((rows,), 3), torch.ones(rows), what="label of -inf")


def test_token_logprobs_shapes_strides_types():
    say("token_logprobs shapes and strides")
    big = randn(3, 6, 5, 72, seed=27)
    lab = torch.randint(0, 64, (3, 6, 5), generator=torch.Generator().manual_seed(28))
    dy = randn(3, 6, 5, seed=29)
    views = {
        "sliced": (big[..., 3:67], lab, dy),
        "short sequences": (big[0, :, :4, :64], lab[0, :, :4], dy[0, :, :4]),
        "four axes that do not fold": (big[:, ::2, 1:, :64], lab[:, ::2, 1:], dy[:, ::2, 1:]),
        "transposed": (big[0, 0].t()[:64, :][:, :5].t(), lab[0, 0], dy[0, 0]),
        "one row": (big[0, 0, 0, :64], lab[0, 0, 0], dy[0, 0, 0]),
        "expanded": (big[0, :1, 0, :64].expand(6, 64), lab[0, :, 0], dy[0, :, 0]),
        "other ignore_index": (big[0, 0, :, :64], lab[0, 0], dy[0, 0]),
    }
    for name, (x, y, g) in views.items():
        dev = torch.empty_strided(x.shape, x.stride(), device=DEV) if name != "expanded" else x[:1].to(DEV).expand(x.shape)
        if name != "expanded":
            dev.copy_(x)
        dev = dev.detach().requires_grad_()
        kw = dict(ignore_index=int(y.flatten()[0])) if name == "other ignore_index" else {}
        for labels in (y, y.to(torch.int32)):
            lp = nq.token_logprobs(dev, labels.to(DEV), **kw)
            (dx,) = torch.autograd.grad(lp, dev, g.to(DEV))
            want, dwant, tol, dtol = token_reference(x, y, g, 1.0, kw.get("ignore_index", -100))
            within(lp, want, tol, name)
            within(dx, dwant, dtol + half_step(F32) * dwant.abs(), name)
    # a gradient broadcast by a sum, and rows at a misaligned base address
    for dt in (BF, F32):
        x = randn(4, 66, seed=30, dtype=dt)
        y = torch.tensor([0, 64, 3, -100])
        dev = x.to(DEV)
        leaf = dev[:, 1:].detach().requires_grad_()
        (dx,) = torch.autograd.grad(nq.token_logprobs(leaf, y.to(DEV)).sum(), leaf)
        _, dwant, _, dtol = token_reference(x[:, 1:], y, torch.ones(4), 1.0)
        within(dx, dwant, dtol + half_step(dt) * dwant.abs(), "misaligned")
    for shape in ((0, 7), (2, 0, 7)):
        x = torch.zeros(shape, device=DEV, requires_grad=True)
        lp = nq.token_logprobs(x, torch.zeros(shape[:-1], dtype=torch.long, device=DEV))
        assert lp.shape == shape[:-1] and torch.autograd.grad(lp.sum(), x)[0].shape == shape


def test_token_logprobs_past_32_bits():
    """Rows whose offsets pass 2^31 elements and 2^32 bytes."""
    say("token_logprobs past 2^31 elements")
    V, S = 150000, 15000
    x = torch.zeros(S, V, dtype=BF, device=DEV)
    assert x.numel() > 2 ** 31
    rows = torch.tensor([0, 14316, 14317, 14999])
    part = randn(4, V, seed=31, dtype=BF)
    x[rows.to(DEV)] = part.to(DEV)
    labels = torch.full((S,), -100)
    labels[rows] = torch.tensor([0, 1, V - 1, 7])
    dy = randn(S, seed=32)
    x.requires_grad_()
    lp = nq.token_logprobs(x, labels.to(DEV))
    (dx,) = torch.autograd.grad(lp, x, dy.to(DEV))
    want, dwant, tol, dtol = token_reference(part, labels[rows], dy[rows], 1.0)
    within(lp[rows.to(DEV)], want, tol, "far rows")
    within(dx[rows.to(DEV)], dwant, dtol + half_step(BF) * dwant.abs(), "far rows' gradient")
    dx[rows.to(DEV)] = 0
    assert not dx.any()


def test_token_logprobs_differences():
    """The gradient against central differences of the operator itself."""
    say("token_logprobs differences")
    x, v = randn(6, 37, seed=33).to(DEV), randn(6, 37, seed=34).to(DEV)
    y, g = torch.arange(6, device=DEV) * 5, randn(6, seed=35).to(DEV)

    def f(t):
        return (nq.token_logprobs(x + t * v, y, temperature=1.3) * g).sum(dtype=torch.float64)
    xg = x.clone().requires_grad_()
    (dx,) = torch.autograd.grad(nq.token_logprobs(xg, y, temperature=1.3), xg, g)
    h = 2.0 ** -6
    diff = float((f(h) - f(-h)) / (2 * h))
    # third derivative along v under 6 |g| |v/T|^3 per row, each value off by some 100 u
    bound = float(6 * g.abs().sum() * (v.abs().max() / 1.3) ** 3) * h * h / 6 + 2 * 100 * U * float(g.abs().sum()) / (2 * h)
    assert abs(diff - float((dx * v).double().sum())) <= bound


def test_token_logprobs_refusals():
    x, y = torch.zeros(4, 9, device=DEV), torch.zeros(4, dtype=torch.long, device=DEV)
    with pytest.raises(RuntimeError, match="HIP device"):
        nq.token_logprobs(x.cpu(), y)
    with pytest.raises(RuntimeError, match="HIP device"):
        nq.token_logprobs(x, y.cpu())
    with pytest.raises(TypeError, match="unsupported dtype"):
        nq.token_logprobs(x.half(), y)
    with pytest.raises(TypeError, match="labels"):
        nq.token_logprobs(x, y.float())
    with pytest.raises(ValueError, match="one label per row"):
        nq.token_logprobs(x, y[:3])
    with pytest.raises(ValueError, match="last axis"):
        nq.token_logprobs(x[:, :0], y)
    for t in (0.0, -1.0, float("inf"), float("nan")):
        with pytest.raises(ValueError, match="temperature"):
            nq.token_logprobs(x, y, temperature=t)
    with pytest.raises(RuntimeError):
        xg = x.clone().requires_grad_()
        (d,) = torch.autograd.grad(nq.token_logprobs(xg, y).sum(), xg, create_graph=True)
        torch.autograd.grad(d.sum(), xg)


# ---------------------------------------------------------------- preference_loss

def preference_reference(c, r, rc, rr, mc, mr, kind, beta, e, average):
    c, r = (t.double().requires_grad_() for t in (c, r))
    d = []
    for lp, ref, m in ((c, rc, mc), (r, rr, mr)):
        t = lp - (0 if ref is None else ref.double())
        m = torch.ones_like(t, dtype=torch.bool) if m is None else m
        t = torch.where(m, t, 0.0).reshape(len(lp), -1).sum(1)
        d.append(t / m.reshape(len(lp), -1).sum(1).clamp(min=1) if average else t)
    h = beta * (d[0] - d[1])
    if kind == "sigmoid":
        ls = torch.nn.functional.logsigmoid
        loss = -(1 - e) * ls(h) - e * ls(-h)
    elif kind == "hinge":
        loss = torch.relu(1 - h)
    else:
        loss = (d[0] - d[1] - 1 / (2 * beta)) ** 2
    loss = loss.mean()
    return [t.detach() for t in (loss, beta * d[0], beta * d[1], *torch.autograd.grad(loss, (c, r)))]


def ragged(B, S, seed):
    g = torch.Generator().manual_seed(seed)
    m = torch.arange(S) < torch.randint(0, S + 1, (B, 1), generator=g)
    m[B // 2] = False  # a sequence with nothing left
    return m


@pytest.mark.parametrize("B,Sc,Sr", [(1, 1, 1), (3, 40, 17), (16, 1024, 5), (17, 9, 33), (4, 1025, 300), (300, 70, 64),
                                     (2, 0, 3)])
@pytest.mark.parametrize("kind,e", [("sigmoid", 0.0), ("sigmoid", 0.2), ("hinge", 0.0), ("ipo", 0.0)])
@pytest.mark.parametrize("average", [False, True])
def test_preference_loss(B, Sc, Sr, kind, e, average):
    say(f"preference_loss {B} {Sc} {Sr} {kind} {e} {average}")
    c, r, rc, rr = (-randn(B, S, seed=40 + i).abs() for i, S in enumerate((Sc, Sr, Sc, Sr)))
    mc, mr = ragged(B, Sc, 44), ragged(B, Sr, 45)
    for masks, refs in (((mc, mr), (rc, rr)), ((None, mr), (None, rr)), ((mc, None), (rc, None))):
        want = preference_reference(c, r, *refs, *masks, kind, 0.3, e, average)
        # what a masked token holds has no effect
        ins = [t.clone() for t in (c, r)] + [None if t is None else t.clone() for t in refs]
        for t, m in zip(ins, masks * 2):
            if t is not None and m is not None:
                t[~m] = float("nan")
        cd, rd, rcd, rrd = (None if t is None else t.to(DEV) for t in ins)
        cd.requires_grad_(), rd.requires_grad_()
        loss, wc, wr = nq.preference_loss(cd, rd, rcd, rrd, chosen_mask=None if masks[0] is None else masks[0].to(DEV),
                                          rejected_mask=None if masks[1] is None else masks[1].to(DEV), beta=0.3,
                                          label_smoothing=e, kind=kind, average=average)
        grads = torch.autograd.grad(2.5 * loss, (cd, rd))
        assert loss.shape == () and wc.shape == wr.shape == (B,) and not wc.requires_grad
        # sums in 64 bits; results rounded once, gradients twice more by the factor
        for name, got, ref, k in zip(("loss", "wc", "wr", "dc", "dr"), (loss, wc, wr, *grads), want, (1, 1, 1, 2.5, 2.5)):
            within(got, k * ref, 4 * U * (k * ref).abs() + 1e-12, name)


def test_preference_loss_far_margins_and_rows():
    """Margins that overflow an exponential; sequences' sums given as such; strided rows; bf16; gradients of broadcasts."""
    say("preference_loss margins, strides")
    c = torch.tensor([1e5, -1e5, 0.0, 3000.0, -800.0])
    r = torch.zeros(5)
    for kind in ("sigmoid", "hinge", "ipo"):
        want = preference_reference(c[:, None], r[:, None], None, None, None, None, kind, 1.0, 0.0, False)
        cd, rd = c.to(DEV).requires_grad_(), r.to(DEV).requires_grad_()
        loss, *_ = nq.preference_loss(cd, rd, beta=1.0, kind=kind)
        grads = torch.autograd.grad(loss, (cd, rd))
        within(loss, want[0], 4 * U * want[0].abs(), kind)
        for g, w in zip(grads, want[3:]):
            within(g, w[:, 0], 4 * U * w[:, 0].abs() + 1e-40, kind)
    both = -randn(8, 30, seed=46).abs()      # one forward over both sides, the views of it as they are
    mask = ragged(8, 30, 47)
    leaf = both.to(DEV).requires_grad_()
    m = mask.to(DEV)
    ref = -randn(30, 8, seed=48).abs()
    loss, *_ = nq.preference_loss(leaf[::2, 1:], leaf[1::2, 1:], ref.to(DEV).t()[:4, 1:], ref.to(DEV).t()[4:, 1:],
                                  chosen_mask=m[::2, 1:], rejected_mask=m[1::2, 1:].int())
    (g,) = torch.autograd.grad(loss, leaf)
    want = preference_reference(both[::2, 1:], both[1::2, 1:], ref.t()[:4, 1:], ref.t()[4:, 1:], mask[::2, 1:],
                                mask[1::2, 1:], "sigmoid", 0.1, 0.0, False)
    within(loss, want[0], 4 * U * want[0].abs(), "strided")
    full = torch.zeros(8, 30, dtype=torch.float64)
    full[::2, 1:], full[1::2, 1:] = want[3], want[4]
    within(g, full, 4 * U * full.abs(), "strided gradient")
    # bf16 log-probabilities, one side without a gradient, an expanded side
    one = both[:1].to(BF)
    leaf = one.to(DEV).requires_grad_()
    loss, *_ = nq.preference_loss(leaf.expand(4, 30), both[:4].to(DEV))
    (g,) = torch.autograd.grad(loss, leaf)
    want = preference_reference(one.float().expand(4, 30), both[:4], None, None, None, None, "sigmoid", 0.1, 0.0, False)
    within(loss, want[0], 4 * U * want[0].abs(), "expanded")
    # torch sums the four rows' gradients, each rounded to bf16
    within(g, want[3].sum(0, keepdim=True), 4 * 2.0 ** -8 * want[3].abs().sum(0, keepdim=True), "expanded gradient")


@pytest.mark.parametrize("kind", ["sigmoid", "hinge", "ipo"])
def test_preference_loss_differences(kind):
    """The gradients against central differences of the operator itself."""
    say(f"preference_loss differences {kind}")
    c, r, v, w = (0.3 * randn(5, 6, seed=49 + i).to(DEV) for i in range(4))

    def f(t):
        return nq.preference_loss(c + t * v, r + t * w, kind=kind, beta=0.5)[0]
    cg, rg = c.clone().requires_grad_(), r.clone().requires_grad_()
    dc, dr = torch.autograd.grad(nq.preference_loss(cg, rg, kind=kind, beta=0.5)[0], (cg, rg))
    h = 2.0 ** -7
    diff = float(f(h).double() - f(-h).double()) / (2 * h)
    # along the step a pair's margin moves by s t: third derivatives under (beta s)^3 / 8 (sigmoid), none (the others,
    # with no hinge within h of a corner); the ends off by u of the loss and of their rounded inputs
    s = float((v.abs().sum(1) + w.abs().sum(1)).max())
    size = float(f(0.0).abs()) + s + float((c.abs().sum(1) + r.abs().sum(1)).max()) * (1 + 2 * s)
    bound = (0.5 * s) ** 3 * h * h / 6 + 4 * U * size / h
    margin = 0.5 * (c.double().sum(1) - r.double().sum(1))
    assert kind != "hinge" or float((margin - 1).abs().min()) > 0.5 * s * h
    assert abs(diff - float((dc * v).double().sum() + (dr * w).double().sum())) <= bound


def test_policy_loss_differences():
    """The gradient against central differences of the operator itself, no token within a step of a border."""
    say("policy_loss differences")
    lp, v = -randn(4, 9, seed=61).abs(), randn(4, 9, seed=62)
    d = 0.5 * randn(4, 9, seed=63)
    h = 2.0 ** -8
    for border in (math.log1p(0.2), math.log1p(-0.2)):
        near = (d - border).abs() < 2 * h * v.abs().max()
        d = torch.where(near, d + 4 * h * v.abs().max(), d)
    for border in (math.log1p(0.2), math.log1p(-0.2)):
        assert ((d - border).abs() > h * v.abs().max()).all()
    old, ref, adv = lp - d, lp + 0.4 * randn(4, 9, seed=64), randn(4, seed=65)

    def f(x):
        return nq.policy_loss(x, old.to(DEV), adv.to(DEV), ref_logprobs=ref.to(DEV), kl_coef=0.3)[0]
    x = lp.to(DEV).requires_grad_()
    (g,) = torch.autograd.grad(f(x), x)
    with torch.no_grad():
        diff = float(f((lp + h * v).to(DEV)).double() - f((lp - h * v).to(DEV)).double()) / (2 * h)
    # a term's third derivative is under (|r A| + 0.3 e^q) |v|^3, its value off by some 16 u and by u |lp| of its input
    big = float((d.exp() * 2).max() * adv.abs().max() + 0.3 * 2 * (ref - lp).exp().max())
    bound = big * float(v.abs().max()) ** 3 * h * h / 6 + big * (16 + float(lp.abs().max()) * 2) * U / h
    assert abs(diff - float((g.cpu().double() * v).sum())) <= bound


def test_preference_loss_refusals():
    x = torch.zeros(3, 5, device=DEV)
    bad = [(ValueError, dict(kind="other")), (ValueError, dict(beta=0.0)), (ValueError, dict(beta=float("inf"))),
           (ValueError, dict(label_smoothing=0.5)), (ValueError, dict(label_smoothing=0.1, kind="ipo")),
           (ValueError, dict(ref_chosen=x[:2])), (ValueError, dict(rejected_mask=x[:, :4] > 0)),
           (TypeError, dict(ref_chosen=x.half())), (RuntimeError, dict(chosen_mask=x.cpu() > 0))]
    for err, kw in bad:
        with pytest.raises(err):
            nq.preference_loss(x, x, **kw)
    for a, b in ((x, x[:2]), (x[:0], x[:0]), (x[None], x[None]), (x.half(), x.half()), (x.cpu(), x.cpu())):
        with pytest.raises((ValueError, TypeError, RuntimeError)):
            nq.preference_loss(a, b)


# ---------------------------------------------------------------- policy_loss

def policy_reference(lp, old, adv, ref, mask, low, high, c, reduction):
    lp = lp.double().requires_grad_()
    mask = torch.ones(lp.shape, dtype=torch.bool) if mask is None else mask
    a = adv.double() if adv.dim() == 2 else adv.double()[:, None].expand(lp.shape)
    d = torch.where(mask, lp - old.double(), 0.0)
    r = torch.exp(d)
    clip = r.clamp(1 - low, 1 + high)
    each = -torch.minimum(r * a, clip * a)
    cut = (clip * a < r * a) & mask
    kl = torch.zeros_like(d)
    if ref is not None:
        q = torch.where(mask, ref.double() - lp, 0.0)
        kl = torch.expm1(q) - q
        each = each + c * kl
    n = mask.sum().clamp(min=1)
    rows = mask.sum(1).clamp(min=1)
    kept = torch.where(mask, each, 0.0)
    loss = kept.sum() / n if reduction == "token" else (kept.sum(1) / rows).mean()
    (grad,) = torch.autograd.grad(loss, lp)
    # a term: the exponent's rounding |d| u, some 8 operations; its share likewise in the gradient
    share = (1 / n if reduction == "token" else 1 / (rows[:, None] * len(lp))).double()
    size = ((r * a).abs() + abs(c) * (kl.abs() + (lp - lp + 1) * (torch.expm1(-torch.log1p(kl))).abs() + kl.abs().sqrt() * 2)).detach()
    tol = torch.where(mask, size * (d.abs().detach() + 16) * U * share, 0.0)
    kl_mean = torch.where(mask, kl, 0.0).sum().detach() / n
    return loss.detach(), kl_mean, cut.sum() / n.double(), grad, tol


@pytest.mark.parametrize("B,S", [(1, 1), (3, 40), (16, 1024), (17, 33), (2, 1025), (2, 5000), (300, 70), (3, 0)])
@pytest.mark.parametrize("reduction", ["token", "sequence"])
@pytest.mark.parametrize("c,per_token", [(0.0, False), (0.05, False), (0.3, True)])
def test_policy_loss(B, S, reduction, c, per_token):
    say(f"policy_loss {B} {S} {reduction} {c} {per_token}")
    lp = -randn(B, S, seed=50).abs()
    old, ref = lp + 0.3 * randn(B, S, seed=51), lp + 0.4 * randn(B, S, seed=52)
    adv = randn(B, S, seed=53) if per_token else randn(B, seed=53)
    for mask in (ragged(B, S, 54), None, torch.zeros(B, S, dtype=torch.bool)):
        want = policy_reference(lp, old, adv, ref if c else None, mask, 0.2, 0.28, c, reduction)
        ins = [t.clone() for t in (lp, old, ref)]
        if mask is not None:
            for t in ins:
                t[~mask] = float("nan")  # what a masked token holds has no effect
        l, o, r = (t.to(DEV) for t in ins)
        l.requires_grad_()
        loss, kl, clipped = nq.policy_loss(l, o, adv.to(DEV), ref_logprobs=r if c else None,
                                           mask=None if mask is None else mask.to(DEV), clip_low=0.2, clip_high=0.28,
                                           kl_coef=c, reduction=reduction)
        (g,) = torch.autograd.grad(3.0 * loss, l)
        assert loss.shape == kl.shape == clipped.shape == () and not kl.requires_grad
        within(loss, want[0], float(want[4].sum()) + U * want[0].abs() + 1e-14, "loss")
        within(kl, want[1], 16 * U * want[1] + 1e-14, "kl")
        within(clipped, want[2], U * want[2], "clipped")
        within(g, 3 * want[3], 3 * want[4] + 4 * U * (3 * want[3]).abs(), "gradient")


def test_policy_loss_borders_and_small_ratios():
    """Tokens next to a clip border, KL terms of nearly equal policies, ratios that overflow."""
    say("policy_loss borders")
    hi = math.log1p(0.2)
    base = torch.tensor(-3.0)
    steps = torch.arange(-40, 41) * 2.0 ** -23
    old = torch.full((2, 81), -3.0)
    lp = (base.double() + hi + steps.double()).float().expand(2, 81).clone()
    lp[1] = (base.double() + math.log1p(-0.2) + steps.double()).float()
    adv = torch.tensor([1.0, -1.0])
    want = policy_reference(lp, old, adv, None, None, 0.2, 0.2, 0.0, "token")
    l = lp.to(DEV).requires_grad_()
    loss, _, clipped = nq.policy_loss(l, old.to(DEV), adv.to(DEV))
    (g,) = torch.autograd.grad(loss, l)
    assert 0 < float(want[2]) < 1
    within(clipped, want[2], U, "share at the border")
    within(g, want[3], want[4] + 4 * U * want[3].abs(), "gradient at the border")
    # e^q - q - 1 of q from 2^-20 to 8, both signs
    q = torch.cat([2.0 ** torch.arange(-20, 3.1, 0.1), -2.0 ** torch.arange(-20, 3.1, 0.1)])
    for i in range(0, len(q), 20):
        lp = torch.zeros(1, len(q[i:i + 20]))
        ref = q[i:i + 20].float()[None]
        want = policy_reference(lp, lp, torch.zeros(1), ref, None, 0.2, 0.2, 1.0, "token")
        l = lp.to(DEV).requires_grad_()
        loss, kl, _ = nq.policy_loss(l, lp.to(DEV), torch.zeros(1, device=DEV), ref_logprobs=ref.to(DEV), kl_coef=1.0)
        (g,) = torch.autograd.grad(loss, l)
        within(kl, want[1], 16 * U * want[1], "kl")
        within(g, want[3], 8 * U * want[3].abs(), "kl gradient")
    # ratios that overflow: the clip decides where it applies, infinity where it does not
    l = torch.zeros(2, 2, device=DEV, requires_grad=True)
    o = torch.full((2, 2), -200.0, device=DEV)
    loss, _, clipped = nq.policy_loss(l[:1].detach(), o[:1], torch.ones(1, device=DEV))
    assert abs(float(loss) + 1.2) < 1e-6 and float(clipped) == 1
    assert float(nq.policy_loss(l[:1].detach(), o[:1], -torch.ones(1, device=DEV))[0]) == float("inf")


def test_policy_loss_strides_and_refusals():
    say("policy_loss strides, refusals")
    lp = -randn(4, 20, seed=56).abs()
    old = lp + 0.2 * randn(4, 20, seed=57)
    adv, m = randn(8, seed=58), ragged(4, 20, 59)
    want = policy_reference(lp[:, 3:], old[:, 3:], adv[::2], None, m[:, 3:], 0.2, 0.2, 0.0, "sequence")
    l = lp.to(DEV).requires_grad_()
    loss, *_ = nq.policy_loss(l[:, 3:], old.t().contiguous().to(DEV).t()[:, 3:], adv.to(DEV)[::2], mask=m.to(DEV)[:, 3:].float(),
                              reduction="sequence")
    (g,) = torch.autograd.grad(loss, l)
    within(loss, want[0], float(want[4].sum()) + U * want[0].abs(), "strided")
    within(g[:, 3:], want[3], want[4] + 4 * U * want[3].abs(), "strided gradient")
    assert not g[:, :3].any()
    x, a = torch.zeros(3, 5, device=DEV), torch.zeros(3, device=DEV)
    bad = [(ValueError, dict(clip_low=1.5)), (ValueError, dict(clip_low=-0.1)), (ValueError, dict(clip_high=float("nan"))),
           (ValueError, dict(kl_coef=0.1)), (ValueError, dict(reduction="sum")), (ValueError, dict(mask=x[:2] > 0)),
           (ValueError, dict(ref_logprobs=x[:, :2])), (TypeError, dict(ref_logprobs=x.half())),
           (RuntimeError, dict(mask=x.cpu() > 0)), (ValueError, dict(kl_coef=float("inf"), ref_logprobs=x))]
    for err, kw in bad:
        with pytest.raises(err):
            nq.policy_loss(x, x, a, **kw)
    for args in ((x[0], x[0], a), (x[:0], x[:0], a[:0]), (x, x[:2], a), (x, x, a[:2]), (x, x, x[:, :2]), (x.half(), x, a),
                 (x.cpu(), x.cpu(), a.cpu())):
        with pytest.raises((ValueError, TypeError, RuntimeError)):
            nq.policy_loss(*args)


# ---------------------------------------------------------------- streams, graphs, bits

def test_losses_on_another_stream_and_twice():
    """On a stream of their own, beside the same calls on another, each call's bits are those of the call alone."""
    say("losses on streams")
    x = randn(64, 30011, seed=60, dtype=BF).to(DEV)
    y = torch.randint(0, 30011, (64,), device=DEV)
    m = ragged(32, 2, 61).to(DEV)

    def step():
        leaf = x.detach().requires_grad_()
        lp = nq.token_logprobs(leaf, y)
        loss, *_ = nq.preference_loss(lp[:32, None].expand(32, 2), lp[32:, None].expand(32, 2), chosen_mask=m)
        pol, *_ = nq.policy_loss(lp.view(8, 8), lp.detach().view(8, 8) + 0.1, torch.ones(8, device=DEV))
        return [loss.detach(), pol.detach(), lp.detach(), *torch.autograd.grad(loss + pol, leaf)]

    want = step()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(2):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(step())
    torch.cuda.synchronize()
    for g in got:
        assert all(torch.equal(a, b) for a, b in zip(g, want))


def test_losses_in_a_graph():
    """Forward and backward captured, replayed on new inputs with eager work between."""
    say("losses in a HIP graph")
    B, S, V = 6, 11, 5003
    x = torch.empty(2 * B, S, V, device=DEV, dtype=BF, requires_grad=True)
    y = torch.empty(2 * B, S, device=DEV, dtype=torch.long)
    ref = torch.empty(2 * B, S, device=DEV)

    def fill(i):
        with torch.no_grad():
            x.copy_(randn(2 * B, S, V, seed=70 + i, dtype=BF, scale=2))
            y.copy_(torch.randint(-1, V, (2 * B, S), generator=torch.Generator().manual_seed(80 + i)))
            y.masked_fill_(y == -1, -100)
            ref.copy_(-randn(2 * B, S, seed=90 + i).abs() * 10)

    def step():
        lp = nq.token_logprobs(x, y)
        keep = y != -100
        loss, rc, rr = nq.preference_loss(lp[:B], lp[B:], ref[:B], ref[B:], chosen_mask=keep[:B], rejected_mask=keep[B:])
        pol, kl, cut = nq.policy_loss(lp, ref, ref[:, 0], ref_logprobs=ref, mask=keep, kl_coef=1e-3)
        grads = torch.autograd.grad(loss + pol, x)
        return [t.detach() for t in (loss, rc, rr, pol, kl, cut, *grads)]

    fill(0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for i in range(3):
        fill(i)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in outs]
        for a, b in zip(got, step()):
            assert torch.equal(a, b)


def test_losses_under_autograd_modes():
    """Saved tensors that travel to the host and back, a graph gone through twice, inputs written to before
    the backward, inference mode, a mask or labels that change: the same bits or an error, never stale values."""
    say("losses under autograd modes")
    x = randn(2, 9, 301, seed=95, dtype=BF).to(DEV)
    h = randn(2, 70, 64, seed=96).to(BF).to(DEV)
    w = randn(90, 64, seed=97).to(BF).to(DEV)
    y = torch.randint(0, 90, (2, 70), device=DEV)
    m = ragged(2, 9, 98).to(DEV)
    old = randn(2, 9, seed=99).to(DEV)

    def losses(x, h, w, y=y, m=m):
        lp = nq.token_logprobs(x, y[:, :9])
        pref, *_ = nq.preference_loss(lp[:1], lp[1:], chosen_mask=m[:1], rejected_mask=m[1:])
        pol, *_ = nq.policy_loss(lp, old, old[:, 0], mask=m)
        return pref + pol + nq.linear_logprobs(h, w, y).sum()

    def leaves():
        return [t.clone().requires_grad_() for t in (x, h, w)]

    ins = leaves()
    loss = losses(*ins)
    want = torch.autograd.grad(loss, ins, retain_graph=True)
    for a, b in zip(torch.autograd.grad(loss, ins), want):
        assert torch.equal(a, b)
    ins = leaves()
    with torch.autograd.graph.save_on_cpu():
        loss = losses(*ins)
    torch.empty(1 << 24, device=DEV).fill_(7)  # over what the forward held
    for a, b in zip(torch.autograd.grad(loss, ins), want):
        assert torch.equal(a, b)
    for change in ("labels", "mask", "hidden"):
        ins = leaves()
        y2, m2, mid = y.clone(), m.clone(), ins[1] * 1
        loss = losses(ins[0], mid, ins[2], y2, m2)
        {"labels": y2, "mask": m2, "hidden": mid}[change].zero_()
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            torch.autograd.grad(loss, ins)
    with torch.inference_mode():
        inside = losses(x, h, w)
    with torch.no_grad():
        assert torch.equal(inside, losses(x, h, w))
    # transforms that the kernels have no part in are refused, not answered with other numbers
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda t: nq.token_logprobs(t, y[:, :9]), (x.float(),), (x.float(),))
    with pytest.raises(Exception):
        torch.vmap(lambda t: nq.token_logprobs(t, y[0, :9]))(x.float())


@pytest.mark.filterwarnings("ignore::torch.jit.TracerWarning", "ignore:.*jit.*:DeprecationWarning")
def test_losses_traced_and_compiled():
    """A trace, which would hold uninitialised outputs, is refused; a compiled function breaks its graph at the
    kernels and gives their bits; tensors without memory of their own are refused."""
    from torch.fx.experimental.proxy_tensor import make_fx
    from torch.testing._internal.two_tensor import TwoTensor
    say("losses traced and compiled")
    y = torch.randint(0, 77, (2, 6), generator=torch.Generator().manual_seed(1)).to(DEV)
    h, w = randn(2, 6, 64, seed=2, dtype=BF).to(DEV), randn(77, 64, seed=3, dtype=BF).to(DEV)
    x, lp = randn(2, 6, 77, seed=4).to(DEV), randn(2, 6, seed=5).to(DEV)
    m = ragged(2, 6, 6).to(DEV)
    calls = [(lambda x: nq.token_logprobs(x, y), x), (lambda h: nq.linear_logprobs(h, w, y), h),
             (lambda t: nq.preference_loss(t[:1], t[1:], chosen_mask=m[:1], rejected_mask=m[1:])[0], lp),
             (lambda t: nq.policy_loss(t, lp + 0.1, lp[:, 0], mask=m)[0], lp)]
    for call, first in calls:
        with pytest.raises(RuntimeError, match="trace"):
            torch.jit.trace(call, (first,), check_trace=False)
        with pytest.raises(RuntimeError, match="trace"):
            make_fx(call)(first)
        with pytest.raises(TypeError, match="memory"):
            call(TwoTensor(first, first))
        torch._dynamo.reset()
        compiled = torch.compile(lambda t: call(t * 2) * 3, backend="eager")
        assert torch.equal(compiled(first), call(first * 2) * 3)
        a, b = first.clone().requires_grad_(), first.clone().requires_grad_()
        got, want = compiled(a), call(b * 2) * 3
        assert torch.equal(got, want)
        d = torch.ones_like(want)
        assert torch.equal(torch.autograd.grad(got, a, d)[0], torch.autograd.grad(want, b, d)[0])
    torch._dynamo.reset()
    for kw in (dict(mask=TwoTensor(m, m)), dict(ref_logprobs=TwoTensor(lp, lp))):
        with pytest.raises(TypeError, match="memory"):
            nq.policy_loss(lp, lp, lp, **kw)


@pytest.mark.parametrize("B,S", [(2, 3), (20, 3)])
@pytest.mark.parametrize("reduction", ["token", "sequence"])
def test_policy_loss_zero_advantage(B, S, reduction):
    """A token without an advantage adds its KL term alone, also where its ratio overflows; NaN stays NaN."""
    say(f"policy_loss zero advantage {B} {S} {reduction}")
    lp = -randn(B, S, seed=62).abs()
    old = lp + 0.1 * randn(B, S, seed=63)
    old[1, 1], old[1, 2] = -300.0, -float("inf")
    ref = lp + 0.3 * randn(B, S, seed=64)
    adv = randn(B, seed=65)
    adv[1] = 0
    for c in (0.0, 0.2):
        # the same tokens with ratios that do not overflow: the row's policy term is 0 either way
        plain = old.clone()
        plain[1] = lp[1]
        want = policy_reference(lp, plain, adv, ref, None, 0.2, 0.28, c, reduction)
        l = lp.to(DEV).requires_grad_()
        loss, _, clipped = nq.policy_loss(l, old.to(DEV), adv.to(DEV), ref_logprobs=ref.to(DEV), clip_high=0.28, kl_coef=c,
                                          reduction=reduction)
        (g,) = torch.autograd.grad(loss, l)
        within(loss, want[0], float(want[4].sum()) + U * want[0].abs() + 1e-14, "loss")
        within(clipped, want[2], U * want[2], "clipped")
        within(g, want[3], want[4] + 4 * U * want[3].abs(), "gradient")
        assert c or not g[1].any()
    old[1, 0] = float("nan")
    l = lp.to(DEV).requires_grad_()
    loss, *_ = nq.policy_loss(l, old.to(DEV), adv.to(DEV), reduction=reduction)
    (g,) = torch.autograd.grad(loss, l)
    assert torch.isnan(loss) and torch.isnan(g).sum() == 1 and torch.isnan(g[1, 0])


@pytest.mark.parametrize("B", [3, 20])
@pytest.mark.parametrize("kind", ["sigmoid", "hinge", "ipo"])
def test_preference_loss_of_nan(B, kind):
    """A pair whose margin is NaN has NaN gradients, as its loss; the other pairs' are their own."""
    say(f"preference_loss NaN {B} {kind}")
    c, r = randn(B, 5, seed=66), randn(B, 5, seed=67)
    c[1, 2] = float("nan")
    leaves = [t.to(DEV).requires_grad_() for t in (c, r)]
    loss, wc, wr = nq.preference_loss(*leaves, kind=kind)
    assert torch.isnan(loss) and torch.isnan(wc).sum() == 1 and torch.isnan(wc[1]) and torch.isfinite(wr).all()
    for g in torch.autograd.grad(loss, leaves):
        assert torch.isnan(g[1]).all() and torch.isnan(g).sum() == 5


@pytest.mark.parametrize("B", [2, 20])
@pytest.mark.parametrize("e", [0.0, 0.25])
def test_preference_loss_of_infinite_margins(B, e):
    """A label that the policy rules out: the margin is infinite, and so is the loss that weighs it."""
    say(f"preference_loss infinite margins {B} {e}")
    inf = float("inf")
    for side, want in ((0, inf), (1, inf if e else 0.0)):
        lps = [torch.zeros(B, 4), torch.zeros(B, 4)]
        lps[side][1, 3] = -inf
        leaves = [t.to(DEV).requires_grad_() for t in lps]
        loss, *rewards = nq.preference_loss(*leaves, beta=0.5, label_smoothing=e)
        # the other pairs' margins are 0: log 2 each
        within(loss, torch.tensor(want + (B - 1) / B * math.log(2), dtype=torch.float64), 4 * U, f"side {side}")
        assert float(rewards[side][1]) == -inf and torch.isfinite(rewards[1 - side]).all()
        # beta (e - s(-h)): s(-h) is 1 at -inf, 0 at inf, 1/2 at 0
        slope = torch.full((B,), 0.5 * (e - 0.5), dtype=torch.float64)
        slope[1] = 0.5 * (e - (1 if side == 0 else 0))
        for g, sign in zip(torch.autograd.grad(loss, leaves), (1, -1)):
            within(g, (sign * slope / B)[:, None].expand(B, 4), 2 * U * slope.abs().max() / B, f"side {side} gradient")


def test_token_logprobs_more_rows_than_one_launch():
    """A launch has fewer than 2^32 threads: 2^26 rows of a wave, 2^24 workgroups of the backward."""
    rows, V = 2 ** 26 + 5, 3
    say(f"token_logprobs {rows} rows")
    g = torch.Generator(device=DEV).manual_seed(68)
    x = torch.randn(rows, V, generator=g, device=DEV, dtype=BF).requires_grad_()
    labels = torch.randint(0, V, (rows,), generator=g, device=DEV)
    dy = torch.randn(rows, generator=g, device=DEV)
    lp = nq.token_logprobs(x, labels)
    (dx,) = torch.autograd.grad(lp, x, dy)
    # the first and last rows, those around the launches' ends, and a sample of the rest
    at = torch.cat([torch.arange(0, rows, 8191), torch.arange(2 ** 24 - 9, 2 ** 24 + 9), torch.arange(2 ** 26 - 99, rows)]).to(DEV)
    xs = x.detach()[at].cpu()
    want, dwant, tol, dtol = token_reference(xs, labels[at].cpu(), dy[at].cpu(), 1.0)
    within(lp[at], want, tol, "logprobs")
    within(dx[at], dwant, dtol + half_step(BF) * dwant.abs(), "dlogits")
    # every row was written, once
    assert bool((lp < 0).all()) and float(dx.sum(-1, dtype=torch.float32).abs().max()) < 0.1


def test_losses_of_more_sequences_than_one_launch():
    """2^24 workgroups of 256 threads, 2^22 of 1024."""
    g = torch.Generator(device=DEV).manual_seed(69)
    B = 2 ** 24 + 3
    say(f"preference_loss and policy_loss {B} sequences")
    c, r = (torch.randn(B, generator=g, device=DEV) for _ in range(2))
    leaves = [t.clone().requires_grad_() for t in (c, r)]
    loss, wc, wr = nq.preference_loss(*leaves, beta=0.5)
    h = 0.5 * (c.double() - r.double())
    # 1 / (1 + e^h) / B: a rounding of the slope, of the coefficient and of the mean
    assert abs(float(loss.detach()) - float(torch.nn.functional.softplus(-h).mean())) < 4 * U
    slope = -0.5 / (1 + torch.exp(h)) / B
    for got, sign in zip(torch.autograd.grad(loss, leaves), (1, -1)):
        assert float((got.double() / (sign * slope) - 1).abs().max()) < 4 * U
    assert float((wc.double() - 0.5 * c).abs().max()) == 0 and float((wr.double() - 0.5 * r).abs().max()) == 0
    l = (0.1 * c)[:, None].requires_grad_()
    loss, _, clipped = nq.policy_loss(l, torch.zeros_like(l), r, reduction="sequence")
    d, a = l.detach()[:, 0].double(), r.double()
    hi, lo = (a > 0) & (d > math.log1p(0.2)), (a < 0) & (d < math.log1p(-0.2))
    term = -torch.where(hi, 1.2 * a, torch.where(lo, 0.8 * a, d.exp() * a))
    # each term in fp32: |d| < 1, the exponential and two products under 4 roundings of |term|
    assert abs(float(loss.detach()) - float(term.mean())) < 8 * U * float(term.abs().mean())
    assert abs(float(clipped) - float((hi | lo).double().mean())) < 2 * U
    grad = torch.where(hi | lo, 0.0, -d.exp() * a) / B
    (got,) = torch.autograd.grad(loss, l)
    assert bool(((got[:, 0].double() - grad).abs() <= 8 * U * grad.abs()).all())
    B = 2 ** 22 + 3
    with torch.no_grad():
        loss, wc, _ = nq.preference_loss(c[:B, None].expand(B, 1025), r[:B, None].expand(B, 1025), average=True, beta=0.5)
    # averages of 1025 equal values in 64 bits
    assert abs(float(loss) - float(torch.nn.functional.softplus(-h[:B]).mean())) < 4 * U
    assert float((wc.double() - 0.5 * c[:B]).abs().max()) <= U * float(c[:B].abs().max())


# Logits of more than 256 MB are loaded past the cache: rows cut into slices, a wave each and a workgroup each
@pytest.mark.parametrize("rows,V,dt", [(1000, 151936, BF), (70000, 2055, BF), (16500, 8201, BF),
                                       (600, 151936, F32), (70000, 1033, F32), (2100, 50257, F32)])
def test_token_logprobs_past_the_cache(rows, V, dt):
    say(f"token_logprobs past the cache {rows} x {V} {dt}")
    assert rows * V * (2 if dt == BF else 4) > 2 ** 28
    g = torch.Generator(device=DEV).manual_seed(33)
    x = torch.randn(rows, V, generator=g, device=DEV, dtype=dt).mul_(3).requires_grad_()
    labels = torch.randint(0, V, (rows,), generator=g, device=DEV)
    labels[5::7], labels[3], labels[11] = -100, V - 1, 0
    dy = torch.randn(rows, generator=g, device=DEV)
    lp = nq.token_logprobs(x, labels, temperature=0.8)
    (dx,) = torch.autograd.grad(lp, x, dy)
    assert bool(torch.isfinite(lp).all())
    for at in torch.arange(rows, device=DEV).split(max(1, 2 ** 25 // V)):
        want, dwant, tol, dtol = token_reference(x.detach()[at], labels[at], dy[at], 0.8)
        assert bool(((lp[at].double() - want).abs() <= tol).all()), int(at[0])
        assert bool(((dx[at].double() - dwant).abs() <= dtol + half_step(dt) * dwant.abs()).all()), int(at[0])


def test_losses_with_a_negative_view_as_gradient():
    """A complex number's backward gives the imaginary part of a conjugate: its memory holds the opposite."""
    say("losses with a negative view as gradient")
    y = torch.tensor([1, 2, 0]).to(DEV)
    h, w = randn(3, 64, seed=91, dtype=BF).to(DEV), randn(77, 64, seed=92, dtype=BF).to(DEV)
    x, lp = randn(3, 77, seed=93).to(DEV), randn(3, 6, seed=94).to(DEV)
    for call, first in ((lambda t: nq.token_logprobs(t, y), x), (lambda t: nq.linear_logprobs(t, w, y), h),
                        (lambda t: nq.preference_loss(t, lp)[0], 0.5 * lp), (lambda t: nq.policy_loss(t, lp, lp[:, 0])[0], 0.9 * lp)):
        leaf = first.clone().requires_grad_()
        out = call(leaf)
        d = randn(out.numel(), seed=95).view(out.shape).to(DEV)
        view = torch._neg_view(-d)
        assert view.is_neg()
        want, got = (torch.autograd.grad(out, leaf, t, retain_graph=True)[0] for t in (d, view))
        assert torch.equal(got, want) and bool(want.any())
